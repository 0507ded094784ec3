"""The gated feed-forward over every way its launches are cut: tile size (128 square, 256 x 192, 256 square), whole rounds, a last
round split along k, and both in one launch, for each of its five products.  The shapes were searched for that: each brings cuts
that the ones before it do not reach."""
import ctypes

import pytest
import torch

import train_refs as R

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
ACTS = (("erf", "EPI_GELU_ERF"), ("tanh", "EPI_GELU_TANH"), ("silu", "EPI_SILU"))

# tile (8: 256 square, 6: 256 x 192, 4: 128 square) and cut that the shape is the first to bring; up / down: the forward products
CUTS = [(70, 136, 520),          # 4 whole: up, dvalue / dgate, weights; split: 6 down, 4 dx
        (6549, 1160, 8),         # 4 split: up, dvalue / dgate, weights; 4 rounds: down; 8 whole: dx
        (227, 4488, 520),        # 4 whole: down, dx; 8 whole: weights
        (5400, 3624, 208),       # 8 split: up, weights; rounds: 6 down, 4 dx
        (64, 264, 7528),         # 4 split: down; 4 rounds: weights
        (2328, 3520, 1672),      # 8 split: dvalue / dgate; 8 rounds and split: weights; 4 rounds and split: dx; 6 whole: up, down
        (16286, 776, 392),       # rounds: 4 dvalue / dgate, 8 up, down, dx
        (2947, 952, 2728),       # 8 whole: dvalue / dgate; 8 split: dx; 4 rounds and split: weights; 6 rounds: up
        (10958, 968, 648),       # 4 rounds and split: dvalue / dgate; 4 rounds: up; 8 whole: down
        (522, 544, 8760),        # 8 whole: up; 8 rounds: weights
        (7215, 2192, 1136),      # 8 rounds and split: up, down, dx
        (3561, 1224, 4776),      # 8 rounds and split: dvalue / dgate; 8 split: down
        (16236, 760, 800),       # 8 rounds: dvalue / dgate
        (6841, 3472, 1096)]      # 6 rounds and split: down


def rnd(*shape, scale=1.0, seed=0, dt=BF, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)


def case(M, D, F, dt, bias, seed=0):
    W = (rnd(F, D, scale=D ** -0.5, seed=seed + 2, dt=dt), rnd(F, D, scale=D ** -0.5, seed=seed + 3, dt=dt), rnd(D, F, scale=F ** -0.5, seed=seed + 4, dt=dt))
    b = [rnd(n, scale=0.3, seed=seed + 6 + i, dt=dt) if bias else None for i, n in enumerate((F, F, D))]
    return rnd(M, D, seed=seed + 1, dt=dt), rnd(M, D, seed=seed + 5, dt=dt), W, b


def check(got, pair, what):
    """train_refs.check on the device"""
    ref, bound = pair
    off = (got.double() - ref).abs()
    bad = ~(off <= bound)
    assert got.shape == ref.shape and not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / bound).nan_to_num(9e9).max()):.3g} x"


def d64(t):
    return None if t is None else t.double()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("i", range(len(CUTS)), ids=["x".join(map(str, c)) for c in CUTS])
def test_every_cut(dev, i, dt):
    from flux_generator_amd import ops
    M, D, F = CUTS[i]
    kind, name = ACTS[(i + (dt == HF)) % 3]
    act, bias = getattr(ops, name), (i + (dt == HF)) % 2 == 0
    x, dy, W, b = case(M, D, F, dt, bias, seed=100 + i)
    y, saved = ops.gated_ff(x, *W, *b, act=act, save=True)
    for what, got, pair in zip(("y", "value", "gate", "hidden"), (y, *saved), R.ff_forward_bound(d64(x), *map(d64, W), *map(d64, b), kind, dt)):
        check(got, pair, what)
    again, saved2 = ops.gated_ff(x, *W, *b, act=act, save=True)
    assert torch.equal(y, again) and all(torch.equal(p, q) for p, q in zip(saved, saved2))
    assert torch.equal(y, ops.gated_ff(x, *W, *b, act=act))
    out = ops.gated_ff_backward(dy, x, saved, *W, act=act, bias_grads=True)
    pairs = R.ff_backward_bound(d64(dy), d64(x), *map(d64, saved), *map(d64, W), kind, dt)
    for what, got, pair in zip(("dx", "dw_value", "dw_gate", "dw_out", "db_value", "db_gate", "db_out"), out, pairs):
        check(got, pair, what)
    assert all(torch.equal(p, q) for p, q in zip(out, ops.gated_ff_backward(dy, x, saved, *W, act=act, bias_grads=True)))
    frozen = ops.gated_ff_backward(dy, x, (*saved[:2], None), *W, act=act, weight_grads=False)
    assert torch.equal(frozen[0], out[0])


@pytest.mark.parametrize("M,D,F", [(10958, 968, 648), (3561, 1224, 4776), (2328, 3520, 1672), (1744, 992, 4704), (2947, 952, 2728)])
def test_cut_launches_write_nothing_else(dev, M, D, F):
    """Outputs and workspace between guard words, where whole and split tiles share one workspace."""
    from flux_generator_amd import ops
    from flux_generator_amd._lib import GatedFfDesc, GatedFfGradDesc, load
    lib = load()
    x, dy, W, b = case(M, D, F, BF, True, seed=40)
    st = torch.cuda.current_stream().cuda_stream
    ptr = lambda *ts: [q.data_ptr() for q in ts]

    def guarded(*bytes_):
        offs, n = [], 4096
        for k in bytes_:
            offs.append(n)
            n = -(-(n + k) // 256) * 256 + 4096
        return torch.full((n,), 0xA5, dtype=torch.uint8, device=dev), offs

    def look(buf, offs, sizes, want):
        keep = torch.ones_like(buf, dtype=torch.bool)
        for o, k in zip(offs, sizes):
            keep[o:o + k] = False
        assert bool((buf[keep] == 0xA5).all())
        for o, w in zip(offs, want):
            assert torch.equal(buf[o:o + w.numel() * 2].view(BF).view(w.shape), w)

    y, sv = ops.gated_ff(x, *W, *b, act=ops.EPI_SILU, save=True)
    sizes = [2 * M * F] * 3 + [2 * M * D, lib.fluxhip_gated_ff_ws(M, D, F)]
    buf, offs = guarded(*sizes)
    at = [buf.data_ptr() + o for o in offs]
    d = GatedFfDesc(*ptr(x, *W, *b), *at[:4], M, D, D, F, ops.EPI_SILU, 0, at[4], sizes[4])
    assert lib.fluxhip_gated_ff(d, st) == 0
    look(buf, offs, sizes, (*sv, y))

    out = ops.gated_ff_backward(dy, x, sv, *W, act=ops.EPI_SILU, bias_grads=True)
    sizes = [2 * q.numel() for q in out] + [2 * M * F] * 2 + [lib.fluxhip_gated_ff_grad_ws(M, D, F)]
    buf, offs = guarded(*sizes)
    at = [buf.data_ptr() + o for o in offs]
    d = GatedFfGradDesc(*ptr(dy, x, *sv, *W), at[7], at[8], *at[:7], M, D, D, D, F, ops.EPI_SILU, 0, at[9], sizes[9])
    assert lib.fluxhip_gated_ff_grad(d, st) == 0
    look(buf, offs, sizes, out)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,D,F", [(609, 4768, 3384), (559, 5104, 3224), (14143, 4736, 136), (2152, 4720, 784), (531, 3208, 2528), (77, 264, 520)])
def test_weight_gradients_one_by_one(dev, M, D, F, dt):
    """The C entry point's dw_out alone, and dw_value with dw_gate alone: launches of one and of two products."""
    from flux_generator_amd import ops
    from flux_generator_amd._lib import GatedFfGradDesc, load
    lib = load()
    x, dy, W, b = case(M, D, F, dt, False, seed=60)
    _, sv = ops.gated_ff(x, *W, act=ops.EPI_SILU, save=True)
    pairs = R.ff_backward_bound(d64(dy), d64(x), *map(d64, sv), *map(d64, W), "silu", dt)
    n = lib.fluxhip_gated_ff_grad_ws(M, D, F)
    st = torch.cuda.current_stream().cuda_stream
    for which in ((1, 2), (3,)):
        dw = {k: torch.empty(pairs[k][0].shape, dtype=dt, device=dev) for k in which}
        mid, ws = torch.empty(2, M, F, dtype=dt, device=dev), torch.empty(n, dtype=torch.uint8, device=dev)
        d = GatedFfGradDesc()
        for k, t in zip(("dy", "x", "value", "gate", "hidden", "w_value", "w_gate", "w_out", "dvalue", "dgate", "ws"), (dy, x, *sv, *W, mid[0], mid[1], ws)):
            setattr(d, k, t.data_ptr())
        for k, t in dw.items():
            setattr(d, ("", "dw_value", "dw_gate", "dw_out")[k], t.data_ptr())
        d.M, d.ldx, d.lddy, d.D, d.F, d.act, d.dtype, d.ws_bytes = M, D, D, D, F, ops.EPI_SILU, int(dt == HF), n
        assert lib.fluxhip_gated_ff_grad(ctypes.byref(d), st) == 0
        for k, t in dw.items():
            check(t, pairs[k], ("dx", "dw_value", "dw_gate", "dw_out")[k])

"""Adapter-training operators with infinities, NaN and extreme values in their operands, and in place over many rows."""
import pytest
import torch

import train_refs as R

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def rnd(*shape, scale=1.0, mean=0.0, seed=0, dt=BF):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dt)


def D64(t):
    return t.detach().cpu().double()


# ------------------------------------------------------------------------------------------------ LayerNorm
# (rows, width): one block and several, every number of threads a row, last rounds that leave row groups without a row, and (rows
# up to 512) sums over the inputs themselves; 9001: rows too wide for registers
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("per", [False, True])
@pytest.mark.parametrize("T,D", [(5, 64), (1001, 64), (2051, 100), (1003, 771), (517, 1280), (1, 8), (301, 640), (2050, 2560), (1030, 4100), (70, 9001)])
def test_layernorm_infinities_stay_in_their_row_and_column(dev, T, D, per, dt):
    from flux_generator_amd import ops
    B = 2 if per else 1
    x, dy = rnd(B, T, D, mean=0.5, seed=1, dt=dt).to(dev), rnd(B, T, D, seed=2, dt=dt).to(dev)
    g = rnd(*((B, D) if per else (D,)), scale=0.2, mean=1.0, seed=3, dt=dt).to(dev)
    y, mu, r = ops.layernorm(x, g, None)
    for row in (T - 1, 0, T // 2):
        c = (7 * row + 3) % D
        clean = dy.clone()
        clean[-1, row, c] = 0
        bad = dy.clone()
        bad[-1, row, c] = INF
        cx, cg, cb = ops.layernorm_backward(clean, x, mu, r, g)
        bx, bg, bb = ops.layernorm_backward(bad, x, mu, r, g)
        other = torch.ones(B, T, dtype=torch.bool, device=dev)
        other[-1, row] = False
        assert torch.equal(bx[other], cx[other]) and not bool(bx[-1, row].isfinite().any())
        col = torch.ones_like(g, dtype=torch.bool)
        col.view(-1, D)[-1, c] = False
        assert torch.equal(bg[col], cg[col]) and torch.equal(bb[col], cb[col])
        xh = (x[-1, row, c].double() - mu[-1, row]) * r[-1, row]
        assert float(bb.view(-1, D)[-1, c]) == INF, (row, bb.view(-1, D)[-1, c])
        assert float(bg.view(-1, D)[-1, c]) == (INF if float(xh) > 0 else -INF), (row, float(xh))
        # an activation that overflowed: its row's outputs and the weight's gradient are lost, everything else stands
        hot = x.clone()
        hot[-1, row, c] = NAN
        hy, hm, hr = ops.layernorm(hot, g, None)
        assert torch.equal(hy[other], y[other]) and bool(hy[-1, row].isnan().all()) and torch.equal(hm[other], mu[other])
        hx, hg, hb = ops.layernorm_backward(dy, hot, hm, hr, g)
        gx, gg, gb = ops.layernorm_backward(dy, x, mu, r, g)
        assert torch.equal(hx[other], gx[other]) and torch.equal(hb, gb)
        assert bool(hg.view(-1, D)[-1].isnan().all()) and torch.equal(hg.view(-1, D)[:-1], gg.view(-1, D)[:-1])


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("per", [False, True])
@pytest.mark.parametrize("T,D", [(2100, 640), (2048, 1024), (2049, 1032), (2300, 1536), (2050, 2056), (2048, 2560), (2047, 640), (2047, 2560)])
def test_layernorm_of_many_rows_at_every_chunk_count(dev, T, D, per, dt):
    """From 2048 rows on, 16-bit rows of whole chunks have two or three chunks a lane in the forward pass and in dx alone."""
    from flux_generator_amd import ops
    B, off = (2, 1.0) if per else (1, 0.0)
    T //= B
    x, dy = rnd(B, T, D, mean=0.5, seed=1, dt=dt), rnd(B, T, D, seed=2, dt=dt)
    shape = (B, D) if per else (D,)
    g, b = rnd(*shape, scale=0.3, mean=1 - off, seed=3, dt=dt), rnd(*shape, scale=0.3, seed=4, dt=dt)
    c = lambda t: t.to(dev)
    y, mu, r = ops.layernorm(c(x), c(g), c(b), unit_offset=per)
    gd, bd = D64(g).reshape(-1, 1, D), D64(b).reshape(-1, 1, D)
    for what, got, pair in zip(("y", "mean", "rstd"), (y, mu, r), R.ln_forward_bound(D64(x), gd, bd, 1e-5, off, dt)):
        R.check(got, pair, what)
    pairs = R.ln_backward_bound(D64(dy), D64(x), D64(mu), D64(r), gd, off, dt, dt, per)
    for what, got, pair in zip(("dx", "dgamma", "dbeta"), ops.layernorm_backward(c(dy), c(x), mu, r, c(g), unit_offset=per), pairs):
        R.check(got, pair, what)
    R.check(ops.layernorm_backward(c(dy), c(x), mu, r, c(g), unit_offset=per, param_grads=False)[0], pairs[0], "dx alone")
    R.check(ops.layernorm_backward(c(dy), c(x), mu, r)[0], R.ln_backward_bound(D64(dy), D64(x), D64(mu), D64(r), torch.ones(1, 1, D).double(), 0.0, dt, dt, False)[0],
            "dx without parameters")


# ------------------------------------------------------------------------------------------------ gated feed-forward
@pytest.mark.parametrize("kind,name", [("erf", "EPI_GELU_ERF"), ("tanh", "EPI_GELU_TANH"), ("silu", "EPI_SILU")])
@pytest.mark.parametrize("dt", [BF, HF])
def test_gated_ff_gradient_over_the_whole_range_of_gates(dev, kind, name, dt):
    """One token whose gates run over everything finite: the derivative is 0 or 1 far out, never NaN."""
    from flux_generator_amd import ops
    big = [1e-30, 1e-6, 0.3, 2.0, 5.5, 12.0, 40.0, 90.0, 1e3, 6e4] + ([1e9, 1e12, 1e18, 1.8e19, 1.9e19, 1e20, 1e30, 3.3e38] if dt == BF else [])
    gate = torch.tensor([s * b for b in big for s in (1, -1)] + [0.0] * (40 - 2 * len(big)), dtype=dt)[None]
    F, D = gate.shape[1], 64
    x, dy, value = rnd(1, D, seed=1, dt=dt), rnd(1, D, seed=2, dt=dt), rnd(1, F, seed=3, dt=dt)
    wv, wg, wo = rnd(F, D, scale=1e-3, seed=4, dt=dt), rnd(F, D, scale=D ** -0.5, seed=5, dt=dt), rnd(D, F, scale=1e-3, seed=6, dt=dt)
    hidden = torch.zeros(1, F, dtype=dt)
    c = lambda t: t.to(dev)
    out = ops.gated_ff_backward(c(dy), c(x), (c(value), c(gate), c(hidden)), c(wv), c(wg), c(wo), act=getattr(ops, name), bias_grads=True)
    pairs = R.ff_backward_bound(D64(dy), D64(x), D64(value), D64(gate), D64(hidden), D64(wv), D64(wg), D64(wo), kind, dt)
    for what, got, pair in zip(("dx", "dw_value", "dw_gate", "dw_out", "db_value", "db_gate", "db_out"), out, pairs):
        assert bool(got.isfinite().all()), (what, gate[0, got.isfinite().logical_not().nonzero()[0, 0]])
        R.check(got, pair, what)


@pytest.mark.parametrize("M,D,F", [(2, 64, 136), (5, 72, 40), (130, 128, 384), (1000, 1280, 2568), (2947, 952, 2728)])
def test_gated_ff_keeps_rows_apart(dev, M, D, F):
    """A token that is NaN, and one whose gradient is infinite, leave every other token's results as they are."""
    from flux_generator_amd import ops
    x, dy = rnd(M, D, seed=1).to(dev), rnd(M, D, seed=2).to(dev)
    W = [t.to(dev) for t in (rnd(F, D, scale=D ** -0.5, seed=3), rnd(F, D, scale=D ** -0.5, seed=4), rnd(D, F, scale=F ** -0.5, seed=5))]
    y, s = ops.gated_ff(x, *W, save=True)
    dx = ops.gated_ff_backward(dy, x, s, *W)[0]
    for row in {0, M // 2, M - 1}:
        other = torch.arange(M, device=dev) != row
        hot = x.clone()
        hot[row, D // 2] = NAN
        hy, hs = ops.gated_ff(hot, *W, save=True)
        assert bool(hy[row].isnan().all()) and torch.equal(hy[other], y[other])
        assert all(torch.equal(p[other], q[other]) and bool(p[row].isnan().all()) for p, q in zip(hs, s))
        bad = dy.clone()
        bad[row, D // 2] = INF
        bx = ops.gated_ff_backward(bad, x, s, *W)[0]
        assert torch.equal(bx[other], dx[other]) and not bool(bx[row].isfinite().any())


# ------------------------------------------------------------------------------------------------ rotary
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("inter", [True, False])
def test_rotary_keeps_pairs_apart(dev, inter, dt):
    from flux_generator_amd import ops
    B, T, H, K, hd, rot = 2, 37, 5, 2, 84, 44
    q, k = rnd(B, T, H, hd, seed=1, dt=dt).to(dev), rnd(B, T, K, hd, seed=2, dt=dt).to(dev)
    freqs, _ = ops.rotary_frequencies(rot, device=dev)
    pos = torch.arange(T, device=dev)
    want = ops.rotary(q, k, pos, freqs, interleaved=inter)
    for col in (0, 1, 9, 21, 22, 43, 44, 83):
        mate = col if col >= rot else col ^ 1 if inter else (col + rot // 2) % rot
        bad = q.clone()
        bad[1, 5, 3, col] = NAN
        got = ops.rotary(bad, k, pos, freqs, interleaved=inter)
        assert torch.equal(got[1], want[1]) and bool(got[0][1, 5, 3, [col, mate]].isnan().all())
        keep = torch.ones_like(q, dtype=torch.bool)
        keep[1, 5, 3, [col, mate]] = False
        assert torch.equal(got[0][keep], want[0][keep]), col


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("rot,hd", [(30, 48), (44, 48), (26, 84), (1030, 1031), (2054, 2060)])
def test_rotary_in_place_over_many_tokens(dev, rot, hd, inter, dt):
    """Widths whose last vector is moved back, with more (token, head) items than a block takes at once."""
    from flux_generator_amd import ops
    B, T, H, K = (2, 5000, 24, 8) if hd < 100 else (2, 60, 24, 8)
    qkv = rnd(B, T, (H + 2 * K) * hd, seed=1, dt=dt).to(dev)
    q, k = qkv[..., : H * hd].unflatten(-1, (H, hd)), qkv[..., H * hd: (H + K) * hd].unflatten(-1, (K, hd))
    values = qkv[..., (H + K) * hd:].clone()
    freqs, _ = ops.rotary_frequencies(rot, device=dev)
    pos = torch.arange(T, device=dev) + 5
    want = ops.rotary(q, k, pos, freqs, interleaved=inter)
    a, b = ops.rotary(q, k, pos, freqs, interleaved=inter, out=(q, k))
    assert a is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[..., (H + K) * hd:], values)

"""LayerNorm, gated feed-forward and rotary positions, forward and backward, against float64 with per-element bounds
(train_refs.py)."""
import math

import pytest
import torch

import train_refs as R

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rnd(*shape, scale=1.0, mean=0.0, seed=0, dt=BF):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dt)


def D64(t):
    return None if t is None else t.detach().cpu().double()


# ------------------------------------------------------------------------------------------------ LayerNorm
LN_SHAPES = [(1, 1, 1), (1, 1, 8), (2, 3, 7), (1, 5, 64), (2, 700, 19), (1, 3000, 128), (5, 33, 72), (3, 77, 771), (1, 2050, 513), (2, 9, 1280), (1, 2300, 1280), (1, 2049, 1999),
             (1, 6, 2560), (3, 170, 320), (2, 300, 72), (1, 513, 136), (1, 3, 4097), (2, 2, 8192), (1, 3, 8193), (1, 70, 9001)]


@pytest.mark.parametrize("dt,kind", [(dt, k) for dt in (BF, HF, F32) for k in ("shared", "sample", "none", "f32") if (dt, k) != (F32, "f32")])
@pytest.mark.parametrize("B,T,D", LN_SHAPES)
def test_layernorm_forward_backward(dev, B, T, D, kind, dt):
    from flux_generator_amd import ops
    x, dy = rnd(B, T, D, mean=0.5, seed=1, dt=dt), rnd(B, T, D, seed=2, dt=dt)
    pdt, per = (F32 if kind == "f32" else dt), kind == "sample"
    off = 1.0 if per else 0.0
    shape = (B, D) if per else (D,)
    g = b = None
    if kind != "none":
        g, b = rnd(*shape, scale=0.3, mean=1 - off, seed=3, dt=pdt), rnd(*shape, scale=0.3, seed=4, dt=pdt)
    cu = lambda t: None if t is None else t.to(dev)
    y, mu, r = ops.layernorm(cu(x), cu(g), cu(b), eps=1e-5, unit_offset=per)
    gd = torch.ones(1, 1, D).double() if g is None else D64(g).reshape(-1, 1, D)
    bd = torch.zeros(1, 1, D).double() if b is None else D64(b).reshape(-1, 1, D)
    py, pmu, pr = R.ln_forward_bound(D64(x), gd, bd, 1e-5, off, dt)
    R.check(mu, pmu, "mean"); R.check(r, pr, "rstd"); R.check(y, py, "y")
    dx, dg, db = ops.layernorm_backward(cu(dy), cu(x), mu, r, cu(g), unit_offset=per)
    px, pg, pb = R.ln_backward_bound(D64(dy), D64(x), D64(mu), D64(r), gd, off, dt, pdt, per)
    R.check(dx, px, "dx")
    if g is None:
        assert dg is None and db is None
    else:
        R.check(dg, pg, "dgamma"); R.check(db, pb, "dbeta")
        dx2, n1, n2 = ops.layernorm_backward(cu(dy), cu(x), mu, r, cu(g), unit_offset=per, param_grads=False)
        assert n1 is None and n2 is None
        R.check(dx2, px, "dx of a frozen norm")


def test_layernorm_strided_and_repeatable(dev):
    """Slices of packed buffers (samples apart, rows apart, a single column), mixed layouts of x and dy, and the same bits twice."""
    from flux_generator_amd import ops
    B, T, D = 3, 37, 640
    buf, dbuf = (torch.full(s, float("nan"), dtype=BF, device=dev) for s in ((B, T + 11, D + 24), (B, T + 3, D)))
    x, dy = buf[:, 11:, 8:8 + D], dbuf[:, :T]
    x.copy_(rnd(B, T, D, seed=5)); dy.copy_(rnd(B, T, D, seed=6))
    for g in (rnd(D, mean=1, seed=7).to(dev), rnd(B, D, seed=8).to(dev)):
        b = torch.zeros_like(g)
        y, mu, r = ops.layernorm(x, g, b)
        yc, muc, rc = ops.layernorm(x.contiguous(), g, b)
        assert torch.equal(y, yc) and torch.equal(mu, muc) and torch.equal(r, rc)
        ref = ops.layernorm_backward(dy.contiguous(), x.contiguous(), mu, r, g)
        for xx, dd in ((x, dy), (x, dy.contiguous()), (x.contiguous(), dy)):
            got = ops.layernorm_backward(dd, xx, mu, r, g)
            assert torch.equal(got[0], ref[0])
            for a, c in zip(got[1:], ref[1:]):                 # (the partial sums may be cut differently)
                assert torch.allclose(a.float(), c.float(), rtol=2 * R.u(BF) * 2, atol=1e-3)
        again = ops.layernorm_backward(dy, x, mu, r, g)
        assert all(torch.equal(p, q) for p, q in zip(again, ops.layernorm_backward(dy, x, mu, r, g)))
    for xx in (x[0], x[0, 0], x[:, :0], x[:0]):
        y, mu, r = ops.layernorm(xx, rnd(D, seed=9).to(dev), None)
        assert y.shape == xx.shape and mu.shape == xx.shape[:-1]
        dx, dg, db = ops.layernorm_backward(y, xx, mu, r, rnd(D, seed=9).to(dev))
        assert dx.shape == xx.shape and (xx.numel() or (float(dg.abs().max()) == 0 and float(db.abs().max()) == 0))
    wide = rnd(2, 4, 1, seed=1).to(dev).expand(2, 4, 1)
    assert torch.equal(ops.layernorm(wide)[0], torch.zeros_like(wide))


def test_layernorm_gradient_against_differences(dev):
    from flux_generator_amd import ops
    B, T, D = 2, 5, 96
    x, dy, g, b = (rnd(*s, seed=i, dt=F32) for i, s in enumerate(((B, T, D), (B, T, D), (D,), (D,))))
    y, mu, r = ops.layernorm(x.to(dev), g.to(dev), b.to(dev))
    dx, dg, db = ops.layernorm_backward(dy.to(dev), x.to(dev), mu, r, g.to(dev))
    px, pg, pb = R.ln_backward_bound(D64(dy), D64(x), D64(mu), D64(r), D64(g).reshape(1, 1, D), 0.0, F32, F32, False)
    loss = lambda X, G, Bt: (R.ln_forward(X, G, Bt, 1e-5, 0.0)[0] * D64(dy)).sum()
    X, G, Bt, h = D64(x), D64(g).reshape(1, 1, D), D64(b).reshape(1, 1, D), 1e-4
    for k, (got, pair) in enumerate(((dx, px), (dg, pg), (db, pb))):
        v = torch.randn(pair[0].shape, generator=torch.Generator().manual_seed(7 + k), dtype=torch.float64)
        w = [X, G, Bt]
        lo, hi = list(w), list(w)
        lo[k], hi[k] = w[k] - h * v.reshape(w[k].shape), w[k] + h * v.reshape(w[k].shape)
        diff = (loss(*hi) - loss(*lo)) / (2 * h)
        # the statistics are float32 (2^-23 relative on every term) and the difference is cut off at h^2 times third derivatives
        room = float((pair[1] * v.abs()).sum()) + 1e-5 * float((pair[0].abs() * v.abs()).sum() + dy.abs().sum())
        assert abs(float((D64(got) * v).sum() - diff)) <= room


# ------------------------------------------------------------------------------------------------ gated feed-forward
ACTS = {"erf": "EPI_GELU_ERF", "tanh": "EPI_GELU_TANH", "silu": "EPI_SILU"}
FF_SHAPES = [(1, 8, 8), (1, 64, 128), (1, 1288, 5128), (2, 128, 64), (3, 520, 24), (4, 2056, 264), (5, 1032, 40), (7, 72, 200), (16, 320, 136), (17, 64, 264), (33, 640, 128), (65, 136, 72),
             (130, 128, 384), (257, 264, 520), (300, 72, 1032)]


def ff_case(M, D, F, dt, bias, seed=0):
    t = dict(x=rnd(M, D, seed=seed + 1, dt=dt), wv=rnd(F, D, scale=D ** -0.5, seed=seed + 2, dt=dt), wg=rnd(F, D, scale=D ** -0.5, seed=seed + 3, dt=dt),
             wo=rnd(D, F, scale=F ** -0.5, seed=seed + 4, dt=dt), dy=rnd(M, D, seed=seed + 5, dt=dt))
    b = [rnd(n, scale=0.3, seed=seed + 6 + i, dt=dt) if bias else None for i, n in enumerate((F, F, D))]
    return t, b


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kind", list(ACTS))
@pytest.mark.parametrize("M,D,F", FF_SHAPES)
def test_gated_ff_forward_backward(dev, M, D, F, kind, dt):
    from flux_generator_amd import ops
    act = getattr(ops, ACTS[kind])
    bias = (M + D // 8) % 2 == 0
    t, b = ff_case(M, D, F, dt, bias)
    c = {k: v.to(dev) for k, v in t.items()}
    cb = [None if v is None else v.to(dev) for v in b]
    y, (v, a, h) = ops.gated_ff(c["x"], c["wv"], c["wg"], c["wo"], *cb, act=act, save=True)
    assert torch.equal(y, ops.gated_ff(c["x"], c["wv"], c["wg"], c["wo"], *cb, act=act))
    py, pv, pa, ph = R.ff_forward_bound(*(D64(t[k]) for k in ("x", "wv", "wg", "wo")), *(D64(q) for q in b), kind, dt)
    R.check(v, pv, "value"); R.check(a, pa, "gate"); R.check(h, ph, "hidden"); R.check(y, py, "y")
    out = ops.gated_ff_backward(c["dy"], c["x"], (v, a, h), c["wv"], c["wg"], c["wo"], act=act, bias_grads=True)
    pairs = R.ff_backward_bound(D64(t["dy"]), D64(t["x"]), D64(v), D64(a), D64(h), D64(t["wv"]), D64(t["wg"]), D64(t["wo"]), kind, dt)
    for name, got, pair in zip(("dx", "dw_value", "dw_gate", "dw_out", "db_value", "db_gate", "db_out"), out, pairs):
        R.check(got, pair, name)
    frozen = ops.gated_ff_backward(c["dy"], c["x"], (v, a, h), c["wv"], c["wg"], c["wo"], act=act, weight_grads=False)
    assert torch.equal(frozen[0], out[0]) and all(q is None for q in frozen[1:])
    lean = ops.gated_ff_backward(c["dy"], c["x"], (v, a, None), c["wv"], c["wg"], c["wo"], act=act, weight_grads=False, bias_grads=True)
    assert torch.equal(lean[0], out[0]) and all(torch.equal(p, q) for p, q in zip(lean[4:], out[4:]))
    own = ops.gated_ff_backward(c["dy"], c["x"], (v, a, h), c["wv"], c["wg"], c["wo"], act=act, input_grad=False)
    assert own[0] is None and all(torch.equal(p, q) for p, q in zip(own[1:4], out[1:4])) and own[4] is None


@pytest.mark.parametrize("M,D,F", [(1000, 1280, 2568), (2500, 648, 4096), (3, 4096, 10240), (513, 2048, 5128), (1300, 2048, 3080), (700, 2504, 5000)])
def test_gated_ff_larger(dev, M, D, F):
    """The large tiles, split products and many k-steps, against a float64 evaluation on the device."""
    from flux_generator_amd import ops
    t, b = ff_case(M, D, F, BF, True, seed=20)
    c = {k: v.to(dev) for k, v in t.items()}
    cb = [v.to(dev) for v in b]
    y, (v, a, h) = ops.gated_ff(c["x"], c["wv"], c["wg"], c["wo"], *cb, act=ops.EPI_GELU_TANH, save=True)
    d = lambda q: q.double()
    with torch.no_grad():
        for got, pair in zip((y, v, a, h), R_on(dev, R.ff_forward_bound, *(d(c[k]) for k in ("x", "wv", "wg", "wo")), *(d(q) for q in cb), "tanh", BF)):
            R.check(got, pair)
        out = ops.gated_ff_backward(c["dy"], c["x"], (v, a, h), c["wv"], c["wg"], c["wo"], act=ops.EPI_GELU_TANH, bias_grads=True)
        for got, pair in zip(out, R_on(dev, R.ff_backward_bound, d(c["dy"]), d(c["x"]), d(v), d(a), d(h), d(c["wv"]), d(c["wg"]), d(c["wo"]), "tanh", BF)):
            R.check(got, pair)


def R_on(dev, fn, *args):
    return [(p[0].cpu(), p[1].cpu()) for p in fn(*args)]


def test_gated_ff_strided_empty_and_repeatable(dev):
    from flux_generator_amd import ops
    M, D, F = 70, 64, 136
    t, b = ff_case(M, D, F, BF, True)
    c = {k: v.to(dev) for k, v in t.items()}
    nan = float("nan")                                    # what lies around the operands is not looked at
    buf, dbuf = torch.full((M + 9, D + 40), nan, dtype=BF, device=dev), torch.full((M + 9, D + 8), nan, dtype=BF, device=dev)
    buf[2:2 + M, 16:16 + D], dbuf[3:3 + M, :D] = c["x"], c["dy"]
    x, dy = buf[2:2 + M, 16:16 + D], dbuf[3:3 + M, :D]
    W = (c["wv"], c["wg"], c["wo"])
    y, s = ops.gated_ff(x, *W, save=True)
    y2, s2 = ops.gated_ff(c["x"], *W, save=True)
    assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(s, s2))
    a1, a2 = ops.gated_ff_backward(dy, x, s, *W, bias_grads=True), ops.gated_ff_backward(c["dy"], c["x"], s, *W, bias_grads=True)
    assert all(torch.equal(p, q) for p, q in zip(a1, a2))
    y3 = ops.gated_ff(c["x"].view(2, 5, 7, D), *W)
    assert torch.equal(y3.view(M, D), y) and y3.shape == (2, 5, 7, D)
    y0, s0 = ops.gated_ff(c["x"][:0], *W, save=True)
    g0 = ops.gated_ff_backward(c["dy"][:0], c["x"][:0], s0, *W, bias_grads=True)
    assert y0.shape == (0, D) and g0[0].shape == (0, D) and all(float(q.abs().max()) == 0 for q in g0[1:])


def test_gated_ff_gradient_against_differences(dev):
    from flux_generator_amd import ops
    M, D, F = 9, 72, 136
    for kind, name in ACTS.items():
        t, b = ff_case(M, D, F, HF, True)
        c = {k: v.to(dev) for k, v in t.items()}
        y, s = ops.gated_ff(c["x"], c["wv"], c["wg"], c["wo"], *(q.to(dev) for q in b), act=getattr(ops, name), save=True)
        out = ops.gated_ff_backward(c["dy"], c["x"], s, c["wv"], c["wg"], c["wo"], act=getattr(ops, name), bias_grads=True)
        pairs = R.ff_backward_bound(D64(t["dy"]), D64(t["x"]), *(D64(q) for q in s), D64(t["wv"]), D64(t["wg"]), D64(t["wo"]), kind, HF)
        W = [D64(t["x"]), D64(t["wv"]), D64(t["wg"]), D64(t["wo"]), *(D64(q) for q in b)]
        loss = lambda w: (R.ff_forward(*w, kind) * D64(t["dy"])).sum()
        for k, (got, pair) in enumerate(zip(out, pairs)):
            v, h = torch.randn(W[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64), 1e-4
            lo, hi = list(W), list(W)
            lo[k], hi[k] = W[k] - h * v, W[k] + h * v
            diff = (loss(hi) - loss(lo)) / (2 * h)
            # value, gate and hidden are float16: every product of the gradient is off by up to four half-steps more than the
            # bound from the saved values says (value, gate twice, hidden), each at most u of its terms' absolute sum
            # (act'' and act' are below 1.2), which the sums of |dy| |Wo| |.. | below collect
            dh = D64(t["dy"]).abs() @ D64(t["wo"]).abs()
            va, ga = D64(s[0]).abs(), D64(s[1]).abs()
            ev, ea = dh * 1.2 * ga, dh * (1.2 * va + 1.2 * va * ga)
            ax, av, aw = D64(t["x"]).abs(), D64(t["wv"]).abs(), D64(t["wg"]).abs()
            extra = [ev @ av + ea @ aw, ev.t() @ ax, ea.t() @ ax, D64(t["dy"]).abs().t() @ (va * ga + va), ev.sum(0), ea.sum(0), torch.zeros(D).double()][k]
            room = float(((pair[1] + 4 * R.u(HF) * extra) * v.abs()).sum()) + 1e-6 * float(D64(t["dy"]).abs().sum())
            assert abs(float((D64(got) * v).sum() - diff)) <= room, (kind, k)


# ------------------------------------------------------------------------------------------------ rotary
@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("B,T,H,K,hd,dims,far", [(1, 1, 1, 1, 2, [2], 0), (2, 3, 5, 1, 128, [128], 3_000_017), (1, 9, 24, 24, 128, [16, 56, 56], 0),
                                                 (2, 17, 10, 2, 84, [40], 900_001), (1, 5, 3, 3, 85, [42], 12), (3, 1, 32, 8, 64, [64], 2 ** 31 + 5),
                                                 (1, 1300, 2, 1, 96, [6, 10, 2, 4], 77), (3, 40, 4, 4, 142, [142], 7), (2, 7, 3, 1, 38, [10], 0), (1, 30, 2, 2, 51, [30], 9), (2, 11, 3, 3, 48, [12, 16, 16], 5), (1, 9, 2, 1, 70, [4, 2], 3),
                                                 (1, 2, 1, 2, 1030, [1030], 5), (8, 1, 24, 8, 128, [128], 9)]
                         + [(1, 5, 3, 1, 2 * n + 3, [2 * n], 1) for n in range(9, 16)])
def test_rotary_forward_backward(dev, B, T, H, K, hd, dims, far, inter, dt):
    from flux_generator_amd import ops
    q, k = rnd(B, T, H, hd, seed=1, dt=dt), rnd(B, T, K, hd, seed=2, dt=dt)
    freqs, _ = ops.rotary_frequencies(dims, device="cpu")
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 5000, (B, T, len(dims)), generator=g) + far
    p = (pos[..., 0] if len(dims) == 1 else pos).contiguous().to(dev)
    for back in (False, True):
        fn = ops.rotary_backward if back else ops.rotary
        gq, gk = fn(q.to(dev), k.to(dev), p, freqs.to(dev), axes_dim=dims, interleaved=inter, scale=1.2)
        R.check(gq, R.rotary_bound(D64(q), pos, freqs, dims, inter, 1.2, back, dt), "q")
        R.check(gk, R.rotary_bound(D64(k), pos, freqs, dims, inter, 1.2, back, dt), "k")
    if far < 2 ** 31 - 5000:
        i32 = ops.rotary(q.to(dev), None, p.int(), freqs.to(dev), axes_dim=dims, interleaved=inter)
        assert torch.equal(i32, ops.rotary(q.to(dev), None, p, freqs.to(dev), axes_dim=dims, interleaved=inter))


def test_rotary_layouts(dev):
    """Fused projections, transposed heads, shared positions, writing in place and into views: all the bits of the plain call."""
    from flux_generator_amd import ops
    B, T, H, K, hd = 2, 33, 6, 2, 48
    qkv = rnd(B, T, (H + 2 * K) * hd, seed=1).to(dev)
    q, k = qkv[..., : H * hd].unflatten(-1, (H, hd)), qkv[..., H * hd: (H + K) * hd].unflatten(-1, (K, hd))
    freqs, _ = ops.rotary_frequencies(32, device=dev)
    pos = torch.arange(T, device=dev) + 11
    rq, rk = ops.rotary(q.contiguous(), k.contiguous(), pos[None].repeat(B, 1), freqs, interleaved=False)
    for p in (pos, pos[None].expand(B, T), pos.int()):
        a, b = ops.rotary(q, k, p, freqs, interleaved=False)
        assert torch.equal(a, rq) and torch.equal(b, rk)
    qt, kt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k))
    oq = torch.empty(B, H, T, hd, dtype=BF, device=dev).transpose(1, 2)
    a, b = ops.rotary(qt, kt, pos, freqs, interleaved=False, out=(oq, kt))
    assert a is oq and torch.equal(a, rq) and torch.equal(kt, rk)
    values = qkv[..., (H + K) * hd:].clone()
    ops.rotary(q, k, pos, freqs, interleaved=False, out=(q, k))
    assert torch.equal(q, rq) and torch.equal(k, rk) and torch.equal(qkv[..., (H + K) * hd:], values)
    for rot, inter in ((30, True), (30, False), (26, False), (44, False), (10, True)):
        f, _ = ops.rotary_frequencies(rot, device=dev)
        a, b = (rnd(B, T, n, hd, seed=n).to(dev) for n in (H, K))
        want = ops.rotary(a, b, pos, f, interleaved=inter)
        ops.rotary(a, b, pos, f, interleaved=inter, out=(a, b))
        assert torch.equal(a, want[0]) and torch.equal(b, want[1]), (rot, inter)
    e = ops.rotary(q[:, :0], k[:, :0], pos[:0], freqs)
    assert e[0].shape == (B, 0, H, hd) and e[1].shape == (B, 0, K, hd)


@pytest.mark.parametrize("M,D,F", [(1, 40, 72), (3, 72, 40), (130, 136, 200), (517, 648, 1288), (1000, 1280, 2568), (2500, 120, 2056)])
def test_gated_ff_writes_nothing_else(dev, M, D, F):
    """Every output and the workspace between guard words, which stay; the values are those of the public calls."""
    from flux_generator_amd import ops
    from flux_generator_amd._lib import GatedFfDesc, GatedFfGradDesc, load
    lib = load()
    t, b = ff_case(M, D, F, BF, True, seed=40)
    c, cb = {k: v.to(dev) for k, v in t.items()}, [v.to(dev) for v in b]
    st = torch.cuda.current_stream().cuda_stream
    ptr = lambda *ts: [q.data_ptr() for q in ts]

    def guarded(*bytes_):
        offs, n = [], 4096
        for k in bytes_:
            offs.append(n)
            n = -(-(n + k) // 256) * 256 + 4096
        return torch.full((n,), 0xA5, dtype=torch.uint8, device=dev), offs

    def look(buf, offs, want, ws):
        keep = torch.ones_like(buf, dtype=torch.bool)
        for o, w in zip(offs, want):
            k = w.numel() * 2
            assert torch.equal(buf[o:o + k].view(BF).view(w.shape), w)
            keep[o:o + k] = False
        keep[offs[-1]:offs[-1] + ws] = False
        assert bool((buf[keep] == 0xA5).all())

    y, sv = ops.gated_ff(c["x"], c["wv"], c["wg"], c["wo"], *cb, act=ops.EPI_SILU, save=True)
    ws = lib.fluxhip_gated_ff_ws(M, D, F)
    buf, offs = guarded(*[2 * M * F] * 3, 2 * M * D, ws)
    at = [buf.data_ptr() + o for o in offs]
    d = GatedFfDesc(*ptr(c["x"], c["wv"], c["wg"], c["wo"], *cb), *at[:4], M, D, D, F, ops.EPI_SILU, 0, at[4], ws)
    assert lib.fluxhip_gated_ff(d, st) == 0
    look(buf, offs, (*sv, y), ws)

    out = ops.gated_ff_backward(c["dy"], c["x"], sv, c["wv"], c["wg"], c["wo"], act=ops.EPI_SILU, bias_grads=True)
    ws = lib.fluxhip_gated_ff_grad_ws(M, D, F)
    buf, offs = guarded(*[2 * q.numel() for q in out], *[2 * M * F] * 2, ws)
    at = [buf.data_ptr() + o for o in offs]
    d = GatedFfGradDesc(*ptr(c["dy"], c["x"], *sv, c["wv"], c["wg"], c["wo"]), at[7], at[8], *at[:7], M, D, D, D, F, ops.EPI_SILU, 0, at[9], ws)
    assert lib.fluxhip_gated_ff_grad(d, st) == 0
    look(buf, offs, (*out, *(buf[o:o + 2 * M * F].view(BF) for o in offs[7:9])), ws)


def test_offsets_beyond_32_bits(dev):
    """Tensors of more than 2^32 bytes and 2^31 elements: the last rows are those of a call on them alone."""
    from flux_generator_amd import ops
    T, H, hd = 70_000, 256, 128                            # 2.3e9 elements
    q = torch.zeros(1, T, H, hd, dtype=BF, device=dev)
    q[:, -3:] = rnd(1, 3, H, hd, seed=1).to(dev)
    freqs, _ = ops.rotary_frequencies(hd, device=dev)
    pos = torch.arange(T, device=dev) + 2 ** 33
    assert torch.equal(ops.rotary(q, None, pos, freqs)[:, -3:], ops.rotary(q[:, -3:], None, pos[-3:], freqs))
    D = 4096
    x = q.view(-1, D)                                       # 560 000 rows
    g = rnd(D, mean=1.0, seed=2).to(dev)
    y, mu, r = ops.layernorm(x, g, g)
    tail = ops.layernorm(x[-192:].repeat(20, 1), g, g)      # (3840 rows: the same kernel)
    assert torch.equal(y[-192:], tail[0][-192:]) and torch.equal(mu[-192:], tail[1][-192:]) and torch.equal(r[-192:], tail[2][-192:])
    dx, dg, db = ops.layernorm_backward(y, x, mu, r, g)
    ex, eg, eb = ops.layernorm_backward(y[-192:].repeat(20, 1), x[-192:].repeat(20, 1), tail[1], tail[2], g)
    assert torch.equal(dx[-192:], ex[-192:])
    del q, x, y, dx, ex
    M, D, F = 300_000, 8, 8192                              # value, gate, hidden: 2.5e9 elements each
    t, b = ff_case(64, D, F, BF, True, seed=3)
    W = [t[k].to(dev) for k in ("wv", "wg", "wo")]
    x = torch.zeros(M, D, dtype=BF, device=dev)
    x[-64:] = t["x"].to(dev)
    y, s = ops.gated_ff(x, *W, *(q.to(dev) for q in b), save=True)
    y2, s2 = ops.gated_ff(t["x"].to(dev), *W, *(q.to(dev) for q in b), save=True)
    assert all(torch.equal(p[-64:], q) for p, q in zip(s, s2))
    # (y's product may be split differently along k: hidden is the same, the float32 sums of 8192 terms differ in order)
    room = 2 * F * R.E32 * (D64(s2[2]).abs() @ D64(t["wo"]).abs().t() + 1) + 2 * R.u(BF) * D64(y2).abs() * 1.01
    assert bool(((D64(y[-64:]) - D64(y2)).abs() <= room).all())
    dy = torch.zeros_like(x)
    dy[-64:] = t["dy"].to(dev)
    out = ops.gated_ff_backward(dy, x, s, *W, bias_grads=True)
    del s
    pairs = R.ff_backward_bound(D64(t["dy"]), D64(t["x"]), *(D64(q) for q in s2), *(D64(q) for q in (t["wv"], t["wg"], t["wo"])), "erf", BF)
    R.check(out[0][-64:], pairs[0], "dx")
    for name, got, (ref, bound) in zip(("dw_value", "dw_gate", "dw_out", "db_value", "db_gate", "db_out"), out[1:], pairs[1:]):
        R.check(got, (ref, bound), name)                    # (the other rows' dy is zero: they add zeros)


# ------------------------------------------------------------------------------------------------ together, as they are used
def test_transformer_block_step(dev):
    """norm -> gated feed-forward -> residual, and q / k rotation, chained forward and backward; captured into a graph that is
    replayed on new inputs between eager calls."""
    from flux_generator_amd import ops
    B, T, D, F, H = 2, 50, 128, 264, 2
    t, b = ff_case(B * T, D, F, BF, True, seed=40)
    c = {k: v.to(dev) for k, v in t.items()}
    cb = [v.to(dev) for v in b]
    gamma, beta = rnd(B, D, scale=0.3, seed=1).to(dev), rnd(B, D, scale=0.3, seed=2).to(dev)
    freqs, _ = ops.rotary_frequencies([16, 24, 24], device=dev)
    pos = torch.randint(0, 64, (B, T, 3), generator=torch.Generator().manual_seed(3)).to(dev)
    W = (c["wv"], c["wg"], c["wo"])

    def step(x, dz):
        n, mu, r = ops.layernorm(x, gamma, beta, unit_offset=True)
        y, saved = ops.gated_ff(n, *W, *cb, act=ops.EPI_GELU_TANH, save=True)
        z = ops.rotary((x + y).view(B, T, H, D // H), None, pos, freqs, axes_dim=[16, 24, 24])
        dy = ops.rotary_backward(dz.view(B, T, H, D // H), None, pos, freqs, axes_dim=[16, 24, 24]).view(B, T, D)
        grads = ops.gated_ff_backward(dy, n, saved, *W, act=ops.EPI_GELU_TANH, bias_grads=True)
        dx, dg, db = ops.layernorm_backward(grads[0], x, mu, r, gamma, unit_offset=True)
        return [z, dx + dy, dg, db, *grads[1:]]

    x, dz = rnd(B, T, D, seed=50).to(dev), rnd(B, T, D, seed=51).to(dev)
    got = step(x, dz)

    leaves = [D64(q).requires_grad_() for q in (x, gamma, beta, *W, *cb)]
    X, G, Bt, wv, wg, wo, bv, bg, bo = leaves
    n = R.ln_forward(X, G[:, None], Bt[:, None], 1e-5, 1.0)[0]
    y = ((n @ wv.t() + bv) * act64(n @ wg.t() + bg)) @ wo.t() + bo
    ang = D64(pos)[..., torch.tensor([0] * 8 + [1] * 12 + [2] * 12)] * D64(freqs)
    zz = (X + y).view(B, T, H, D // H)
    cs, sn = torch.cos(ang)[:, :, None], torch.sin(ang)[:, :, None]
    z = torch.stack([zz[..., 0::2] * cs - zz[..., 1::2] * sn, zz[..., 0::2] * sn + zz[..., 1::2] * cs], -1).flatten(-2)
    z.backward(D64(dz).view_as(z))
    want = [z.detach()] + [q.grad for q in (X, G, Bt, wv, wg, wo, bv, bg, bo)]
    for a, w in zip(got, want):
        # bf16 between the operators: n, value, gate, hidden, y, x + y, dy, dvalue / dgate, dx - at most nine roundings on a path,
        # each at most u = 2^-8 of its value; independent ones add in the 2-norm over many elements, 9 u bounds them added up
        assert float((D64(a) - w).norm() / w.norm()) <= 9 * R.u(BF)

    sx, sdz = x.clone(), dz.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sx, sdz)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(sx, sdz)
    for k in range(4):
        a, d = rnd(B, T, D, seed=60 + k).to(dev), rnd(B, T, D, seed=70 + k).to(dev)
        sx.copy_(a); sdz.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(a, d)
        assert all(torch.equal(p, q) for p, q in zip(held, eager)), k


def act64(z):
    return R.act(z, "tanh")[0]


def test_other_streams(dev):
    """Two streams at once, each with its own inputs: per-call scratch memory, so the results are those of one at a time."""
    from flux_generator_amd import ops
    cases = [ff_case(200, 256, 512, BF, True, seed=s) for s in (80, 90)]
    data = [({k: v.to(dev) for k, v in t.items()}, [q.to(dev) for q in b]) for t, b in cases]

    def run(c, b):
        y, s = ops.gated_ff(c["x"], c["wv"], c["wg"], c["wo"], *b, save=True)
        return [y, *ops.gated_ff_backward(c["dy"], c["x"], s, c["wv"], c["wg"], c["wo"], bias_grads=True)]

    want = [run(*d) for d in data]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(*data[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, w))

"""Float64 references of the adapter-training operators, each with a per-element bound on what the kernel may be off.

Bounds.  One rounding to a type is off by at most u = finfo(type).eps / 2 relative (and half the smallest subnormal).  A float32
sum of n products is off by at most (n + 2) 2^-24 times the sum of their absolute values, whatever the order.  Elementary float32
steps (rsqrt, exp, rcp: 1 ulp each) are counted in units of 2^-23.  Every bound below is a sum of such terms carried through the formula."""
import math

import torch

E32 = 2.0 ** -24


def u(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps       # one subnormal step: half of it, and one flushed float32 intermediate


def store(ref, err, dt):
    """(ref, bound) of a value known up to err once it is rounded to dt."""
    return ref, err + u(dt) * (ref.abs() + err) + tiny(dt)


def check(got, pair, what=""):
    ref, bound = pair
    g = got.detach().double().cpu()
    assert g.shape == ref.shape, (what, g.shape, ref.shape)
    off = (g - ref).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside their bound, worst {float((off / bound).nan_to_num(9e9).max()):.3g} x"


# ------------------------------------------------------------------------------------------------ LayerNorm
def ln_forward(x, g, b, eps, off):
    """x [B, T, D] double, g / b [B or 1, 1, D] double."""
    D = x.shape[-1]
    mu = x.mean(-1, keepdim=True)
    var = (x - mu).square().mean(-1, keepdim=True)
    r = (var + eps).rsqrt()
    return (x - mu) * r * (off + g) + b, mu[..., 0], r[..., 0]


def ln_forward_bound(x, g, b, eps, off, dt):
    D = x.shape[-1]
    y, mu, r = ln_forward(x, g, b, eps, off)
    n = D + 4
    e_mu = n * E32 * x.abs().mean(-1)
    c = (x - mu[..., None]).abs()
    e_c = e_mu[..., None] + E32 * (c + x.abs())
    # d(var)/var <= 2 e_c / c averaged ... : var off by mean(2 c e_c + e_c^2) + n E32 var
    var = c.square().mean(-1)
    e_var = (2 * c * e_c + e_c.square()).mean(-1) + (n + 2) * E32 * var
    e_r = r * (0.5 * e_var / (var + eps) + 6 * E32) * 1.01
    gg = (off + g).abs()
    e_y = gg * (e_c * r[..., None] + c * e_r[..., None]) + 6 * E32 * (gg * c * r[..., None] + b.abs())
    return store(y, e_y, dt), (mu, e_mu + E32 * mu.abs()), (r, e_r)


def ln_backward(dy, x, mu, r, g, off):
    mu, r = mu[..., None], r[..., None]
    xh = (x - mu) * r
    e = dy * (off + g)
    dx = r * (e - e.mean(-1, keepdim=True) - xh * (e * xh).mean(-1, keepdim=True))
    return dx, (dy * xh).sum(1), dy.sum(1)


def ln_backward_bound(dy, x, mu, r, g, off, dt, pdt, per):
    D, T = x.shape[-1], x.shape[1] * (1 if per else x.shape[0])
    dx, dg, db = ln_backward(dy, x, mu, r, g, off)
    mu_, r_ = mu[..., None], r[..., None]
    xh = (x - mu_) * r_
    e_xh = 3 * E32 * (xh.abs() + (x.abs() + mu_.abs()) * r_)
    e = (dy * (off + g)).abs()
    s1, s2 = e.mean(-1, keepdim=True), (e * xh.abs()).mean(-1, keepdim=True)
    e_s2 = (e * e_xh).mean(-1, keepdim=True) + (D + 6) * E32 * s2
    e_dx = r_ * (4 * E32 * e + (D + 6) * E32 * s1 + xh.abs() * (e_s2 + 2 * E32 * s2) + e_xh * s2 + 4 * E32 * (e + s1 + xh.abs() * s2))
    t_dg = (dy.abs() * xh.abs()).sum(1)
    e_dg = (dy.abs() * e_xh).sum(1) + (T + 4) * E32 * t_dg
    e_db = (T + 4) * E32 * dy.abs().sum(1)
    if not per:
        dg, db, e_dg, e_db = (t.sum(0) for t in (dg, db, e_dg, e_db))
    return store(dx, e_dx, dt), store(dg, e_dg, pdt), store(db, e_db, pdt)


# ------------------------------------------------------------------------------------------------ gated feed-forward
def act(z, kind):
    """(act(z), act'(z)) in double."""
    if kind == "erf":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


# the float32 activations: erfc of the rational form is off by 1.5e-7 absolute, the sigmoids by a few ulp of exp and rcp at
# arguments up to ~20 (20 * 2^-23 relative where the sigmoid is not saturated): below 3e-6 |z| and 6e-6 in the derivative
ACT, DACT = 3e-6, 6e-6


def ff_forward_bound(x, wv, wg, wo, bv, bg, bo, kind, dt):
    D, F = wv.shape[1], wv.shape[0]
    z = torch.zeros((), dtype=torch.float64)
    bv, bg, bo = (z if t is None else t for t in (bv, bg, bo))
    v, a = x @ wv.t() + bv, x @ wg.t() + bg
    e_v = (D + 4) * E32 * (x.abs() @ wv.abs().t() + bv.abs())
    e_a = (D + 4) * E32 * (x.abs() @ wg.abs().t() + bg.abs())
    f, _ = act(a, kind)
    h = v * f
    e_f = 1.2 * e_a + ACT * a.abs()                       # |act'| < 1.2 everywhere
    e_h = e_v * f.abs() + v.abs() * e_f + e_v * e_f + 2 * E32 * h.abs()
    y = h @ wo.t() + bo
    _, b_h = store(h, e_h, dt)
    e_y = b_h @ wo.abs().t() + (F + 4) * E32 * ((h.abs() + b_h) @ wo.abs().t() + bo.abs())
    return store(y, e_y, dt), store(v, e_v, dt), store(a, e_a, dt), (h, b_h)


def ff_forward(x, wv, wg, wo, bv, bg, bo, kind):
    z = torch.zeros((), dtype=torch.float64)
    bv, bg, bo = (z if t is None else t for t in (bv, bg, bo))
    return ((x @ wv.t() + bv) * act(x @ wg.t() + bg, kind)[0]) @ wo.t() + bo


def ff_backward_bound(dy, x, v, a, h, wv, wg, wo, kind, dt):
    """Pairs for dx, dwv, dwg, dwo, dbv, dbg, dbo (value, gate, hidden as saved)."""
    (M, D), F = x.shape, wv.shape[0]
    f, df = act(a, kind)
    dh = dy @ wo
    e_dh = (D + 4) * E32 * (dy.abs() @ wo.abs())
    dv, da = dh * f, dh * v * df
    e_dv = e_dh * f.abs() + (dh.abs() + e_dh) * ACT * a.abs() + 2 * E32 * dv.abs()
    e_da = (e_dh * df.abs() + (dh.abs() + e_dh) * DACT) * v.abs() + 4 * E32 * da.abs()
    _, b_dv = store(dv, e_dv, dt)
    _, b_da = store(da, e_da, dt)
    tv, ta = dv.abs() + b_dv, da.abs() + b_da
    out = [store(dv @ wv + da @ wg, b_dv @ wv.abs() + b_da @ wg.abs() + (2 * F + 8) * E32 * (tv @ wv.abs() + ta @ wg.abs()), dt)]
    ax = x.abs()
    out.append(store(dv.t() @ x, b_dv.t() @ ax + (M + 8) * E32 * (tv.t() @ ax), dt))
    out.append(store(da.t() @ x, b_da.t() @ ax + (M + 8) * E32 * (ta.t() @ ax), dt))
    out.append(store(dy.t() @ h, (M + 8) * E32 * (dy.abs().t() @ h.abs()), dt))
    out.append(store(dv.sum(0), e_dv.sum(0) + (M + 8) * E32 * dv.abs().sum(0), dt))
    out.append(store(da.sum(0), e_da.sum(0) + (M + 8) * E32 * da.abs().sum(0), dt))
    out.append(store(dy.sum(0), (M + 8) * E32 * dy.abs().sum(0), dt))
    return out


# ------------------------------------------------------------------------------------------------ rotary
def rotary_bound(x, pos, freqs, dims, interleaved, scale, inverse, dt):
    """x [B, T, H, hd] double, pos [B, T, axes] integers."""
    rot = 2 * freqs.shape[0]
    axis = torch.cat([torch.full((d // 2,), i) for i, d in enumerate(dims)]).long()
    ang = pos.double()[..., axis] * freqs
    if inverse:
        ang = -ang
    c, s = (scale * torch.cos(ang))[:, :, None], (scale * torch.sin(ang))[:, :, None]
    z = x[..., :rot]
    p, q = (z[..., 0::2], z[..., 1::2]) if interleaved else (z[..., : rot // 2], z[..., rot // 2:])
    a, b = p * c - q * s, p * s + q * c
    # cos / sin: the fraction of a turn carries 2^-53 |turns| of the double product and one float32 rounding (2 pi 2^-26 rad),
    # the function 2 ulp, times the scale: 8 units of 2^-24 and the far positions' share
    e = scale * (8 * E32 + 2 * math.pi * 2.0 ** -51 * (1 + ang.abs()))[:, :, None] * (p.abs() + q.abs()) + 3 * E32 * scale * (p.abs() + q.abs())
    join = (lambda m, n: torch.stack([m, n], -1).flatten(-2)) if interleaved else (lambda m, n: torch.cat([m, n], -1))
    ref, err = join(a, b), join(e, e)
    tail = x[..., rot:]
    ref, bound = store(ref, err, dt)
    return torch.cat([ref, tail], -1), torch.cat([bound, torch.zeros_like(tail)], -1)

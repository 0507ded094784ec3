"""Refusals of the adapter-training operators, the rotary frequencies, and the float64 references themselves (no GPU)."""
import math

import pytest
import torch

import train_refs as R

BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def z(*s, dt=BF):
    return torch.zeros(*s, dtype=dt)


def refuses(fn, *a, match=None, **k):
    from flux_generator_amd import ops
    with pytest.raises(ops.FluxHipError, match=match):
        fn(*a, **k)


def test_layernorm_refusals():
    from flux_generator_amd import ops
    x, g = z(2, 3, 8), z(8)
    refuses(ops.layernorm, x, g, g, match="device tensors")
    refuses(ops.layernorm, z(2, 8, dt=F64), match="bfloat16, float16 or float32")
    refuses(ops.layernorm, x, None, g, match="beta needs gamma")
    refuses(ops.layernorm, x, z(7), match="gamma must be")
    refuses(ops.layernorm, x, z(3, 8), match="gamma must be")
    refuses(ops.layernorm, x, z(8, dt=HF), match="x's type or float32")
    refuses(ops.layernorm, x, g, z(2, 8), match="one shape")
    refuses(ops.layernorm, x, g, z(8, dt=F32), match="one shape and one type")
    refuses(ops.layernorm, x.transpose(1, 2), match="contiguous last dimension")
    refuses(ops.layernorm, z(2, 3, 4, 8)[:, ::2, ::3], g, match="one stride")
    refuses(ops.layernorm, z(16)[::2], match="contiguous last dimension")
    m = z(2, 3, dt=F32)
    refuses(ops.layernorm_backward, z(2, 3, 8, dt=F32), x, m, m, g, match="dy must have")
    refuses(ops.layernorm_backward, z(2, 4, 8), x, m, m, g, match="dy must have")
    refuses(ops.layernorm_backward, x, x, z(2, 3), m, g, match="mean must be")
    refuses(ops.layernorm_backward, x, x, m, z(6, dt=F32), g, match="rstd must be")
    refuses(ops.layernorm_backward, x[:1, :1].expand(2, 3, 8)[..., :1].expand(2, 3, 8), x, m, m, g, match="contiguous last dimension")
    refuses(ops.layernorm_backward, x, x, m, m, g, match="device tensors")


def test_rotary_refusals():
    from flux_generator_amd import ops
    q, k, p, f = z(2, 3, 4, 8), z(2, 3, 2, 8), torch.arange(3), torch.ones(4, dtype=F64)
    refuses(ops.rotary, q, k, p, f, match="device tensors")
    refuses(ops.rotary, z(2, 3, 8), None, p, f, match="q must be")
    refuses(ops.rotary, z(2, 3, 4, 8, dt=F64), None, p, f, match="q must be")
    for bad in (z(2, 4, 2, 8), z(1, 3, 2, 8), z(2, 3, 2, 16), z(2, 3, 2, 8, dt=HF)):
        refuses(ops.rotary, q, bad, p, f, match="k must be")
    refuses(ops.rotary, q, k, p, f.float(), match="freqs must be")
    refuses(ops.rotary, q, k, p, torch.ones(5, dtype=F64), match="rot = ")
    refuses(ops.rotary, q, k, p, torch.ones(0, dtype=F64), match="rot = ")
    refuses(ops.rotary, q, k, p, f, axes_dim=[4, 2], match="rot = ")
    refuses(ops.rotary, q, k, p, f, axes_dim=[3, 5], match="rot = ")
    refuses(ops.rotary, q, k, p.float(), f, match="int32 or int64")
    refuses(ops.rotary, q, k, torch.arange(4), f, match="positions must be")
    refuses(ops.rotary, q, k, torch.zeros(3, 3, dtype=torch.int64), f, match="positions must be")
    refuses(ops.rotary, q, k, torch.zeros(2, 3, dtype=torch.int64), f, axes_dim=[4, 4], match="positions must be")
    refuses(ops.rotary, q, k, torch.zeros(2, 2, 3, dtype=torch.int64).transpose(1, 2), f, axes_dim=[4, 4], match="positions must be")
    refuses(ops.rotary, q.transpose(2, 3).contiguous().transpose(2, 3), k, p, f, match="contiguous last dimension")
    refuses(ops.rotary, q, k, p, f, out=q, match="out must give")
    refuses(ops.rotary, q, k, p, f, out=(q, z(2, 3, 4, 8)), match="out must have")
    refuses(ops.rotary, q, q, p, f, out=(q, q), match="memory of their own")
    refuses(ops.rotary, q, z(2, 3, 4, 8), p, f, out=(z(2, 3, 4, 8), q), match="memory of their own")
    refuses(ops.rotary, q, k, p, f, out=(z(1, 3, 4, 8).expand(2, 3, 4, 8), k), match="broadcast")
    refuses(ops.rotary_backward, q, k, p, f, match="device tensors")


def test_gated_ff_refusals():
    from flux_generator_amd import ops
    x, wv, wo = z(3, 16), z(24, 16), z(16, 24)
    refuses(ops.gated_ff, x, wv, wv, wo, match="device tensors")
    refuses(ops.gated_ff, z(3, 16, dt=F32), wv, wv, wo, match="bfloat16 or float16")
    refuses(ops.gated_ff, x, wv, wv, wo, act=ops.EPI_BIAS, match="act must be")
    refuses(ops.gated_ff, z(3, 12), z(24, 12), z(24, 12), z(12, 24), match="multiples of 8")
    refuses(ops.gated_ff, x, wv, z(16, 24), wo, match="w_gate must be")
    refuses(ops.gated_ff, x, wv, wv, wo.t().contiguous(), match="w_out must be")
    refuses(ops.gated_ff, x, z(24, 16, dt=HF), wv, wo, match="w_value must be")
    refuses(ops.gated_ff, x, z(16, 24).t(), wv, wo, match="w_value must be")
    refuses(ops.gated_ff, z(3, 24), wv, wv, wo, match="x must be")
    refuses(ops.gated_ff, z(3, 17)[:, :16], wv, wv, wo, match="16-byte aligned")
    refuses(ops.gated_ff, z(3, 32)[:, 1:17], wv, wv, wo, match="16-byte aligned")
    refuses(ops.gated_ff, z(1, 16).expand(3, 16), wv, wv, wo, match="overlap")
    refuses(ops.gated_ff, z(4, 5, 16)[:, :3], wv, wv, wo, match="one stride")
    refuses(ops.gated_ff, x, wv, wv, wo, z(24), match="go together")
    refuses(ops.gated_ff, x, wv, wv, wo, z(24), z(16), match="b_gate must be")
    refuses(ops.gated_ff, x, wv, wv, wo, None, None, z(24), match="b_out must be")
    s = (z(3, 24), z(3, 24), z(3, 24))
    refuses(ops.gated_ff_backward, z(2, 16), x, s, wv, wv, wo, match="dy must have")
    refuses(ops.gated_ff_backward, x, x, (z(3, 24), z(3, 16), z(3, 24)), wv, wv, wo, match="gate must be")
    refuses(ops.gated_ff_backward, x, x, (z(3, 24), z(3, 24), z(3, 24, dt=HF)), wv, wv, wo, match="hidden must be")
    refuses(ops.gated_ff_backward, x, x, None, wv, wv, wo, match="saved must be")
    refuses(ops.gated_ff_backward, x, x, (z(3, 24), z(3, 24), None), wv, wv, wo, match="hidden must be")
    refuses(ops.gated_ff_backward, x, x, (z(3, 24), z(3, 24), None), wv, wv, wo, weight_grads=False, match="device tensors")
    refuses(ops.gated_ff_backward, x, x, s, wv, wv, wo, match="device tensors")


def test_entry_points_refuse_bad_descriptors():
    """The C entry points return -1 for what the Python checks keep from them (host code only: nothing is launched)."""
    import ctypes
    from flux_generator_amd import _lib, ops
    lib = _lib.load()
    assert lib.fluxhip_layernorm_stats(1, 0, 8, None, None, 0, 0, 0.0, 1, 1, 1, 1, 1, 0, 1e-5, 0, None) == -1       # D = 0
    assert lib.fluxhip_layernorm_stats(None, 0, 8, None, None, 0, 0, 0.0, 1, 1, 1, 1, 1, 8, 1e-5, 0, None) == -1    # no x
    assert lib.fluxhip_layernorm_stats(16, 0, 8, None, None, 0, 0, 0.0, 16, 16, 16, 1, 1, 8, 1e-5, 3, None) == -1   # type
    assert lib.fluxhip_layernorm_stats(16, 0, 8, None, 16, 0, 0, 0.0, 16, 16, 16, 1, 1, 8, 1e-5, 0, None) == -1     # beta alone
    assert lib.fluxhip_layernorm_stats(None, 0, 8, None, None, 0, 0, 0.0, None, None, None, 0, 1, 8, 1e-5, 0, None) == 0
    assert lib.fluxhip_layernorm_grad(16, 0, 8, 16, 0, 8, 16, 16, 16, 0, 0, 0.0, 16, 16, 16, 1, 9000, 8, 0, None, 0, None) == -1   # no scratch
    assert lib.fluxhip_layernorm_grad(16, 0, 8, 16, 0, 8, 16, 16, 16, 0, 0, 0.0, 16, 16, None, 1, 100, 8, 0, 16, 1 << 20, None) == -1
    assert lib.fluxhip_layernorm_grad_ws(1, 100, 0) == -1 and lib.fluxhip_layernorm_grad_ws(1, 9000, 8) > 0 and lib.fluxhip_layernorm_grad_ws(1, 100, 8) == 0
    d = _lib.RotaryDesc()
    assert lib.fluxhip_rotary(None, None) == -1 and lib.fluxhip_rotary(ctypes.byref(d), None) == -1
    d.B, d.T, d.H, d.hd, d.rot, d.n_axes = 1, 1, 1, 8, 8, 1
    d.axis_pairs[0] = 3
    assert lib.fluxhip_rotary(ctypes.byref(d), None) == -1
    d.axis_pairs[0] = 4
    assert lib.fluxhip_rotary(ctypes.byref(d), None) == -1          # no tensors
    d.T = 0
    assert lib.fluxhip_rotary(ctypes.byref(d), None) == 0
    for cls, fn in ((_lib.GatedFfDesc, lib.fluxhip_gated_ff), (_lib.GatedFfGradDesc, lib.fluxhip_gated_ff_grad)):
        d = cls()
        assert fn(None, None) == -1 and fn(ctypes.byref(d), None) == -1
        d.M, d.D, d.F, d.act = 1, 16, 24, ops.EPI_SILU
        assert fn(ctypes.byref(d), None) == -1                      # no tensors
        d.M = 0
        assert fn(ctypes.byref(d), None) == 0
        d.D = 12
        assert fn(ctypes.byref(d), None) == -1
    assert lib.fluxhip_gated_ff_ws(4, 12, 16) == -1 and lib.fluxhip_gated_ff_grad_ws(4, 16, 16) > 0


def test_descriptor_layouts():
    import ctypes
    from flux_generator_amd import _lib
    assert ctypes.sizeof(_lib.RotaryDesc) == 232 and _lib.RotaryDesc.positions.offset == 128 and _lib.RotaryDesc.scale.offset == 228
    assert ctypes.sizeof(_lib.GatedFfDesc) == 136 and _lib.GatedFfDesc.M.offset == 88 and _lib.GatedFfDesc.ws.offset == 120
    assert ctypes.sizeof(_lib.GatedFfGradDesc) == 192 and _lib.GatedFfGradDesc.M.offset == 136 and _lib.GatedFfGradDesc.ws.offset == 176


def test_rotary_frequencies():
    from flux_generator_amd import ops
    f, s = ops.rotary_frequencies([16, 56, 56], theta=10000.0, device="cpu")
    want = torch.cat([torch.tensor([10000.0 ** (-2 * j / d) for j in range(d // 2)], dtype=F64) for d in (16, 56, 56)])
    assert s == 1.0 and torch.allclose(f, want, rtol=1e-14, atol=0)
    lin, s = ops.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    base, _ = ops.rotary_frequencies(64, device="cpu")
    assert s == 1.0 and torch.allclose(lin * 4, base, rtol=1e-14, atol=0)
    ntk, _ = ops.rotary_frequencies(64, scaling="ntk", factor=4.0, device="cpu")
    assert float(ntk[0]) == 1.0 and math.isclose(float(base[-1] / ntk[-1]), 4.0, rel_tol=1e-12)
    y, s = ops.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    turns = 4096 * base / (2 * math.pi)
    assert math.isclose(s, 0.1 * math.log(8) + 1)
    assert torch.equal(y[turns > 40], base[turns > 40]) and torch.allclose(y[turns < 0.5] * 8, base[turns < 0.5], rtol=1e-12, atol=0)
    assert bool((y <= base * (1 + 1e-12)).all()) and bool((y * 8 >= base * (1 - 1e-12)).all()) and bool((y[1:] < y[:-1]).all())
    assert ops.rotary_frequencies(2, scaling="ntk", factor=4.0, device="cpu")[0].tolist() == [1.0]
    for bad in (dict(dims=3), dict(dims=[]), dict(dims=0), dict(dims=8, scaling="cubic"), dict(dims=8, scaling="linear", factor=0.5),
                dict(dims=8, scaling="yarn", factor=2.0), dict(dims=8, scaling="yarn", factor=2.0, original_length=9, beta_fast=1.0)):
        refuses(ops.rotary_frequencies, device="cpu", **bad)


def test_references_against_autograd():
    """The float64 gradients the kernels are held to are those of the forward formulas."""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F64)
    x, ga, be, dy = r(2, 5, 12).requires_grad_(), r(1, 1, 12).requires_grad_(), r(1, 1, 12).requires_grad_(), r(2, 5, 12)
    y, mu, rs = R.ln_forward(x, ga, be, 1e-5, 1.0)
    y.backward(dy)
    dx, dg, db = R.ln_backward(dy, x.detach(), mu.detach(), rs.detach(), ga.detach(), 1.0)
    assert torch.allclose(dx, x.grad) and torch.allclose(dg.sum(0), ga.grad[0, 0]) and torch.allclose(db.sum(0), be.grad[0, 0])
    for kind in ("erf", "tanh", "silu"):
        t = [q.requires_grad_() for q in (r(6, 8), r(16, 8), r(16, 8), r(8, 16), r(16), r(16), r(8))]
        dy = r(6, 8)
        R.ff_forward(*t, kind).backward(dy)
        d = [q.detach() for q in t]
        v, a = d[0] @ d[1].t() + d[4], d[0] @ d[2].t() + d[5]
        pairs = R.ff_backward_bound(dy, d[0], v, a, v * R.act(a, kind)[0], d[1], d[2], d[3], kind, BF)
        for q, (ref, _) in zip(t, pairs):
            assert torch.allclose(ref, q.grad), kind

"""Adapter-training operators where they can go wrong at the ends of their ranges (no GPU)."""
import math

import pytest
import torch

F64 = torch.float64


def yarn_by_definition(d, theta, factor, length, fast, slow):
    """Pair by pair, in Python floats: the pair index at which a frequency turns n times over `length` positions is
    d ln(length / (2 pi n)) / (2 ln theta); the blend runs from the whole index below the one of `fast` (not before pair 0) to the
    whole index above the one of `slow` (not behind d - 1)."""
    at = lambda n: d * math.log(length / (2 * math.pi * n)) / (2 * math.log(theta))
    lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), d - 1)
    out = []
    for j in range(d // 2):
        f = theta ** (-2 * j / d)
        turns = length * f / (2 * math.pi)
        if turns < slow:
            share = 1.0
        elif j <= lo:
            share = 0.0
        else:
            share = min(1.0, (j - lo) / (hi - lo))
        out.append(f / factor * share + f * (1 - share))
    return torch.tensor(out, dtype=F64)


@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (8.0, 2.0)])
@pytest.mark.parametrize("theta", [10.0, 500.0, 1e4, 1e6])
@pytest.mark.parametrize("d", [2, 16, 56, 128])
@pytest.mark.parametrize("length", [1, 5, 6, 7, 100, 4096, 54_000, 65_536, 131_072, 262_144, 10 ** 7])
def test_yarn_at_every_length(length, d, theta, fast, slow):
    from flux_generator_amd import ops
    factor = 8.0
    f, s = ops.rotary_frequencies(d, theta=theta, scaling="yarn", factor=factor, original_length=length, beta_fast=fast, beta_slow=slow, device="cpu")
    base, _ = ops.rotary_frequencies(d, theta=theta, device="cpu")
    # a power, a logarithm and a few products in 64 bits: below 100 units of 2^-53
    assert torch.allclose(f, yarn_by_definition(d, theta, factor, length, fast, slow), rtol=100 * 2.0 ** -53, atol=0)
    turns = length * base / (2 * math.pi)
    assert torch.allclose(f[turns < slow * (1 - 1e-12)] * factor, base[turns < slow * (1 - 1e-12)], rtol=1e-14, atol=0)
    assert bool((f[turns > slow * (1 + 1e-12)] * factor > base[turns > slow * (1 + 1e-12)]).all())     # only slower pairs are divided whole


def test_yarn_long_original_context():
    """At 131072 positions the slowest of 64 pairs turns 2.4 times: it keeps 0.37 of its frequency at factor 8, not 1 / 8."""
    from flux_generator_amd import ops
    f, _ = ops.rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=131_072, device="cpu")
    base, _ = ops.rotary_frequencies(128, device="cpu")
    assert 0.36 < float(f[-1] / base[-1]) < 0.38


@pytest.mark.parametrize("bad", [dict(scaling="yarn", factor=2.0, original_length=100, theta=1.0), dict(scaling="yarn", factor=2.0, original_length=100, theta=0.5),
                                 dict(scaling="linear", factor=float("nan")), dict(scaling="ntk", factor=float("inf")), dict(theta=float("nan")),
                                 dict(theta=float("inf")), dict(scaling="yarn", factor=2.0, original_length=float("nan")),
                                 dict(scaling="yarn", factor=2.0, original_length=100, beta_fast=float("inf"))])
def test_frequency_refusals(bad):
    from flux_generator_amd import ops
    with pytest.raises(ops.FluxHipError):
        ops.rotary_frequencies(16, device="cpu", **bad)


def test_gated_ff_entry_points_refuse_misaligned_outputs():
    """Every tensor that the kernels move in 16-byte pieces must lie at 16 bytes: the outputs as well (host code only)."""
    import ctypes
    from flux_generator_amd import _lib, ops
    lib = _lib.load()
    M, D, F = 5, 16, 24
    n = lib.fluxhip_gated_ff_ws(M, D, F)
    for name in ("x", "w_value", "w_gate", "w_out", "value", "gate", "hidden", "y", "ws"):
        d = _lib.GatedFfDesc()
        for k in ("x", "w_value", "w_gate", "w_out", "value", "gate", "hidden", "y", "ws"):
            setattr(d, k, 4096 + (8 if k == name else 0))
        d.M, d.ldx, d.D, d.F, d.act, d.ws_bytes = M, D, D, F, ops.EPI_SILU, n
        assert lib.fluxhip_gated_ff(ctypes.byref(d), None) == -1, name
    n = lib.fluxhip_gated_ff_grad_ws(M, D, F)
    names = ("dy", "x", "value", "gate", "hidden", "w_value", "w_gate", "w_out", "dvalue", "dgate", "dx", "dw_value", "dw_gate", "dw_out", "ws")
    for name in names:
        d = _lib.GatedFfGradDesc()
        for k in names:
            setattr(d, k, 4096 + (8 if k == name else 0))
        d.M, d.ldx, d.lddy, d.D, d.F, d.act, d.ws_bytes = M, D, D, D, F, ops.EPI_SILU, n
        assert lib.fluxhip_gated_ff_grad(ctypes.byref(d), None) == -1, name

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


def _rotary_args(T=6, rot=8):
    return torch.arange(T), torch.ones(rot // 2, dtype=F64)


def _accepted(q, k, out, T=6):
    """Every check of the arguments passes: what stops the call is that these are host tensors."""
    from flux_generator_amd import ops
    p, f = _rotary_args(T)
    for fn in (ops.rotary, ops.rotary_backward):
        with pytest.raises(ops.FluxHipError, match="device tensors"):
            fn(q, k, p, f, out=out)


def _refused(q, k, out, match, T=6):
    from flux_generator_amd import ops
    p, f = _rotary_args(T)
    for fn in (ops.rotary, ops.rotary_backward):
        with pytest.raises(ops.FluxHipError, match=match):
            fn(q, k, p, f, out=out)


def test_rotary_outputs_that_overlap_are_refused():
    B, T, H, hd = 2, 6, 4, 8
    n = B * T * H * hd
    for step in (1, hd, H * hd):                        # an output shifted against its input
        buf = torch.zeros(n + step)
        q, o = buf[:n].view(B, T, H, hd), buf[step:].view(B, T, H, hd)
        _refused(q, None, o, "q itself")
        _refused(o, None, q, "q itself")
        _refused(torch.zeros(B, T, H, hd), q, (torch.zeros(B, T, H, hd), o), "k itself")
        _refused(q, torch.zeros(B, T, H, hd), (torch.zeros(B, T, H, hd), o), "memory of their own")
        _refused(torch.zeros(B, T, H, hd), torch.zeros(B, T, H, hd), (q, o), "memory of their own")
    buf = torch.zeros(n)                                # the input's memory with other strides
    _refused(buf.view(B, T, H, hd), None, buf.view(B, H, T, hd).transpose(1, 2), "q itself")
    _refused(buf.view(B, T, H, hd), None, buf.view(T, B, H, hd).transpose(0, 1), "q itself")
    _refused(torch.zeros(B, T, H, hd), buf.view(B, T, H, hd), (buf.view(B, H, T, hd).transpose(1, 2), torch.zeros(B, T, H, hd)), "memory of their own")
    _refused(buf.view(B, T, H, hd), buf.view(B, T, H, hd)[:, :, 1:3], (buf.view(B, T, H, hd), buf.view(B, T, H, hd)[:, :, 1:3]), "memory of their own")
    qkv = torch.zeros(B, T, 3 * H, hd)                  # heads of a fused projection, one too many
    _refused(qkv[:, :, :H + 1], qkv[:, :, H:2 * H], (qkv[:, :, :H + 1], qkv[:, :, H:2 * H]), "memory of their own")
    wide = torch.zeros(4 * n)                           # an output that meets itself
    _refused(torch.zeros(B, T, H, hd), None, wide.as_strided((B, T, H, hd), (T * H * hd, hd, hd, 1)), "overlap itself")
    _refused(torch.zeros(B, T, H, hd), None, wide.as_strided((B, T, H, hd), (hd, H * hd, hd, 1)), "overlap itself")


def test_rotary_outputs_that_do_not_overlap_are_accepted():
    B, T, H, K, hd = 2, 6, 4, 2, 8
    z = lambda *s: torch.zeros(*s)
    q, k = z(B, T, H, hd), z(B, T, K, hd)
    _accepted(q, k, (q, k))
    _accepted(q, k, (z(B, T, H, hd), k))
    _accepted(q, k, (q, z(B, K, T, hd).transpose(1, 2)))
    _accepted(q, None, q)
    _accepted(q, None, (q, None))
    _accepted(z(1, T, 1, hd).expand(B, T, H, hd), None, q)
    for qkv in (z(B, T, H + 2 * K, hd), z(B, T + 5, H + 2 * K, hd)[:, 5:], z(T, B, H + 2 * K, hd).transpose(0, 1), z(B, T, H + 2 * K, hd + 3)[..., 3:]):
        a, b, v = qkv[:, :, :H], qkv[:, :, H:H + K], qkv[:, :, H + K:]
        _accepted(a, b, (a, b))                         # q and k inside one projection
        _accepted(a, b, (a, v))                         # .. k written over the values
        _accepted(q, b, (a, v))
    for five, d in ((z(B, T, 3, H, hd), 2), (z(B, T, H, 3, hd), 3), (z(B, 3, H, T, hd).permute(0, 3, 2, 1, 4), 3), (z(3, B, T, H, hd).movedim(0, 2), 2)):
        a, b = five.select(d, 0), five.select(d, 1)
        assert a.shape == (B, T, H, hd)
        _accepted(a, b, (a, b))
        _accepted(a, None, b)
    flat = z(B * (T * H * hd + 5) + T * K * hd + 5)     # samples apart by what is no multiple of a row
    a = flat.as_strided((B, T, H, hd), (T * H * hd + 5, H * hd, hd, 1))
    _accepted(a, None, a)
    packed = z(B * (T * (H + K) * hd + 5))
    a = packed.as_strided((B, T, H, hd), (T * (H + K) * hd + 5, (H + K) * hd, hd, 1))
    b = packed.as_strided((B, T, K, hd), (T * (H + K) * hd + 5, (H + K) * hd, hd, 1), H * hd)
    _accepted(a, b, (a, b))
    cols = z(B, T, H, 2 * hd)                           # halves of wider heads
    _accepted(cols[..., :hd], cols[..., hd:], (cols[..., :hd], cols[..., hd:]))
    _accepted(z(B, 0, H, hd), z(B, 0, K, hd), (z(B, 0, H, hd), z(B, 0, K, hd)), T=0)
    _accepted(q[:, :, :0], k, (q[:, :, :0], k))


def test_rotary_overlap_is_judged_as_by_the_addresses():
    """Random pairs of views of one small buffer: an output that is let through shares no element with its input but as that input
    itself, and holds each of its elements once; most of those that lie apart are let through."""
    import ctypes
    import random
    from flux_generator_amd import _lib
    lib, rng = _lib.load(), random.Random(0)
    index = torch.arange(8192)
    count = dict(met=0, apart=0, proved=0, same=0, inside=0)
    for _ in range(20000):
        def strides():
            return [rng.choice((0, 1, 2, 3, 4, 5, 8, 12, 16, 32, 48, 96, 100)) for _ in range(3)]
        shape, sa, sb = [rng.randint(1, 4) for _ in range(4)], strides(), strides()
        at, bt = rng.randint(0, 60), rng.randint(0, 60)
        if rng.random() < 0.6:
            sb = sa
        if rng.random() < 0.05:
            sb, bt = sa, at
        ia, ib = (index.as_strided(shape, s + [1], o).reshape(-1).tolist() for s, o in ((sa, at), (sb, bt)))
        d = _lib.RotaryDesc()
        d.B, d.T, d.H, d.hd = shape
        d.dtype = rng.choice((0, 2))
        e = 4 if d.dtype == 2 else 2
        d.q, d.q_out, d.q_strides, d.qo_strides = (1 << 20) + e * at, (1 << 20) + e * bt, tuple(sa), tuple(sb)
        said, once, met = lib.fluxhip_rotary_overlap(ctypes.byref(d)), len(set(ib)) == len(ib), bool(set(ia) & set(ib))
        if said == 0:
            assert once and (not met or ia == ib), (shape, sa, at, sb, bt)
        if once and ia == ib and said != 3:
            assert said == 0
        count["inside"] += not once
        count["same"] += ia == ib
        count["met"] += once and met and ia != ib
        count["apart"] += once and not met
        count["proved"] += once and not met and said == 0
    assert all(n > 200 for n in count.values()) and count["proved"] > 0.5 * count["apart"], count


@pytest.mark.parametrize("version,match", [(9, "lacks fluxhip_.*build"), (8, "ABI version mismatch")])
def test_a_library_of_older_sources_is_named_as_such(tmp_path, monkeypatch, version, match):
    """A build from before a symbol came in (same ABI number), and one of another ABI number: each says so."""
    import shutil
    import subprocess
    from flux_generator_amd import _lib
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    (tmp_path / "old.c").write_text(f'int fluxhip_abi_version(void) {{ return {version}; }}\nconst char* fluxhip_arch(void) {{ return "gfx950"; }}\n')
    subprocess.run([cc, "-shared", "-fPIC", "-o", str(tmp_path / "old.so"), str(tmp_path / "old.c")], check=True)
    monkeypatch.setattr(_lib, "LIB_PATH", tmp_path / "old.so")
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.delenv("FLUXHIP_LIB_AB", raising=False)
    with pytest.raises(RuntimeError, match=match):
        _lib.load()
    assert _lib._lib is None

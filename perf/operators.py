"""Workloads of the operators that training an adapter needs on top of the sampling path: LayerNorm, the gated
feed-forward block and rotary positions, each forward (keeping what the gradient needs) and backward.

`own = False` computes them in plain torch (32-bit arithmetic, 64-bit angles, one rounding at the end); `own = True` calls the
framework.  Shapes are those of the framework's models: the SDXL UNet's transformer blocks (width 640 / 1280, GEGLU 4 x), the
T5-XXL feed-forward (4096 -> 10240), CLIP-L (768), Flux's joint attention (24 heads of 128, positions on three axes of
16 + 56 + 56), and odd sizes around them.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one pooled text vector through a norm while sampling: nothing but latency
        dict(name="ln_fwd_one_row", op="layernorm", batch=1, rows=1, width=1280, dtype="bf16", mod=False, packed=False),
        # norm3 of the UNet's 32 x 32 blocks, 16 images, float16
        dict(name="ln_fwd_unet", op="layernorm", batch=16, rows=1024, width=1280, dtype="f16", mod=False, packed=False),
        # three captions of 77 tokens through a CLIP-L norm in a training step; float32 master activations, odd width
        dict(name="ln_bwd_captions", op="layernorm_backward", batch=3, rows=77, width=771, dtype="f32", mod=False, packed=False),
        # adaLN of an image stream that lives inside a packed text + image buffer: per-image scale and shift, and their gradient
        dict(name="ln_bwd_modulated", op="layernorm_backward", batch=4, rows=4096, width=2560, dtype="bf16", mod=True, packed=True),
        # one token (a pooled vector) through the T5-XXL feed-forward: reads the weights once
        dict(name="ff_fwd_one_token", op="gated_ff", tokens=1, width=4096, hidden=10240, dtype="bf16", act="gelu_tanh", bias=False, save=False),
        # one prompt of 512 tokens through the T5-XXL feed-forward
        dict(name="ff_fwd_prompt", op="gated_ff", tokens=512, width=4096, hidden=10240, dtype="bf16", act="gelu_tanh", bias=False, save=False),
        # adapter training on a frozen 64 x 64 UNet block (width 640) with a ragged batch: gradient of the input alone
        dict(name="ff_bwd_frozen_ragged", op="gated_ff_backward", tokens=3407, width=640, hidden=2568, dtype="f16", act="gelu_erf", bias=False, weights=False),
        # full training step of the 32 x 32 UNet block on 16 images: gradients of the input, three weights and three biases
        dict(name="ff_bwd_unet", op="gated_ff_backward", tokens=16384, width=1280, hidden=5120, dtype="bf16", act="gelu_erf", bias=True, weights=True),
        # the newest position of 8 sequences, grouped heads, half layout: nothing but latency
        dict(name="rope_one_token", op="rotary", batch=8, tokens=1, heads=24, kv_heads=8, head=128, rot=128, axes=1, inter=False, far=0, dtype="bf16", fused=True),
        # Flux's positions at 1024 x 1024: 512 text tokens + 4096 patches, q and k inside the fused projection
        dict(name="rope_flux", op="rotary", batch=1, tokens=4608, heads=24, kv_heads=24, head=128, rot=128, axes=3, inter=True, far=0, dtype="bf16", fused=True),
        # a part of an odd-sized head, positions far out in a long context, float32
        dict(name="rope_partial_far", op="rotary", batch=2, tokens=2047, heads=10, kv_heads=2, head=84, rot=40, axes=1, inter=False, far=900001, dtype="f32", fused=False),
        # the gradient through the same rotation for a training batch of 4
        dict(name="rope_bwd_batch", op="rotary_backward", batch=4, tokens=4352, heads=24, kv_heads=24, head=128, rot=128, axes=3, inter=True, far=0, dtype="f16", fused=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("layernorm", "gated_ff", "rotary"))
    back = rng.random() < 0.5
    op = kind + ("_backward" if back else "")
    if kind == "layernorm":
        width = _log(rng, 16, 5120)
        batch = rng.choice((1, 2, 3, 5, 8))
        rows = _log(rng, 1, max(1, min(16384, 40_000_000 // (width * batch))))
        return dict(op=op, batch=batch, rows=rows, width=width, dtype=rng.choice(("bf16", "bf16", "f16", "f32")), mod=rng.random() < 0.4,
                    packed=rng.random() < 0.3)
    if kind == "gated_ff":
        width, hidden = 8 * _log(rng, 8, 512), 8 * _log(rng, 16, 1280)
        tokens = _log(rng, 1, max(1, min(16384, 16384 * 1280 * 5120 // (width * hidden))))
        c = dict(op=op, tokens=tokens, width=width, hidden=hidden, dtype=rng.choice(("bf16", "bf16", "f16")),
                 act=rng.choice(("gelu_tanh", "gelu_erf", "silu")), bias=rng.random() < 0.5)
        c["weights" if back else "save"] = rng.random() < 0.6
        return c
    head = 2 * _log(rng, 8, 128)
    kv = rng.choice((1, 2, 4, 8, 24))
    heads = kv * rng.choice((1, 1, 3, 5))
    heads = heads if heads <= 40 else kv
    axes = rng.choice((1, 1, 2, 3))
    rot = head if rng.random() < 0.5 else 2 * rng.randint(axes, head // 2)
    batch = rng.choice((1, 2, 3, 8))
    most = 4 * 4352 * 48 * 128 // (batch * (heads + kv) * head)
    return dict(op=op, batch=batch, tokens=_log(rng, 1, max(1, min(20000, most))), heads=heads, kv_heads=kv, head=head, rot=rot, axes=axes,
                inter=rng.random() < 0.5, far=rng.choice((0, 0, 7, 100_003, 3_000_017)), dtype=rng.choice(("bf16", "bf16", "f16", "f32")),
                fused=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _axes_dim(c):
    """Rotated width per position axis: Flux's 16 + 56 + 56 in general form (a small first axis, the rest shared evenly)."""
    n, pairs = c["axes"], c["rot"] // 2
    if n == 1:
        return [2 * pairs]
    first = max(1, pairs // 8)
    each = (pairs - first) // (n - 1)
    return [2 * first] + [2 * each] * (n - 2) + [2 * (pairs - first - each * (n - 2))]


def _frequencies(c):
    """theta^(-2 j / d) for the pairs of every axis, in 64 bits."""
    parts = [10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d) for d in _axes_dim(c) if d]
    return torch.cat(parts)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[c["dtype"]]

    def rnd(*shape, scale=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)

    s = {"case": dict(c)}
    if c["op"].startswith("layernorm"):
        B, T, D = c["batch"], c["rows"], c["width"]
        lead = 13 if c["packed"] else 0                   # rows of another stream in front of this one
        chan = torch.exp(0.5 * torch.randn(D, generator=g, device="cuda"))      # channels of unlike size, as norms see them
        s["x"] = ((torch.randn(B, T + lead, D, generator=g, device="cuda") * chan) + 0.3).to(dt)[:, lead:]
        shape = (B, D) if c["mod"] else (D,)
        s["gamma"] = rnd(*shape, scale=0.2, mean=0.0 if c["mod"] else 1.0)
        s["beta"] = rnd(*shape, scale=0.2)
        if c["op"].endswith("backward"):
            s["dy"] = rnd(B, T, D)
            x = s["x"].float()
            s["mean"] = x.mean(-1)
            s["rstd"] = torch.rsqrt((x - s["mean"][..., None]).square().mean(-1) + 1e-6)
    elif c["op"].startswith("gated_ff"):
        M, D, F = c["tokens"], c["width"], c["hidden"]
        s["x"] = rnd(M, D)
        s["wv"], s["wg"], s["wo"] = rnd(F, D, scale=D ** -0.5), rnd(F, D, scale=D ** -0.5), rnd(D, F, scale=F ** -0.5)
        s["bv"], s["bg"], s["bo"] = (rnd(F, scale=0.2), rnd(F, scale=0.2), rnd(D, scale=0.2)) if c["bias"] else (None, None, None)
        if c["op"].endswith("backward"):
            s["dy"] = rnd(M, D)
            v, a = s["x"] @ s["wv"].t(), s["x"] @ s["wg"].t()
            if c["bias"]:
                v, a = v + s["bv"], a + s["bg"]
            s["saved"] = (v, a, (v.float() * _act(a.float(), c["act"])).to(dt))
    else:
        B, T, H, K, h = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["head"]
        if c["fused"]:                                    # q and k inside one projection's output, with the values behind them
            qkv = rnd(B, T, (H + 2 * K) * h)
            s["q"], s["k"] = qkv[..., : H * h].unflatten(-1, (H, h)), qkv[..., H * h: (H + K) * h].unflatten(-1, (K, h))
        else:
            s["q"], s["k"] = rnd(B, T, H, h), rnd(B, T, K, h)
        at = torch.arange(T, device="cuda", dtype=torch.int64)[None].repeat(B, 1)
        at = at + c["far"] + torch.randint(0, 50, (B, 1), generator=g, device="cuda")
        if c["axes"] > 1:                                 # (text index, row, column) of a patch
            side = max(1, int(math.sqrt(T)))
            at = torch.stack([at // 4096, at // side, at % side][: c["axes"]], -1)
        s["positions"] = at.contiguous()
        s["freqs"] = _frequencies(c)
        s["axes_dim"] = _axes_dim(c)
        s["scale"] = 1.0 if not c["far"] else 0.1 * math.log(8.0) + 1.0       # the amplitude long-context scaling asks for
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _phi(x):
    return 0.5 * torch.erfc(x * -math.sqrt(0.5))


def _act(x, kind):
    if kind == "gelu_erf":
        return x * _phi(x)
    if kind == "silu":
        return x * torch.sigmoid(x)
    return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x))


def _act_grad(x, kind):
    if kind == "gelu_erf":
        return _phi(x) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    if kind == "silu":
        p = torch.sigmoid(x)
        return p * (1 + x * (1 - p))
    u = 2 * math.sqrt(2 / math.pi)
    p = torch.sigmoid(u * (x + 0.044715 * x * x * x))
    return p + x * p * (1 - p) * u * (1 + 3 * 0.044715 * x * x)


def _plain_layernorm(s, c):
    x, off = s["x"].float(), 1.0 if c["mod"] else 0.0
    gamma, beta = s["gamma"].float() + off, s["beta"].float()
    if c["mod"]:
        gamma, beta = gamma[:, None], beta[:, None]
    if not c["op"].endswith("backward"):
        mean = x.mean(-1, keepdim=True)
        rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + 1e-6)
        return ((x - mean) * rstd * gamma + beta).to(s["x"].dtype), mean[..., 0], rstd[..., 0]
    dy, rstd = s["dy"].float(), s["rstd"][..., None]
    xh = (x - s["mean"][..., None]) * rstd
    g = dy * gamma
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    over = (1,) if c["mod"] else (0, 1)
    dt = s["x"].dtype
    return dx.to(dt), (dy * xh).sum(over).to(dt), dy.sum(over).to(dt)


def _plain_gated_ff(s, c):
    dt = s["x"].dtype
    x, wv, wg, wo = s["x"].float(), s["wv"].float(), s["wg"].float(), s["wo"].float()
    if not c["op"].endswith("backward"):
        v, a = x @ wv.t(), x @ wg.t()
        if c["bias"]:
            v, a = v + s["bv"].float(), a + s["bg"].float()
        h = v * _act(a, c["act"])
        y = h @ wo.t()
        if c["bias"]:
            y = y + s["bo"].float()
        return (y.to(dt), (v.to(dt), a.to(dt), h.to(dt))) if c["save"] else y.to(dt)
    v, a, h = (t.float() for t in s["saved"])
    dy = s["dy"].float()
    dh = dy @ wo
    dv, da = dh * _act(a, c["act"]), dh * v * _act_grad(a, c["act"])
    out = [(dv @ wv + da @ wg).to(dt)]
    if c["weights"]:
        out += [(dv.t() @ x).to(dt), (da.t() @ x).to(dt), (dy.t() @ h).to(dt)]
        if c["bias"]:
            out += [dv.sum(0).to(dt), da.sum(0).to(dt), dy.sum(0).to(dt)]
    return out


def _plain_rotary(s, c):
    at = s["positions"].double()
    if c["axes"] == 1:
        at = at[..., None]
    axis = torch.cat([torch.full((d // 2,), i, device=at.device) for i, d in enumerate(s["axes_dim"])]).long()
    ang = at[..., axis] * s["freqs"]
    cos, sin = (torch.cos(ang) * s["scale"]).float()[:, :, None], (torch.sin(ang) * s["scale"]).float()[:, :, None]
    if c["op"].endswith("backward"):
        sin = -sin

    def turn(x):
        r, y = c["rot"], x.float()
        z = y[..., :r]
        a, b = (z[..., 0::2], z[..., 1::2]) if c["inter"] else (z[..., : r // 2], z[..., r // 2:])
        p, q = a * cos - b * sin, a * sin + b * cos
        z = torch.stack([p, q], -1).flatten(-2) if c["inter"] else torch.cat([p, q], -1)
        return torch.cat([z, y[..., r:]], -1).to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["op"].startswith("layernorm"):
        return _plain_layernorm(s, c)
    if c["op"].startswith("gated_ff"):
        return _plain_gated_ff(s, c)
    return _plain_rotary(s, c)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s, c):
    from flux_generator_amd import ops
    op = c["op"]
    if op == "layernorm":
        return ops.layernorm(s["x"], s["gamma"], s["beta"], eps=1e-6, unit_offset=c["mod"])
    if op == "layernorm_backward":
        return ops.layernorm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"], unit_offset=c["mod"])
    if op.startswith("gated_ff"):
        act = {"gelu_erf": ops.EPI_GELU_ERF, "gelu_tanh": ops.EPI_GELU_TANH, "silu": ops.EPI_SILU}[c["act"]]
        if op == "gated_ff":
            return ops.gated_ff(s["x"], s["wv"], s["wg"], s["wo"], s["bv"], s["bg"], s["bo"], act=act, save=c["save"])
        out = ops.gated_ff_backward(s["dy"], s["x"], s["saved"], s["wv"], s["wg"], s["wo"], act=act, weight_grads=c["weights"],
                                    bias_grads=c["weights"] and c["bias"])
        return [t for t in out if t is not None]
    turn = ops.rotary if op == "rotary" else ops.rotary_backward
    return turn(s["q"], s["k"], s["positions"], s["freqs"], axes_dim=s["axes_dim"], interleaved=c["inter"], scale=s["scale"])


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"].startswith("layernorm"):
        n, rows = c["batch"] * c["rows"] * c["width"], c["batch"] * c["rows"]
        par = (c["batch"] if c["mod"] else 1) * c["width"]
        if c["op"].endswith("backward"):
            return {"bytes": 3 * n * e + 3 * par * e + 8 * rows, "flops": 14 * n}
        return {"bytes": 2 * n * e + 2 * par * e + 8 * rows, "flops": 8 * n}
    if c["op"].startswith("gated_ff"):
        M, D, F = c["tokens"], c["width"], c["hidden"]
        if not c["op"].endswith("backward"):
            par = 3 * D * F + (2 * F + D if c["bias"] else 0)
            return {"bytes": e * (par + 2 * M * D + (3 * M * F if c["save"] else 0)), "flops": 6 * M * D * F}
        if not c["weights"]:                               # the hidden values and x are not needed for the gradient of x alone
            return {"bytes": e * (3 * D * F + 2 * M * D + 2 * M * F), "flops": 6 * M * D * F}
        par = 6 * D * F + (2 * F + D if c["bias"] else 0)
        return {"bytes": e * (par + 3 * M * D + 3 * M * F), "flops": 12 * M * D * F}
    n = c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["head"]
    return {"bytes": 2 * n * e + 8 * c["batch"] * c["tokens"] * c["axes"] + 4 * c["rot"], "flops": 3 * n}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"].startswith("layernorm"):
        x, D = s["x"].double(), c["width"]
        gamma, beta = s["gamma"].double(), s["beta"].double()
        if c["mod"]:
            gamma, beta = (1 + gamma).unsqueeze(1), beta.unsqueeze(1)
        if c["op"] == "layernorm":
            mu = x.sum(-1, keepdim=True) / D
            sd = torch.sqrt(((x - mu) ** 2).sum(-1, keepdim=True) / D + 1e-6)
            return (x - mu) / sd * gamma + beta, mu.squeeze(-1), 1 / sd.squeeze(-1)
        dy, r = s["dy"].double(), s["rstd"].double().unsqueeze(-1)
        n = (x - s["mean"].double().unsqueeze(-1)) * r
        e = dy * gamma
        dx = (D * e - e.sum(-1, keepdim=True) - n * (e * n).sum(-1, keepdim=True)) * r / D
        dg, db = (dy * n).sum(1), dy.sum(1)
        return (dx, dg, db) if c["mod"] else (dx, dg.sum(0), db.sum(0))
    if c["op"].startswith("gated_ff"):
        d = {k: None if s.get(k) is None else s[k].double() for k in ("x", "wv", "wg", "wo", "bv", "bg", "bo", "dy")}
        F64 = torch.float64
        tanh = math.sqrt(2 / math.pi)

        def gate(z):                                       # the activation and its derivative
            if c["act"] == "gelu_erf":
                cdf = (1 + torch.erf(z / math.sqrt(2))) / 2
                return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
            if c["act"] == "silu":
                sg = 1 / (1 + torch.exp(-z))
                return z * sg, sg + z * sg * (1 - sg)
            t = torch.tanh(tanh * (z + 0.044715 * z ** 3))
            return z * (1 + t) / 2, (1 + t) / 2 + z / 2 * (1 - t * t) * tanh * (1 + 0.134145 * z * z)

        if c["op"] == "gated_ff":
            v, z = torch.mm(d["x"], d["wv"].t().contiguous()), torch.mm(d["x"], d["wg"].t().contiguous())
            if c["bias"]:
                v, z = v + d["bv"], z + d["bg"]
            h = v * gate(z)[0]
            y = torch.mm(h, d["wo"].t().contiguous())
            if c["bias"]:
                y = y + d["bo"]
            return (y, (v, z, h)) if c["save"] else y
        v, z, h = (t.to(F64) for t in s["saved"])
        a, da = gate(z)
        dh = torch.mm(d["dy"], d["wo"])
        dv, dz = dh * a, dh * v * da
        out = [torch.mm(dv, d["wv"]) + torch.mm(dz, d["wg"])]
        if c["weights"]:
            out += [torch.mm(dv.t().contiguous(), d["x"]), torch.mm(dz.t().contiguous(), d["x"]), torch.mm(d["dy"].t().contiguous(), h)]
            if c["bias"]:
                out += [dv.sum(0), dz.sum(0), d["dy"].sum(0)]
        return out
    at, dims, col, angles = s["positions"].double().reshape(c["batch"], c["tokens"], c["axes"]), _axes_dim(c), 0, []
    for i, d in enumerate(dims):
        for j in range(d // 2):
            angles.append(at[..., i] * s["freqs"][col])
            col += 1
    unit = torch.polar(torch.full_like(angles[0], s["scale"]), torch.zeros_like(angles[0]))
    turn = torch.stack([unit * torch.polar(torch.ones_like(a), -a if c["op"].endswith("backward") else a) for a in angles], -1).unsqueeze(2)
    got = []
    for name in ("q", "k"):
        x, r = s[name].double(), c["rot"]
        head, tail = x[..., :r], x[..., r:]
        if c["inter"]:
            z = torch.view_as_complex(head.reshape(*head.shape[:-1], r // 2, 2).contiguous()) * turn
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(head[..., : r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
            y = torch.cat([z.real, z.imag], -1)
        got.append(torch.cat([y, tail], -1))
    return tuple(got)

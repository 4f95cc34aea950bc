"""Measured cases of the 8-bit integer linear, the 8-bit checkpoints and the sandwich norm.

Operators: ``int8_linear`` (product in 8-bit integers with a scale per token and
per channel, and its input gradient), ``gelu_int8`` with ``gelu_int8_bwd`` (the
GELU of an MLP whose input is kept in 8 bits for the backward pass),
``int8_wgrad`` (weight gradient from 8-bit checkpoints) and ``sandwich_norm``
with ``sandwich_norm_bwd`` (norms before and after a block with its gate and
residual scale).  ``run`` computes each in plain 32-bit torch, or with ``own``
through the framework's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FLOOR = 1e-30  # smallest row maximum that is quantised
EPS = 1e-6


def listed():
    return [
        # the modulation vectors of one sample: one timestep embedding row through a wide projection
        dict(name="linear_1", op="linear", M=1, K=2048, N=6144, dtype="bf16", bias=True),
        # a trimmed text context into the cross attention's keys, odd on both sides
        dict(name="linear_77", op="linear", M=77, K=1024, N=2047, dtype="fp16", bias=False),
        # the fused qkv projection of one 1024x1024 image's tokens
        dict(name="linear_4096", op="linear", M=4096, K=2048, N=6144, dtype="bf16", bias=False),
        # the MLP's up projection at guidance batch two
        dict(name="linear_8192", op="linear", M=8192, K=2048, N=8192, dtype="bf16", bias=True),
        # training through the frozen down projection: output and input gradient
        dict(name="linear_train_4096", op="linear_train", M=4096, K=8192, N=2048, dtype="bf16", bias=False),
        # a short context through the MLP's activation, forward and backward
        dict(name="gelu_77", op="gelu", M=77, K=8192, dtype="bf16"),
        # the MLP hidden of two images, forward and backward
        dict(name="gelu_8192", op="gelu", M=8192, K=8192, dtype="bf16"),
        # a rank-16 adapter's first factor over one image's tokens
        dict(name="wgrad_lora_4096", op="wgrad", M=4096, K=2048, N=16, dtype="bf16"),
        # the full gradient of the up projection over one image's tokens
        dict(name="wgrad_4096", op="wgrad", M=4096, K=2048, N=8192, dtype="bf16"),
        # one token through the block's norms
        dict(name="sandwich_1", op="sandwich", B=1, S=1, D=2048, dtype="bf16"),
        # the forward at guidance batch two
        dict(name="sandwich_8192", op="sandwich", B=2, S=4096, D=2048, dtype="bf16"),
        # the backward of one image
        dict(name="sandwich_bwd_4096", op="sandwich_bwd", B=1, S=4096, D=2048, dtype="bf16"),
    ]


def _size(rng, lo, hi, unit=1):
    """A multiple of `unit`, spread over the logarithm of its range: a power of two, as models have, or odd."""
    n = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    if rng.random() < 0.4:
        return unit * 2 ** min(round(math.log2(n)), int(math.log2(hi)))
    return unit * (min(int(n), hi - 1) | 1)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_train", "gelu", "wgrad", "sandwich", "sandwich_bwd"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("linear", "linear_train", "wgrad"):
        K = _size(rng, 8, 512, 16)
        N = _size(rng, 1, 512, 16) if op == "linear_train" else _size(rng, 4, 4096 if op == "wgrad" else 8192)
        # no more products than the largest listed case
        M = _size(rng, 1, min(8192, 4096 * 2048 * 8192 // (K * N)))
        case = dict(op=op, M=M, K=K, N=N, dtype=dtype)
        if op != "wgrad":
            case["bias"] = rng.random() < 0.5
        return case
    if op == "gelu":
        return dict(op=op, M=_size(rng, 1, 8192), K=_size(rng, 8, 256, 16), dtype=dtype)
    B = rng.choice([1, 1, 2, 3, 4])
    return dict(op=op, B=B, S=_size(rng, 1, 8192 // B), D=_size(rng, 8, 256, 8), dtype=dtype)


# ---------------------------------------------------------------- inputs --
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _acts(g, M, K, dtype):
    """Activations with outlier channels, as a DiT's residual stream has them."""
    hot = 1.0 + 7.0 * (torch.rand(K, generator=g, device="cuda") < 0.02)
    return (_randn(g, M, K) * hot).to(dtype)


def _codes(x):
    """8-bit codes and scales of a 2-D tensor's rows, in 32 bits."""
    x = x.float()
    amax = x.abs().amax(dim=1, keepdim=True).clamp_min(FLOOR)
    return torch.round(x * 127.0 / amax), amax / 127.0


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    op = case["op"]
    st = {"op": op, "dtype": dt}
    if op in ("linear", "linear_train"):
        M, K, N = case["M"], case["K"], case["N"]
        st["x"] = _acts(g, M, K, dt)
        wq, ws = _codes(_randn(g, N, K) * (0.5 / math.sqrt(K)))
        st["wq"], st["ws"] = wq.to(torch.int8), ws.flatten()
        st["bias"] = (0.1 * _randn(g, N)).to(dt) if case["bias"] else None
        if op == "linear_train":
            st["wt"] = st["wq"].t().contiguous()
            st["dy"] = (1e-2 * _randn(g, M, N)).to(dt)
            st["x"].requires_grad_(True)
    elif op == "gelu":
        M, K = case["M"], case["K"]
        st["x"] = (1.5 * _randn(g, M, K)).to(dt)
        st["dy"] = (1e-2 * _randn(g, M, K)).to(dt)
    elif op == "wgrad":
        M, K, N = case["M"], case["K"], case["N"]
        q, s = _codes(_acts(g, M, K, dt))
        st["q"], st["s"] = q.to(torch.int8), s
        st["dy"] = (1e-2 * _randn(g, M, N)).to(dt)
    else:
        B, S, D = case["B"], case["S"], case["D"]
        st["alpha"] = 1.25
        st["x"] = (2.0 * _randn(g, B, S, D)).to(dt)
        st["res"] = _acts(g, B * S, D, dt).view(B, S, D)
        st["gate"] = (0.3 * _randn(g, B, D)).to(dt)
        st["shift"] = (0.1 * _randn(g, B, D)).to(dt)
        st["scale"] = (1.0 + 0.1 * _randn(g, B, D)).to(dt)
        st["post"] = 1.0 + 0.1 * _randn(g, D)
        st["pre"] = 1.0 + 0.1 * _randn(g, D)
        if op == "sandwich_bwd":
            st["z"] = _sandwich(st)[1]
            st["gh"] = (1e-2 * _randn(g, B, S, D)).to(dt)
            st["gz"] = (1e-2 * _randn(g, B, S, D)).to(dt)
    return st


# ----------------------------------------------------------- plain forms --
def _linear(st):
    q, s = _codes(st["x"].detach())
    y = (q @ st["wq"].float().t()) * s * st["ws"]
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if st["op"] == "linear":
        return y.to(st["dtype"])
    gq, gs = _codes(st["dy"].float() * st["ws"])
    return y.to(st["dtype"]), ((gq @ st["wq"].float()) * gs).to(st["dtype"])


def _gelu(st):
    x = st["x"].float()
    q, s = _codes(0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5))))
    c, cs = _codes(x)
    v = c * cs
    d = 0.5 * (1.0 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2.0 * math.pi)
    return (q * s).to(st["dtype"]), (st["dy"].float() * d).to(st["dtype"])


def _wgrad(st):
    return (st["dy"].float().t() @ (st["q"].float() * st["s"])).to(st["dtype"])


def _rstd(v):
    return torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS)


def _sandwich(st):
    x, gate, scale, shift = (st[k].float() for k in ("x", "gate", "scale", "shift"))
    u = x * _rstd(x) * st["post"]
    z = (st["alpha"] * st["res"].float() + gate[:, None] * u).to(st["dtype"])
    v = z.float()
    h = v * _rstd(v) * st["pre"] * scale[:, None] + shift[:, None]
    return h.to(st["dtype"]), z


def _sandwich_bwd(st):
    gh, gz, z, x, gate, scale = (st[k].float() for k in ("gh", "gz", "z", "x", "gate", "scale"))
    dt, pre, post = st["dtype"], st["pre"], st["post"]
    r1, r2 = _rstd(x), _rstd(z)
    xh, zh = x * r1, z * r2
    p = gh * scale[:, None] * pre
    dz = gz + r2 * (p - zh * (p * zh).mean(dim=-1, keepdim=True))
    m = dz * gate[:, None] * post
    dx = r1 * (m - xh * (m * xh).mean(dim=-1, keepdim=True))
    P, Q = (gh * zh).sum(dim=1), (dz * xh).sum(dim=1)
    return (dx.to(dt), (st["alpha"] * dz).to(dt), (Q * post).to(dt), (gate * Q).sum(dim=0),
            (scale * P).sum(dim=0), gh.sum(dim=1).to(dt), (P * pre).to(dt))


def run(st):
    op = st["op"]
    if not own:
        return {"linear": _linear, "linear_train": _linear, "gelu": _gelu, "wgrad": _wgrad,
                "sandwich": _sandwich, "sandwich_bwd": _sandwich_bwd}[op](st)
    import anima_flat_b200 as afb

    if op == "linear":
        return afb.int8_linear(st["x"], afb.Int8Weight(st["wq"], st["ws"]), st["bias"])
    if op == "linear_train":
        y = afb.int8_linear(st["x"], afb.Int8Weight(st["wq"], st["ws"], st["wt"]), st["bias"])
        (dx,) = torch.autograd.grad(y, st["x"], st["dy"])
        return y.detach(), dx
    if op == "gelu":
        q, s, c, cs = afb.gelu_int8(st["x"])
        return afb.int8_restore(q, s, st["dtype"]), afb.gelu_int8_bwd(st["dy"], c, cs)
    if op == "wgrad":
        return afb.int8_wgrad(st["dy"], st["q"], st["s"])
    if op == "sandwich":
        return afb.sandwich_norm(st["x"], st["res"], st["gate"], st["post"], st["pre"], st["shift"],
                                 st["scale"], st["alpha"], EPS)
    return afb.sandwich_norm_bwd(st["gh"], st["gz"], st["z"], st["x"], st["gate"], st["post"], st["pre"],
                                 st["scale"], st["alpha"], EPS)


# ------------------------------------------------------------------ work --
def work(case):
    op = case["op"]
    if op in ("linear", "linear_train", "wgrad"):
        M, K, N = case["M"], case["K"], case["N"]
        if op == "wgrad":
            return {"bytes": 2 * M * N + M * K + 4 * M + 2 * N * K, "flops": 2 * M * N * K}
        fwd = 2 * M * K + N * K + 4 * N + (2 * N if case["bias"] else 0) + 2 * M * N
        if op == "linear":
            return {"bytes": fwd, "flops": 2 * M * N * K}
        return {"bytes": fwd + 2 * M * N + N * K + 2 * M * K, "flops": 4 * M * N * K}
    if op == "gelu":
        # x and dy read, the restored output and dx written
        return {"bytes": 8 * case["M"] * case["K"], "flops": 40 * case["M"] * case["K"]}
    B, S, D = case["B"], case["S"], case["D"]
    if op == "sandwich":
        return {"bytes": 8 * B * S * D + 6 * B * D + 8 * D, "flops": 15 * B * S * D}
    return {"bytes": 12 * B * S * D + 10 * B * D + 16 * D, "flops": 40 * B * S * D}


# ----------------------------------------------------------------- exact --
def _exact_codes(x):
    top = x.abs().max(dim=1).values.clamp(min=FLOOR)[:, None]
    return (127.0 * x / top).round(), top / 127.0


def exact(case, seed):
    st = prepare(case, seed)
    d = {k: (v.detach().double() if isinstance(v, torch.Tensor) else v) for k, v in st.items()}
    op = case["op"]
    if op in ("linear", "linear_train"):
        q, s = _exact_codes(d["x"])
        y = torch.einsum("mk,nk->mn", q, d["wq"]) * s * d["ws"][None, :]
        y = y if d["bias"] is None else y + d["bias"][None, :]
        if op == "linear":
            return y
        gq, gs = _exact_codes(d["dy"] * d["ws"][None, :])
        return y, torch.einsum("mn,nk->mk", gq, d["wq"]) * gs
    if op == "gelu":
        q, s = _exact_codes(d["x"] * torch.special.ndtr(d["x"]))
        c, cs = _exact_codes(d["x"])
        v = c * cs
        pdf = torch.exp(-v.square() / 2) / math.sqrt(2 * math.pi)
        return q * s, d["dy"] * (torch.special.ndtr(v) + v * pdf)
    if op == "wgrad":
        return torch.einsum("mn,mk->nk", d["dy"], d["q"] * d["s"])

    def inv_rms(v):
        return 1.0 / torch.sqrt(v.square().sum(-1, keepdim=True) / v.shape[-1] + EPS)

    row = lambda k: d[k].unsqueeze(1)  # noqa: E731
    if op == "sandwich":
        z = d["alpha"] * d["res"] + row("gate") * d["post"] * d["x"] * inv_rms(d["x"])
        v = z.to(st["dtype"]).double()
        return d["pre"] * row("scale") * v * inv_rms(v) + row("shift"), z
    D = case["D"]
    ix, iz = inv_rms(d["x"]), inv_rms(d["z"])
    # the gradient of v / rms(v) against a cotangent c: i c - i^3 v <c, v> / D
    c = d["gh"] * row("scale") * d["pre"]
    dz = d["gz"] + iz * c - iz**3 * d["z"] * (c * d["z"]).sum(-1, keepdim=True) / D
    c = dz * row("gate") * d["post"]
    dx = ix * c - ix**3 * d["x"] * (c * d["x"]).sum(-1, keepdim=True) / D
    dgate = torch.einsum("bsd,bsd->bd", dz, d["x"] * ix)
    dscale = torch.einsum("bsd,bsd->bd", d["gh"], d["z"] * iz)
    return (dx, d["alpha"] * dz, dgate * d["post"], (dgate * d["gate"]).sum(0), (dscale * d["scale"]).sum(0),
            d["gh"].sum(1), dscale * d["pre"])

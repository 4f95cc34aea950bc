"""Offsets beyond 32 bits, and the registered ops beside the direct calls."""

from __future__ import annotations

import pytest
import torch

import anima_flat_b200 as afb

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_offsets_beyond_32_bits(cuda_dev):
    rows, K = 140000, 16384  # 2.3e9 elements
    assert rows * K > 2**31
    tail = torch.randn(64, K, device=cuda_dev).to(BF)
    x = torch.zeros(rows, K, dtype=BF, device=cuda_dev)
    x[-64:] = tail
    q, s = afb.rowquant_int8(x)
    tq, ts = afb.rowquant_int8(tail)
    assert torch.equal(q[-64:], tq) and torch.equal(s[-64:], ts) and not q[:64].any()
    assert torch.equal(afb.int8_restore(q, s)[-64:], afb.int8_restore(tq, ts))
    w = afb.quantize_weight_int8(torch.randn(40, K, device=cuda_dev).to(BF))
    y = afb.int8_linear((q, s), w)
    assert torch.equal(y[-64:], afb.int8_linear((tq, ts), w)) and not y[: rows - 64].any()
    assert torch.equal(afb.int8_linear(x, w)[-64:], y[-64:])
    dy = torch.zeros(rows, 8, dtype=BF, device=cuda_dev)
    dy[-64:] = 1
    got, want = afb.int8_wgrad(dy, q, s).double(), tq.double().mul(ts.double()).sum(0).expand(8, K)
    mag = tq.double().mul(ts.double()).abs().sum(0)
    assert ((got - want).abs() <= (2.0**-8 + 64 * 2.0**-23) * mag + 2.0**-8 * want.abs()).all()
    del q, s, y
    g = afb.gelu_int8(x)
    tg = afb.gelu_int8(tail)
    assert all(torch.equal(a[-64:], b) for a, b in zip(g, tg))
    dx = afb.gelu_int8_bwd(x, g[2], g[3])
    assert torch.equal(dx[-64:], afb.gelu_int8_bwd(tail, tg[2], tg[3]))


def test_sandwich_offsets_beyond_32_bits(cuda_dev):
    B, S, D = 1, 600000, 4096
    assert B * S * D > 2**31
    x, res = torch.zeros(B, S, D, dtype=BF, device=cuda_dev), torch.zeros(B, S, D, dtype=BF, device=cuda_dev)
    x[:, -7:], res[:, -7:] = torch.randn(2, B, 7, D, device=cuda_dev).to(BF)
    w = 1 + 0.1 * torch.randn(D, device=cuda_dev)
    h, z = afb.sandwich_norm(x, res, None, w, w)
    hs, zs = afb.sandwich_norm(x[:, -7:], res[:, -7:], None, w, w)
    # the two sizes take different kernels, whose sums differ in order: a step of bf16 at most
    for a, b in ((z[:, -7:], zs), (h[:, -7:], hs)):
        assert ((a.float() - b.float()).abs() <= 2.0**-7 * b.float().abs()).all()
    assert not z[:, :-7].any()
    dx, dres, *_ = afb.sandwich_norm_bwd(h, None, z, x, None, w, w)
    dxs, dress, *_ = afb.sandwich_norm_bwd(h[:, -7:], None, z[:, -7:], x[:, -7:], None, w, w)
    for a, b in ((dx[:, -7:], dxs), (dres[:, -7:], dress)):
        scale = b.float().abs().amax()
        assert ((a.float() - b.float()).abs() <= 2.0**-6 * scale).all()


def test_registered_ops_match_the_direct_calls(cuda_dev):
    ops = torch.ops.anima_flat_b200
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, b = rn(37, 256).to(BF), rn(48).to(BF)
    w = afb.quantize_weight_int8(rn(48, 256).to(BF), backward=True)
    xr = x.clone().requires_grad_(True)
    dy = rn(37, 48).to(BF)
    direct = afb.int8_linear(xr, w, b)
    through = ops.int8_linear(xr, *w, b)
    assert torch.equal(direct, through)
    (ga,), (gb,) = torch.autograd.grad(direct, xr, dy), torch.autograd.grad(through, xr, dy)
    assert torch.equal(ga, gb) and torch.equal(ga, afb.int8_linear_dx(dy, w)) and torch.equal(ga, ops.int8_linear_bwd(dy, w.s, w.qt))
    q, s = afb.rowquant_int8(x)
    assert all(torch.equal(a, c) for a, c in zip((q, s), ops.rowquant_int8(x)))
    gl = afb.gelu_int8(x)
    assert all(torch.equal(a, c) for a, c in zip(gl, ops.gelu_int8(x)))
    assert torch.equal(afb.gelu_int8_bwd(x, *gl[2:]), ops.gelu_int8_bwd(x, *gl[2:]))
    assert torch.equal(afb.int8_restore(q, s), ops.int8_restore(q, s, BF))
    assert torch.equal(afb.int8_wgrad(dy, q, s), ops.int8_wgrad(dy, q, s))
    f = 1 + 0.1 * rn(256)
    a3 = [t.requires_grad_(True) for t in (rn(2, 5, 256).to(BF), rn(2, 5, 256).to(BF), rn(2, 256).to(BF), f, f.clone(),
                                           rn(2, 256).to(BF), rn(2, 256).to(BF))]
    out, ref = afb.sandwich_norm(*a3, 1.5, 1e-6), ops.sandwich_norm(*a3, 1.5, 1e-6)
    assert all(torch.equal(a, c) for a, c in zip(out, ref))
    gs = [rn(2, 5, 256).to(BF) for _ in range(2)]
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(out, a3, gs), torch.autograd.grad(ref, a3, gs)))


@pytest.mark.parametrize("name", ["int8_linear", "int8_wgrad", "gelu_int8", "sandwich_norm"])
def test_ops_pass_the_schema_and_fake_checks(name, cuda_dev):
    x, f = torch.randn(2, 6, 64, device=cuda_dev).to(BF), torch.ones(64, device=cuda_dev)
    q, s = afb.rowquant_int8(x)
    w = afb.quantize_weight_int8(torch.randn(48, 64, device=cuda_dev).to(BF))
    args = {"int8_linear": (x, w.q, w.s, None, None), "int8_wgrad": (x, q, s), "gelu_int8": (x,),
            "sandwich_norm": (x, x.clone(), None, f, f.clone(), None, None, 1.0, 1e-6)}[name]
    torch.library.opcheck(getattr(torch.ops.anima_flat_b200, name), args, test_utils=("test_schema", "test_faketensor"))


def test_compiled_code_takes_the_registered_ops(cuda_dev):
    x = torch.randn(2, 6, 64, device=cuda_dev).to(BF)
    w = afb.quantize_weight_int8(torch.randn(48, 64, device=cuda_dev).to(BF))
    fn = torch.compile(lambda t: afb.int8_linear(t, w) * 2, backend="eager", fullgraph=True)
    assert torch.equal(fn(x), afb.int8_linear(x, w) * 2)

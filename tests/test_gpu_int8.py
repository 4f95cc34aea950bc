"""8-bit integer linear and 8-bit checkpoints on the GPU against the definitions in 64 bits.

Bounds.  u is the half-step of the 16-bit type: 2^-8 (bf16) or 2^-11 (fp16),
with a half-step of 2^-25 below fp16's normal range.

- rowquant_int8: codes equal, scales equal to the fp32 quotient (both are
  exactly rounded for 16-bit inputs).
- int8_linear: the integer sum is exact, then four fp32 roundings of 2^-24 and
  the output's: u |y| + 2^-22 (|product| + |bias|).
- gelu_int8: the fast GELU is within 2^-20 + 2^-12 |g| of the exact one, and a
  code within half a step of its value.
- gelu_int8_bwd: the slope's error is 2^-19 at most (A&S 7.1.26 and the
  special-function unit's), then two roundings: u |dx| + 2^-18 |dy|.
- int8_wgrad: each restored value is rounded once to 16 bits and the sum runs
  in fp32: (u + T 2^-23) sum |dy x| + u |dw|.
"""

from __future__ import annotations

import math

import pytest
import torch

import anima_flat_b200 as afb

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0**-8, HF: 2.0**-11}
TINY = {BF: 2.0**-133, HF: 2.0**-25}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _acts(g, shape, dt, hot=True):
    x = torch.randn(*shape, generator=g, device="cuda")
    if hot:
        x = x * (1.0 + 30.0 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.02))
    return x.to(dt)


def _codes64(x):
    a = x.double().abs().amax(-1, keepdim=True).clamp_min(1e-30)
    return torch.round(127.0 * x.double() / a), a


def _scale(a):
    """a / 127 rounded once (a division by a Python number multiplies by its reciprocal on the GPU)."""
    return a.float() / torch.full_like(a, 127.0).float()


def _within(got, want, tol):
    err = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst ratio {(err / tol).max():.3g}"


# ------------------------------------------------------------------- rowquant --
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", [(1, 16), (3, 48), (2, 5, 512), (7, 528), (4, 1024), (5, 1040), (77, 2048),
                                   (3, 4112), (2, 8192), (2, 8208), (3, 16384)])
def test_rowquant_codes_and_scales_are_exact(shape, dt, cuda_dev):
    x = _acts(_gen(sum(shape)), shape, dt)
    x.view(-1, shape[-1])[0] = 0
    q, s = afb.rowquant_int8(x)
    want, a = _codes64(x.view(-1, shape[-1]))
    assert q.shape == x.shape and q.dtype == torch.int8 and s.shape == (x.numel() // shape[-1], 1)
    assert torch.equal(q.view(-1, shape[-1]).double(), want)
    assert torch.equal(s, _scale(a))


@pytest.mark.parametrize("dt", [BF, HF])
def test_rowquant_ties_go_to_even(dt, cuda_dev):
    # a = 127 * 2^e puts every n + 1/2 on a representable value
    for e in (-6, 0, 4):
        k = torch.arange(-64, 64, device=cuda_dev).double() + 0.5
        row = torch.cat([torch.tensor([127.0], device=cuda_dev).double(), k, torch.zeros(15, device=cuda_dev).double()])
        x = (row * 2.0**e).to(dt)[None]
        assert torch.equal(x.double(), row[None] * 2.0**e)
        q, _ = afb.rowquant_int8(x)
        assert torch.equal(q[0].double(), torch.round(row))


def test_rowquant_every_bf16_value(cuda_dev):
    """Rows of all finite values below each of several maxima, the largest finite one among them."""
    v = torch.arange(0, 0x7F80, device=cuda_dev).to(torch.int16).view(BF)
    for top in (1.0, 1.3359375, 2.0**-60, torch.finfo(BF).max, 1e36, 0.75):
        x = v[v.float() <= top]
        x = x[-8176:] if len(x) > 8176 else x
        x = torch.cat([x, torch.full((16 - len(x) % 16,), top, device=cuda_dev, dtype=BF)])[None]
        q, s = afb.rowquant_int8(torch.cat([x, -x]))
        want, a = _codes64(x)
        assert torch.equal(q[0].double(), want[0]) and torch.equal(q[1].double(), -want[0])
        assert torch.equal(s[0], _scale(a)[0])


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("K", [16, 2048, 16384])
def test_non_finite_rows_stay_visible(bad, K, cuda_dev):
    x = _acts(_gen(K), (5, K), BF)
    x[1, K - 1] = bad
    x[3, 0] = bad
    q, s = afb.rowquant_int8(x)
    assert not torch.isfinite(s[[1, 3]]).any() and not q[[1, 3]].any()
    want, _ = _codes64(x[[0, 2, 4]])
    assert torch.equal(q[[0, 2, 4]].double(), want)
    w = afb.quantize_weight_int8(_acts(_gen(1), (40, K), BF))
    y = afb.int8_linear(x, w)
    assert torch.isnan(y[[1, 3]]).all() and torch.isfinite(y[[0, 2, 4]].float()).all()
    assert torch.isnan(afb.int8_restore(q, s)[[1, 3]].float()).all()
    g = afb.gelu_int8(x)
    assert not torch.isfinite(g[3][[1, 3]]).any() and torch.isfinite(g[1][[0, 2, 4]]).all()
    dx = afb.gelu_int8_bwd(torch.ones_like(x), g[2], g[3])
    assert torch.isnan(dx[[1, 3]].float()).all() and torch.isfinite(dx[[0, 2, 4]].float()).all()
    dw = afb.int8_wgrad(torch.ones(5, 8, dtype=BF, device=cuda_dev), q, s)
    assert torch.isnan(dw.float()).all()


# --------------------------------------------------------------------- linear --
def _linear_case(M, N, K, dt, seed, bias):
    g = _gen(seed)
    x = _acts(g, (M, K), dt)
    w = afb.quantize_weight_int8((torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)).to(dt))
    b = torch.randn(N, generator=g, device="cuda").to(dt) if bias else None
    return x, w, b


def _check_linear(y, q64, s, w, b, dt):
    p = (q64 @ w.q.double().t()) * s.double() * w.s.double()
    want = p if b is None else p + b.double()
    mag = p.abs() if b is None else p.abs() + b.double().abs()
    _within(y, want, U[dt] * want.abs() + 2.0**-22 * mag + TINY[dt])


LINEAR = [(1, 16, 16), (6, 300, 4096), (7, 33, 8192), (1, 4097, 16384), (2, 5000, 144), (8, 2049, 4096), (1, 1, 16), (1, 2047, 2048), (2, 130, 144), (3, 7, 4112), (4, 96, 8192), (5, 128, 2064),
          (8, 257, 1024), (9, 64, 1040), (16, 127, 2048), (17, 129, 528), (33, 640, 256), (64, 63, 4096), (65, 1000, 272),
          (77, 2047, 1024), (128, 128, 128), (129, 255, 2032), (200, 256, 16384), (257, 513, 1040), (512, 2048, 2048),
          (1000, 33, 2048), (1537, 1030, 2064), (4096, 2048, 512), (4099, 3001, 1040), (1024, 6144, 272), (1000, 8192, 144),
          (2304, 5000, 528)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear_against_the_exact_product(M, N, K, dt, cuda_dev):
    x, w, b = _linear_case(M, N, K, dt, M + N + K, bias=(M + N) % 2 == 0)
    q64, a = _codes64(x)
    y = afb.int8_linear(x, w, b)
    assert y.shape == (M, N) and y.dtype == dt
    _check_linear(y, q64, _scale(a), w, b, dt)
    q, s = afb.rowquant_int8(x)
    assert torch.equal(afb.int8_linear((q, s), w, b, dt), y)  # both paths round alike


@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_extreme_codes_reach_the_largest_sum(M, cuda_dev):
    K, N = 131072, 144
    q = torch.full((M, K), 127, dtype=torch.int8, device=cuda_dev)
    q[::2] = -127
    wq = torch.full((N, K), -127, dtype=torch.int8, device=cuda_dev)
    s = torch.full((M, 1), 2.0**-20, device=cuda_dev)
    ws = torch.full((N,), 2.0**-10, device=cuda_dev)
    y = torch.ops.anima_flat_b200.int8_linear_codes(q, s, wq, ws, None, BF)
    sign = torch.where(torch.arange(M, device=cuda_dev) % 2 == 0, 1.0, -1.0)
    want = (sign * 127.0**2 * K * 2.0**-30)[:, None].expand(M, N)
    _within(y, want.double(), U[BF] * want.double().abs() + 2.0**-22 * want.double().abs())


def test_linear_leading_dims_and_empty(cuda_dev):
    x, w, _ = _linear_case(6, 48, 64, BF, 3, False)
    y = afb.int8_linear(x.view(2, 3, 64), w)
    assert y.shape == (2, 3, 48) and torch.equal(y.view(6, 48), afb.int8_linear(x, w))
    assert afb.int8_linear(x[:0], w).shape == (0, 48)
    assert afb.int8_linear((x[:0].to(torch.int8), torch.empty(0, 1, device=cuda_dev)), w).shape == (0, 48)


def test_strided_and_misaligned_inputs(cuda_dev):
    base = _acts(_gen(5), (40, 3 * 64), BF)
    _, w, _ = _linear_case(1, 56, 64, BF, 4, False)
    part = base[:, 64:128]  # a slice of a fused projection
    assert torch.equal(afb.int8_linear(part, w), afb.int8_linear(part.contiguous(), w))
    flat = base.flatten()[1 : 1 + 10 * 64].view(10, 64)  # 2 bytes past a 16-byte boundary
    assert torch.equal(afb.int8_linear(flat, w), afb.int8_linear(flat.clone(), w))
    wt = afb.Int8Weight(w.q.t().contiguous().t(), w.s)
    assert torch.equal(afb.int8_linear(part, wt), afb.int8_linear(part, w))
    b = torch.randn(57, device=cuda_dev).to(BF)[1:]
    assert torch.equal(afb.int8_linear(part, w, b), afb.int8_linear(part, w, b.clone()))


def test_on_another_stream(cuda_dev):
    x, w, b = _linear_case(300, 512, 1024, BF, 6, True)
    want = afb.int8_linear(x, w, b)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(3):
            got = afb.int8_linear(x, w, b)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


def test_linear_in_a_graph(cuda_dev):
    for M in (1, 50, 700):
        x, w, b = _linear_case(M, 520, 1024, BF, 7, True)
        out = torch.empty(M, 520, dtype=BF, device=cuda_dev)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            afb.int8_linear(x, w, b)
        torch.cuda.current_stream().wait_stream(st)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.copy_(afb.int8_linear(x, w, b))
        x2 = _acts(_gen(9), (M, 1024), BF)
        x.copy_(x2)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, afb.int8_linear(x2, w, b))


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (5, 48, 144), (8, 1040, 272), (77, 2048, 1024), (300, 1040, 528), (1000, 512, 2048)])
def test_linear_input_gradient(M, N, K, dt, cuda_dev):
    g = _gen(M + N)
    x = _acts(g, (M, K), dt).requires_grad_(True)
    w = afb.quantize_weight_int8((torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)).to(dt), backward=True)
    assert torch.equal(w.qt, w.q.t())
    dy = (0.1 * torch.randn(M, N, generator=g, device="cuda")).to(dt)
    y = afb.int8_linear(x, w)
    (dx,) = torch.autograd.grad(y, x, dy)
    # the definition: codes of the fp32 products dy * v, then the product
    gv = dy.float() * w.s
    a = gv.abs().amax(1, keepdim=True).clamp_min(1e-30)
    q = torch.round(gv * 127.0 / a)
    want = (q.double() @ w.q.double()) * (a / 127.0).double()
    _within(dx, want, U[dt] * want.abs() + 2.0**-22 * want.abs() + TINY[dt])
    # the exact derivative of y in x, which is linear: differences of any size give dy @ W;
    # off by half a code step of the gradient at most, for every channel
    true = gv.double() @ w.q.double()
    step = (a / 127.0).double() * 0.5 * w.q.double().abs().sum(0)
    _within(dx, true, 1.001 * step + U[dt] * true.abs() * 1.01 + U[dt] * step + TINY[dt])


# ----------------------------------------------------------------------- gelu --
def _gelu64(x):
    return x * torch.special.ndtr(x)


def _slope64(v):
    return torch.special.ndtr(v) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", [(1, 16), (3, 48), (2, 5, 528), (77, 2048), (9, 8192), (3, 16384)])
def test_gelu_codes_and_checkpoint(shape, dt, cuda_dev):
    x = (2.0 * torch.randn(*shape, generator=_gen(sum(shape)), device=cuda_dev)).to(dt)
    q, s, c, cs = afb.gelu_int8(x)
    cq, csc = afb.rowquant_int8(x)
    assert torch.equal(c, cq) and torch.equal(cs, csc)
    K = shape[-1]
    y = _gelu64(x.double()).view(-1, K)
    err = 2.0**-20 + 2.0**-12 * y.abs()
    top = y.abs().amax(1, keepdim=True)
    _within(s, top / 127.0, (2.0**-20 + 2.0**-12 * top) / 127.0 + 2.0**-23 * top / 127.0)
    _within(q.view(-1, K).double() * s.double(), y, 0.5001 * s.double() + 2 * err)


@pytest.mark.parametrize("K", [16, 512, 528, 1024, 2048, 4096, 8192, 8208, 16384])
def test_gelu_rows_without_a_large_positive_value(K, cuda_dev):
    """Rows whose largest |GELU| is not that of their largest input, beside rows where it is."""
    g = _gen(K)
    x = 2.0 * torch.randn(11, K, generator=g, device=cuda_dev)
    x[1] = -x[1].abs()
    x[3] *= 0.05
    x[4] = 0
    x[6] = -x[6].abs() * 0.01
    x[7] = -20.0
    x[9, : K - 1] = -x[9, : K - 1].abs()
    x[9, K - 1] = 0.2
    x = x.to(BF)
    q, s, c, cs = afb.gelu_int8(x)
    cq, csc = afb.rowquant_int8(x)
    assert torch.equal(c, cq) and torch.equal(cs, csc)
    y = _gelu64(x.double())
    top = y.abs().amax(1, keepdim=True)
    err = 2.0**-20 + 2.0**-12 * y.abs()
    _within(s, top.clamp_min(1e-30) / 127.0, (2.0**-20 + 2.0**-12 * top) / 127.0 + 2.0**-23 * top / 127.0)
    _within(q.double() * s.double(), y, 0.5001 * s.double() + 2 * err)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", [(1, 16), (3, 48), (2, 5, 528), (77, 2048), (9, 8192), (3, 16384)])
def test_gelu_backward_from_codes(shape, dt, cuda_dev):
    g = _gen(sum(shape))
    x = (2.0 * torch.randn(*shape, generator=g, device=cuda_dev)).to(dt)
    dy = torch.randn(*shape, generator=g, device=cuda_dev).to(dt)
    _, _, c, cs = afb.gelu_int8(x)
    dx = afb.gelu_int8_bwd(dy, c, cs)
    v = c.double() * cs.double().view(*shape[:-1], 1)
    want = dy.double() * _slope64(v)
    tol = U[dt] * want.abs() + 2.0**-18 * dy.double().abs() + TINY[dt]
    _within(dx, want, tol)
    # against differences of GELU in 64 bits at the checkpointed input
    d = 2.0**-13
    diff = dy.double() * (_gelu64(v + d) - _gelu64(v - d)) / (2 * d)
    _within(dx, diff, tol + 2.0**-20 * dy.double().abs())
    # the slope moves by at most 0.8 |x - v|, and |x - v| is half a step at most
    true = dy.double() * _slope64(x.double())
    half = 0.5001 * cs.double().view(*shape[:-1], 1)
    _within(dx, true, tol + (0.8 + U[dt]) * half * dy.double().abs())


def test_gelu_large_inputs(cuda_dev):
    x = torch.tensor([[-1e4, -50.0, -12.0, -6.0, -1.0, -0.0, 0.0, 1e-30, 1e-3, 0.5, 3.0, 6.0, 12.0, 50.0, 1e4, 0.0]],
                     device=cuda_dev).to(BF)
    q, s, c, cs = afb.gelu_int8(x)
    assert s.item() == pytest.approx(9984.0 / 127.0) and q[0, 14] == 127 and q[0, 0] == 0
    for k in range(16):  # one value a row: its code is the largest, the value is restored to rounding
        r = x[:, k : k + 1].expand(1, 16).contiguous()
        _, _, c, cs = afb.gelu_int8(r)
        dx = afb.gelu_int8_bwd(torch.ones_like(r), c, cs)
        want = _slope64(c.double() * cs.double())
        _within(dx, want, U[BF] * want.abs() + 2.0**-18)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", [(1, 16), (2, 5, 528), (300, 8192), (1, 16384)])
def test_restore(shape, dt, cuda_dev):
    x = _acts(_gen(8), shape, dt)
    q, s = afb.rowquant_int8(x)
    y = afb.int8_restore(q, s, dt)
    want = q.double() * s.double().view(*shape[:-1], 1)
    assert y.shape == x.shape and y.dtype == dt
    _within(y, want, (U[dt] + 2.0**-24) * want.abs() + TINY[dt])


def test_empty_tensors(cuda_dev):
    x = torch.empty(0, 64, dtype=BF, device=cuda_dev)
    q, s = afb.rowquant_int8(x)
    assert q.shape == (0, 64) and s.shape == (0, 1)
    assert afb.int8_restore(q, s).shape == (0, 64)
    q, s, c, cs = afb.gelu_int8(x)
    assert afb.gelu_int8_bwd(x, c, cs).shape == (0, 64)
    dw = afb.int8_wgrad(torch.empty(0, 8, dtype=BF, device=cuda_dev), q, s)
    assert dw.shape == (8, 64) and not dw.any()


# ---------------------------------------------------------------------- wgrad --
WGRAD = [(1, 8, 16), (2, 16, 48), (7, 4, 144), (63, 16, 128), (64, 8, 256), (65, 32, 272), (100, 3, 2048), (257, 64, 1040),
         (300, 72, 112), (1000, 16, 2048), (1000, 128, 528), (513, 130, 256), (777, 257, 400), (2048, 512, 512),
         (4096, 16, 8192), (4097, 264, 1040), (1030, 1000, 2048), (200, 2800, 2064), (1000, 1040, 8208), (65, 10000, 528), (130, 24, 8192)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T,N,K", WGRAD)
def test_wgrad_against_the_exact_sum(T, N, K, dt, cuda_dev):
    g = _gen(T + N + K)
    q, s = afb.rowquant_int8(_acts(g, (T, K), dt))
    dy = (0.1 * torch.randn(T, N, generator=g, device=cuda_dev)).to(dt)
    dw = afb.int8_wgrad(dy, q, s)
    x = q.double() * s.double()
    want = dy.double().t() @ x
    mag = dy.double().abs().t() @ x.abs()
    assert dw.shape == (N, K) and dw.dtype == dt
    _within(dw, want, (U[dt] + T * 2.0**-23) * mag + U[dt] * want.abs() + TINY[dt] * (1 + T))
    assert torch.equal(dw, afb.int8_wgrad(dy, q, s))  # one fixed order


def test_wgrad_leading_dims_and_strides(cuda_dev):
    g = _gen(11)
    q, s = afb.rowquant_int8(_acts(g, (3, 40, 96), BF))
    dy = torch.randn(3, 40, 48, generator=g, device=cuda_dev).to(BF)
    want = afb.int8_wgrad(dy.view(120, 48), q.view(120, 96), s)
    assert torch.equal(afb.int8_wgrad(dy, q, s), want)
    wide = torch.cat([dy, dy], -1)
    assert torch.equal(afb.int8_wgrad(wide[..., 48:], q, s), want)


def test_wgrad_padded_tokens_do_not_matter(cuda_dev):
    """Rows of zero gradient contribute nothing, whatever their codes."""
    g = _gen(12)
    q, s = afb.rowquant_int8(_acts(g, (200, 256), BF))
    dy = torch.randn(200, 32, generator=g, device=cuda_dev).to(BF)
    dy[100:] = 0
    assert torch.equal(afb.int8_wgrad(dy, q, s)[:, :16].isfinite(), torch.ones(32, 16, dtype=torch.bool, device=cuda_dev))
    a, b = afb.int8_wgrad(dy, q, s), afb.int8_wgrad(dy[:100], q[:100], s[:100])
    mag = dy.double().abs().t() @ (q.double() * s.double()).abs()
    _within(a, b.double(), (2 * U[BF] + 200 * 2.0**-22) * mag)

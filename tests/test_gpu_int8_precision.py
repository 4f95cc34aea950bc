"""Accuracy of the 8-bit operators where a value held in 16 bits on the way would show.

u is the half-step of the 16-bit type, 2^-8 (bf16) or 2^-11 (fp16).

int8_wgrad: dy s is formed in fp32 and held as two bf16 values, within 2^-16 of
it, and two products a token go into an fp32 sum, whose additions may cut off
2^-23 of it: u |dw| + (2^-16 + T 2^-22) sum |dy x|.  With one token that is one
rounding of the exact result, where a rounding of q s on the way would add
another u; over many tokens the error's norm is that of rounding the exact
result.

gelu_int8: below zero the error function's approximation (A&S 7.1.26) is within
0.0036 of 1 + erf down to -6, and the special-function unit's exponential and
reciprocal within 2^-16 there: 2^-8 of GELU in all.

int8_lora_mlp: an adapter's gradients are products with the scaling, each rounded
once from an fp32 sum: u |db| + T 2^-22 sum of magnitudes for b; for a over one
token u of the inner gradient and u of the result.
"""

from __future__ import annotations

import pytest
import torch

import anima_flat_b200 as afb

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0**-8, HF: 2.0**-11}
TINY = {BF: 2.0**-133, HF: 2.0**-25}


def _codes(g, T, K):
    q = torch.randint(-127, 128, (T, K), dtype=torch.int8, device="cuda", generator=g)
    q[:, 0] = 127
    return q


def _check_wgrad(dy, q, s, T):
    dw = afb.int8_wgrad(dy, q, s)
    x = q.double() * s.double()
    want, mag = dy.double().t() @ x, dy.double().abs().t() @ x.abs()
    tol = U[dy.dtype] * want.abs() + (2.0**-16 + T * 2.0**-22) * mag + TINY[dy.dtype]
    assert torch.isfinite(dw).all()
    err = (dw.double() - want).abs()
    assert (err <= tol).all(), f"{int((err > tol).sum())} of {err.numel()} off, worst {(err / tol).max():.3g}"
    return dw, want


# adapters' columns, padded rows, one tile of 128 columns, single tiles, clusters and pairs
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T,N,K", [(1, 4, 144), (1, 16, 2048), (2, 17, 272), (1, 64, 256), (3, 100, 272), (1, 128, 528),
                                   (1, 300, 1040), (1, 4096, 2048), (2, 4001, 2064), (70, 16, 8192), (66, 4096, 512)])
def test_wgrad_rounds_once(T, N, K, dt, cuda_dev):
    g = torch.Generator(device="cuda").manual_seed(T + N + K)
    s = 2.0**-7 * (0.5 + torch.rand(T, 1, device="cuda", generator=g))
    dy = (0.1 * torch.randn(T, N, device="cuda", generator=g)).to(dt)
    _check_wgrad(dy, _codes(g, T, K), s, T)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T,N,K", [(512, 16, 2048), (1000, 64, 528), (512, 128, 1024), (700, 2048, 2048), (512, 1000, 1040)])
def test_wgrad_error_is_that_of_rounding_the_result(T, N, K, dt, cuda_dev):
    g = torch.Generator(device="cuda").manual_seed(T + N)
    s = 2.0**-7 * (0.5 + torch.rand(T, 1, device="cuda", generator=g))
    dy = (0.1 * torch.randn(T, N, device="cuda", generator=g)).to(dt)
    dw, want = _check_wgrad(dy, _codes(g, T, K), s, T)
    # a rounding of q s would add an error of the same size: 1.41 times the norm
    assert (dw.double() - want).norm() <= 1.1 * (want.to(dt).double() - want).norm()


@pytest.mark.parametrize("N", [16, 64, 128, 1030, 4096])
@pytest.mark.parametrize("top", [1e5, 1e-5, 1e-9])
def test_wgrad_fp16_beside_codes_of_any_range(N, top, cuda_dev):
    """Rows whose largest value fp16 does not hold, or holds in a few bits, as codes with fp32 scales do."""
    T, K = 130, 512
    g = torch.Generator(device="cuda").manual_seed(N)
    s = (top / 127.0) * (0.5 + torch.rand(T, 1, device="cuda", generator=g))
    dy = ((1e-3 if top > 1 else 1e3) * torch.randn(T, N, device="cuda", generator=g)).to(HF)
    _check_wgrad(dy, _codes(g, T, K), s, T)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("N", [16, 100, 4096])
def test_wgrad_infinities_and_nans_stay_what_they_are(N, dt, cuda_dev):
    T, K = 70, 512
    g = torch.Generator(device="cuda").manual_seed(N)
    q, s = _codes(g, T, K), torch.rand(T, 1, device="cuda", generator=g) + 0.5
    q[3, 5] = 0
    dy = torch.randn(T, N, device="cuda", generator=g).to(dt)
    dy[3, 1], dy[9, 2], dy[11, 3] = float("inf"), float("-inf"), float("nan")
    dw, want = afb.int8_wgrad(dy, q, s).double(), dy.double().t() @ (q.double() * s.double())
    assert torch.equal(torch.isnan(dw), torch.isnan(want)) and torch.isnan(want[1, 5])
    assert torch.equal(torch.isinf(dw).logical_and(dw > 0), torch.isinf(want).logical_and(want > 0))
    assert torch.equal(torch.isinf(dw).logical_and(dw < 0), torch.isinf(want).logical_and(want < 0))


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("K", [16, 528, 2048, 8192, 16384])
def test_gelu_rows_far_below_zero(K, dt, cuda_dev):
    """Rows whose largest |GELU| is small: scale and codes to a fraction of the row's own maximum."""
    g = torch.Generator(device="cuda").manual_seed(K)
    x = -4.0 - 2.0 * torch.rand(12, K, device="cuda", generator=g)
    x[0], x[1], x[2] = -5.5, -6.0, -4.0
    x[3] = -1.0 - 5.0 * torch.rand(K, device="cuda", generator=g)
    x[4] = -6.0 * torch.rand(K, device="cuda", generator=g)
    x[5] = x[4] * 2.0**-10
    x[6, :8] = 0.0
    x[7] = 0.33
    x = x.to(dt).clamp_min(-6.0)
    q, s, c, cs = afb.gelu_int8(x)
    want = x.double() * torch.special.ndtr(x.double())
    top = want.abs().amax(1, keepdim=True)
    assert ((s.double() * 127.0 - top).abs() <= 2.0**-8 * top).all()
    assert ((q.double() * s.double() - want).abs() <= 0.5001 * s.double() + 2.0**-8 * top).all()
    assert q.abs().amax(1).eq(127).all()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T", [1, 70])
def test_adapter_gradients_round_once(T, dt, cuda_dev):
    K, H, N, r, scaling = 256, 528, 272, 64, 1.0 / 3.0
    g = torch.Generator(device="cuda").manual_seed(T)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    up = afb.quantize_weight_int8((rn(H, K) / K**0.5).to(dt), backward=True)
    down = afb.quantize_weight_int8((rn(N, H) / H**0.5).to(dt), backward=True)
    x, dy = rn(T, K).to(dt), rn(T, N).to(dt)
    a1, b1, a2, b2 = (t.to(dt).requires_grad_(True) for t in (rn(r, K) / 16, rn(H, r) / 8, rn(r, H) / 16, rn(N, r) / 8))
    y = afb.int8_lora_mlp(x, up, down, afb.LoRA(a1, b1), afb.LoRA(a2, b2), scaling)
    da2, db2 = torch.autograd.grad(y, (a2, b2), dy)
    with torch.no_grad():  # the inner values, as the forward pass has them
        h = afb.int8_linear(afb.rowquant_int8(x), up, dtype=dt).addmm_(x @ a1.t(), b1.t(), alpha=scaling)
        gq, gs, _, _ = afb.gelu_int8(h)
        t2 = (afb.int8_restore(gq, gs, dt) @ a2.t()).double()
    u, d = U[dt], dy.double()
    want, mag = scaling * (d.t() @ t2), scaling * (d.t().abs() @ t2.abs())
    assert ((db2.double() - want).abs() <= u * want.abs() + T * 2.0**-22 * mag + TINY[dt]).all()
    if T == 1:
        inner, imag = scaling * (d @ b2.double()), scaling * (d.abs() @ b2.double().abs())
        v = gq.double() * gs.double()
        want, mag = inner.t() @ v, imag.t() @ v.abs()
        tol = u * want.abs() + (1 + u) * (u * want.abs() + N * 2.0**-23 * mag) + 2.0**-15 * want.abs() + TINY[dt]
        assert ((da2.double() - want).abs() <= tol).all()

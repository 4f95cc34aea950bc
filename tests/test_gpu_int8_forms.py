"""Sizes on either side of the choice between single CTAs, clusters and pairs of CTAs."""

from __future__ import annotations

import pytest
import torch

import anima_flat_b200 as afb

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0**-8, HF: 2.0**-11}


def _codes(rows, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-127, 128, (rows, K), dtype=torch.int8, device="cuda", generator=g)
    return q, torch.rand(rows, 1, device="cuda", generator=g) + 0.5, g


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(200, 1024, 4096), (256, 2048, 2048), (300, 2047, 2048), (512, 2048, 8192),
                                   (700, 1000, 1040), (1024, 1024, 1024), (1000, 1500, 8192), (1500, 3000, 512),
                                   (2048, 1024, 256), (8192, 256, 2048), (4096, 257, 1040)])
def test_product_bits_do_not_depend_on_the_rows_beside(M, N, K, dt, cuda_dev):
    """The integer sum is exact, so 100 rows alone (single CTAs) give the bits they have among M."""
    q, s, g = _codes(M, K, M + N)
    wq, ws, _ = _codes(N, K, K)
    w = afb.Int8Weight(wq, ws.flatten() * 2.0**-20)
    b = torch.randn(N, device="cuda", generator=g).to(dt)
    y = afb.int8_linear((q, s), w, b, dt)
    for r in range(0, M, 100):
        assert torch.equal(y[r : r + 100], afb.int8_linear((q[r : r + 100], s[r : r + 100]), w, b, dt))


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T,N,K", [(1000, 300, 1024), (1024, 1024, 1024), (1024, 512, 2048), (700, 2048, 1040),
                                   (500, 2047, 2048), (130, 4096, 512), (64, 4096, 2048), (2000, 2000, 2000)])
def test_wide_weight_gradient(T, N, K, dt, cuda_dev):
    q, s, g = _codes(T, K, T + N)
    s = s * 2.0**-7
    dy = (0.1 * torch.randn(T, N, device="cuda", generator=g)).to(dt)
    dw = afb.int8_wgrad(dy, q, s)
    x = q.double() * s.double()
    want, mag = dy.double().t() @ x, dy.double().abs().t() @ x.abs()
    # each q s rounded once to the type, T sums in 32 bits, one rounding of the result
    tol = (U[dt] + T * 2.0**-23) * mag + U[dt] * want.abs() + 2.0**-24 * (1 + T)
    assert ((dw.double() - want).abs() <= tol).all()
    assert torch.equal(dw, afb.int8_wgrad(dy, q, s))

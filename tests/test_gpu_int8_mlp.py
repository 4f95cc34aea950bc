"""The MLP on 8-bit weights, checkpoints and adapters, and the example that trains it.

Bound against the exact MLP on the quantized weights: every quantization of a
normal row of K values adds noise of amax / (127 sqrt 12) = 0.9% of its norm at
amax = 4 sigma, 1.5% after GELU, whose values are further from their maximum; at
most four of them meet in one result: 6% of its norm.
"""

from __future__ import annotations

import importlib.util

import pytest
import torch

import anima_flat_b200 as afb
from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


def _case(T, K, H, N, r, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    up = afb.quantize_weight_int8((rn(H, K) / K**0.5).to(dt), backward=True)
    down = afb.quantize_weight_int8((rn(N, H) / H**0.5).to(dt), backward=True)
    l1 = afb.LoRA((rn(r, K) / K**0.5).to(dt), (0.3 * rn(H, r)).to(dt))
    l2 = afb.LoRA((rn(r, H) / H**0.5).to(dt), (0.3 * rn(N, r)).to(dt))
    return rn(T, K).to(dt), up, down, l1, l2, (0.1 * rn(T, N)).to(dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,H,N,r", [(1, 64, 128, 64, 4), (77, 256, 1040, 272, 16), (300, 512, 2048, 512, 8)])
def test_values_and_gradients(T, K, H, N, r, dt, cuda_dev):
    x, up, down, l1, l2, dy = _case(T, K, H, N, r, dt)
    leaves = [t.requires_grad_(True) for t in (x, *l1, *l2)]
    y = afb.int8_lora_mlp(x, up, down, l1, l2, 0.5)
    grads = torch.autograd.grad(y, leaves, dy)
    f = [t.detach().double().requires_grad_(True) for t in leaves]
    w1, w2 = (w.q.double() * w.s.double()[:, None] for w in (up, down))
    h = f[0] @ w1.t() + 0.5 * (f[0] @ f[1].t()) @ f[2].t()
    g = h * torch.special.ndtr(h)
    want = g @ w2.t() + 0.5 * (g @ f[3].t()) @ f[4].t()
    for a, b in zip((y, *grads), (want, *torch.autograd.grad(want, f, dy.double()))):
        assert a.shape == b.shape and a.dtype == dt
        assert (a.double() - b).norm() <= 0.06 * b.norm()


def test_keeps_no_16_bit_activation(cuda_dev):
    x, up, down, l1, l2, dy = _case(64, 256, 1024, 256, 8, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, *l1, *l2)]
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append((t.dtype, tuple(t.shape))) or t, lambda t: t):
        y = afb.int8_lora_mlp(x, up, down, l1, l2)
    wide = [s for d, s in kept if d == torch.bfloat16 and s[0] == 64]
    assert wide == [(64, 8), (64, 8)]  # the adapters' inner values alone
    assert {(torch.int8, (64, 256)), (torch.int8, (64, 1024))} <= set(kept)
    torch.autograd.grad(y, leaves, dy)


def test_leading_dims_and_frozen_input(cuda_dev):
    x, up, down, l1, l2, dy = _case(24, 64, 128, 64, 8, torch.bfloat16)
    a = afb.int8_lora_mlp(x, up, down, l1, l2)
    b = afb.int8_lora_mlp(x.view(2, 12, 64), up, down, l1, l2)
    assert b.shape == (2, 12, 64) and torch.equal(a, b.view(24, 64))
    l1 = afb.LoRA(l1.a.requires_grad_(True), l1.b)
    (ga,) = torch.autograd.grad(afb.int8_lora_mlp(x, up, down, l1, l2), [l1.a], dy)
    assert ga.shape == l1.a.shape


def test_refusals(cuda_dev):
    x, up, down, l1, l2, _ = _case(8, 64, 128, 64, 8, torch.bfloat16)
    for args in ((x, afb.Int8Weight(up.q, up.s), down, l1, l2), (x, up, down, l2, l1), (x, down, up, l1, l2),
                 (x.half(), up, down, l1, l2), (x.cpu(), up, down, l1, l2)):
        with pytest.raises(ValueError):
            afb.int8_lora_mlp(*args)
    with pytest.raises(ValueError):
        afb.int8_linear_dx(x, afb.Int8Weight(up.q, up.s))
    with pytest.raises(ValueError):
        afb.int8_linear_dx(x, up)


def test_example_learns(cuda_dev):
    spec = importlib.util.spec_from_file_location("int8_lora_block", ROOT / "examples" / "int8_lora_block.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(tokens=512, steps=25, rank=8, dim=256, hidden=512, verbose=False)
    assert losses[-1] < 0.5 * losses[0]


def test_a_long_chain_of_calls(cuda_dev):
    """Several hundred quantise-multiply calls queued without a wait between them."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(8192, 512, generator=g, device="cuda").to(torch.bfloat16)
    w = afb.quantize_weight_int8(torch.randn(5120, 512, generator=g, device="cuda").to(torch.bfloat16))
    want = afb.int8_linear(x, w)
    q, s = afb.rowquant_int8(x)
    dw = afb.int8_wgrad(want, q, s)
    for _ in range(400):
        y = afb.int8_linear(x, w)
    for _ in range(100):
        dw2 = afb.int8_wgrad(y, q, s)
    assert torch.equal(y, want) and torch.equal(dw, dw2)

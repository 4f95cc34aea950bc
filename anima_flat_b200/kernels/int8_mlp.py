"""An MLP on 8-bit weights with low-rank adapters and 8-bit checkpoints.

No counterpart in the reference, whose LoRA training keeps its layers and their
activations in bf16.  ``int8_lora_mlp`` runs the 8-bit ops together as a training
step would:

    h = x W1' + t1 b1' c,   t1 = x a1'          W1, W2 frozen, in 8 bits
    y = g W2' + t2 b2' c,   g = GELU(h),  t2 = g a2'

What the forward pass keeps for the backward pass is what the products read: the
codes of x and of g, and the codes of h, one byte an element each, instead of
three bf16 activations.  The adapters' small products are plain matrix products.

Every product is summed in 32 bits or exactly and rounded once to the activations'
type, t1, t2 and their gradients too, as separate layers of that type do; an
adapter's part is added to the rounded product of its layer, and the sum rounded.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .common import _check_same_device
from .int8 import (
    Int8Weight,
    _check_cols,
    _check_weight,
    gelu_int8,
    gelu_int8_bwd,
    int8_linear,
    int8_linear_dx,
    int8_restore,
    int8_wgrad,
    rowquant_int8,
)

__all__ = ["LoRA", "int8_lora_mlp"]


class LoRA(NamedTuple):
    """Low-rank factors of one layer: ``a`` ``[r, K]`` and ``b`` ``[N, r]``."""

    a: torch.Tensor
    b: torch.Tensor


def _scaled_product(a, b, scaling):
    """``scaling * (a @ b)``, rounded once."""
    return a.new_empty((a.shape[0], b.shape[1])).addmm_(a, b, beta=0, alpha=scaling)


def _forward(x, a1, b1, a2, b2, w1, w2, scaling):
    """The output, and the activations that the backward pass reads."""
    rows = x.reshape(-1, x.shape[-1])
    q, s = rowquant_int8(rows)
    t1 = rows @ a1.t()
    h = int8_linear((q, s), w1, dtype=x.dtype).addmm_(t1, b1.t(), alpha=scaling)
    gq, gs, c, cs = gelu_int8(h)
    t2 = int8_restore(gq, gs, x.dtype) @ a2.t()
    y = int8_linear((gq, gs), w2, dtype=x.dtype).addmm_(t2, b2.t(), alpha=scaling)
    return y.view(*x.shape[:-1], y.shape[-1]), (q, s, c, cs, gq, gs, t1, t2)


class _MlpFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a1, b1, a2, b2, w1, w2, scaling):
        y, kept = _forward(x, a1, b1, a2, b2, w1, w2, scaling)
        ctx.save_for_backward(*kept, a1, b1, a2, b2, *w1, *w2)
        ctx.scaling = scaling
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        q, s, c, cs, gq, gs, t1, t2, a1, b1, a2, b2, *w = ctx.saved_tensors
        w1, w2 = Int8Weight(*w[:3]), Int8Weight(*w[3:])
        shape = (*dy.shape[:-1], q.shape[-1])
        dy = dy.reshape(-1, dy.shape[-1])
        dt2 = _scaled_product(dy, b2, ctx.scaling)
        db2 = _scaled_product(dy.t(), t2, ctx.scaling)
        da2 = int8_wgrad(dt2, gq, gs)
        dh = gelu_int8_bwd(int8_linear_dx(dy, w2).addmm_(dt2, a2), c, cs)
        dt1 = _scaled_product(dh, b1, ctx.scaling)
        db1 = _scaled_product(dh.t(), t1, ctx.scaling)
        da1 = int8_wgrad(dt1, q, s)
        dx = int8_linear_dx(dh, w1).addmm_(dt1, a1).view(shape) if ctx.needs_input_grad[0] else None
        return dx, da1, db1, da2, db2, None, None, None


def int8_lora_mlp(
    x: torch.Tensor, up: Int8Weight, down: Int8Weight, lora_up: LoRA, lora_down: LoRA, scaling: float = 1.0
) -> torch.Tensor:
    """MLP (up, GELU, down) on frozen 8-bit weights with low-rank adapters.

    Differentiable in ``x`` and the adapters' factors; activations are kept for
    the backward pass in 8 bits.

    Args:
        x: Tokens, shape ``[..., K]`` bf16 or fp16.
        up: Quantized weight ``[H, K]`` with its transposed codes.
        down: Quantized weight ``[N, H]`` with its transposed codes.
        lora_up: Factors ``[r, K]`` and ``[H, r]`` of the dtype of ``x``.
        lora_down: Factors ``[r, H]`` and ``[N, r]`` of the dtype of ``x``.
        scaling: Factor of both adapters' contributions.

    Returns:
        ``[..., N]``, dtype of ``x``.

    Raises:
        ValueError: On tensors off CUDA, weights without transposed codes, or
            unsupported dtypes or shapes.
        RuntimeError: Inside ``torch.jit.trace`` where a gradient is asked for.
    """
    _check_same_device(x, *up, *down, *lora_up, *lora_down)
    for name, w, lora, K in (("up", up, lora_up, x.shape[-1]), ("down", down, lora_down, up.q.shape[0])):
        _check_weight(w.q, w.s, None, K, x.dtype)
        N, r = w.q.shape[0], lora.a.shape[0]
        _check_cols(f"the {name} weight's channels", w.q.t())
        if w.qt is None or w.qt.shape != (K, N):
            raise ValueError(f"{name} needs its transposed codes: quantize_weight_int8(w, backward=True)")
        if lora.a.shape != (r, K) or lora.b.shape != (N, r) or lora.a.dtype != x.dtype or lora.b.dtype != x.dtype:
            raise ValueError(f"lora_{name} must be {x.dtype} [r, {K}] and [{N}, r], got "
                             f"{lora.a.dtype} {list(lora.a.shape)} and {lora.b.dtype} {list(lora.b.shape)}")
    args = (x, *lora_up, *lora_down, up, down, float(scaling))
    if not torch.is_grad_enabled() or not any(t.requires_grad for t in args[:5]):
        return _forward(*args)[0]
    if torch.jit.is_tracing():
        raise RuntimeError("int8_lora_mlp has no traced backward pass: trace it under torch.no_grad()")
    return _MlpFn.apply(*args)

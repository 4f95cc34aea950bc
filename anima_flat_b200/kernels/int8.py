"""8-bit integer linear layers and 8-bit activation checkpoints.

No counterpart in the reference, whose 8-bit path is FP8 and serves only.

``rowquant_int8`` gives a tensor's rows as codes and a scale per row:

    a = max(max|x|, 1e-30),  s = a / 127,  q = rint(127 x / a)  (half to even)

A row that holds an infinity or a NaN gets that as its scale and zero codes, so
all that is computed from it is NaN.  ``int8_linear`` multiplies such codes by a
weight quantised in the same way along its rows (``quantize_weight_int8``):

    y[m, n] = (sum_k q[m, k] w[n, k]) * s[m] * v[n] + bias[n]

with an exact integer sum.  Its input gradient is the same product, of the
codes of ``dy * v`` with the transposed weight codes.

The codes are also the activation's checkpoint: ``int8_wgrad`` forms a weight
gradient (of a full weight, or of a low-rank adapter's first factor) straight
from them, ``int8_restore`` gives the values back, and ``gelu_int8`` emits the
codes of GELU(x) for the next product together with those of x, from which
``gelu_int8_bwd`` forms the activation's gradient.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .._lib import call
from .common import HALF_TYPES, _check_half, _check_same_device, _dense, _stream

__all__ = [
    "Int8Weight",
    "gelu_int8",
    "gelu_int8_bwd",
    "int8_linear",
    "int8_restore",
    "int8_wgrad",
    "quantize_weight_int8",
    "rowquant_int8",
]

F32 = torch.float32
I8 = torch.int8


class Int8Weight(NamedTuple):
    """A weight ``[N, K]`` as 8-bit codes with a scale per output channel.

    ``qt`` holds the same codes transposed, ``[K, N]``: the input gradient's
    product needs them, inference does not.
    """

    q: torch.Tensor
    s: torch.Tensor
    qt: torch.Tensor | None = None


# ------------------------------------------------------------------ launches --
def _quant(x: torch.Tensor, cols: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    K = x.shape[-1]
    rows = x.numel() // K
    q = torch.empty(x.shape, dtype=I8, device=x.device)
    s = torch.empty((rows, 1), dtype=F32, device=x.device)
    call("afb_rowquant_int8", x.data_ptr(), None if cols is None else cols.data_ptr(), q.data_ptr(),
         s.data_ptr(), rows, K, HALF_TYPES[x.dtype], _stream(x))
    return q, s


def _product(q, s, wq, ws, bias, dtype):
    K, N = q.shape[-1], wq.shape[0]
    y = torch.empty((*q.shape[:-1], N), dtype=dtype, device=q.device)
    call("afb_int8_linear", q.data_ptr(), s.data_ptr(), wq.data_ptr(), ws.data_ptr(),
         None if bias is None else bias.data_ptr(), y.data_ptr(), q.numel() // K, N, K,
         HALF_TYPES[dtype], _stream(q))
    return y


# ----------------------------------------------------------------- custom ops --
@torch.library.custom_op("anima_flat_b200::rowquant_int8", mutates_args=())
def _rowquant_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _quant(x)


@_rowquant_int8.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=I8), x.new_empty((x.numel() // x.shape[-1], 1), dtype=F32)


@torch.library.custom_op("anima_flat_b200::int8_linear_codes", mutates_args=())
def _int8_linear_codes(
    q: torch.Tensor, s: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, bias: torch.Tensor | None,
    dtype: torch.dtype,
) -> torch.Tensor:
    return _product(q, s, wq, ws, bias, dtype)


@_int8_linear_codes.register_fake
def _(q, s, wq, ws, bias, dtype):
    return q.new_empty((*q.shape[:-1], wq.shape[0]), dtype=dtype)


@torch.library.custom_op("anima_flat_b200::int8_linear", mutates_args=())
def _int8_linear(
    x: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, wqt: torch.Tensor | None,
    bias: torch.Tensor | None,
) -> torch.Tensor:
    q, s = _quant(x)
    return _product(q, s, wq, ws, bias, x.dtype)


@_int8_linear.register_fake
def _(x, wq, ws, wqt, bias):
    return x.new_empty((*x.shape[:-1], wq.shape[0]))


@torch.library.custom_op("anima_flat_b200::int8_linear_bwd", mutates_args=())
def _int8_linear_bwd(dy: torch.Tensor, ws: torch.Tensor, wqt: torch.Tensor) -> torch.Tensor:
    dy = _dense(dy)
    q, s = _quant(dy, ws)
    one = torch.ones(wqt.shape[0], dtype=F32, device=dy.device)
    return _product(q, s, wqt, one, None, dy.dtype)


@_int8_linear_bwd.register_fake
def _(dy, ws, wqt):
    return dy.new_empty((*dy.shape[:-1], wqt.shape[0]))


def _int8_linear_setup(ctx, inputs, output):
    _, _, ws, wqt, _ = inputs
    ctx.save_for_backward(ws, wqt)


def _int8_linear_backward(ctx, dy):
    ws, wqt = ctx.saved_tensors
    return _int8_linear_bwd(dy, ws, wqt), None, None, None, None


torch.library.register_autograd(
    "anima_flat_b200::int8_linear", _int8_linear_backward, setup_context=_int8_linear_setup
)


@torch.library.custom_op("anima_flat_b200::gelu_int8", mutates_args=())
def _gelu_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    K = x.shape[-1]
    rows = x.numel() // K
    q, c = torch.empty(x.shape, dtype=I8, device=x.device), torch.empty(x.shape, dtype=I8, device=x.device)
    s, cs = (torch.empty((rows, 1), dtype=F32, device=x.device) for _ in range(2))
    call("afb_gelu_int8", x.data_ptr(), q.data_ptr(), s.data_ptr(), c.data_ptr(), cs.data_ptr(), rows, K,
         HALF_TYPES[x.dtype], _stream(x))
    return q, s, c, cs


@_gelu_int8.register_fake
def _(x):
    rows = x.numel() // x.shape[-1]
    return (x.new_empty(x.shape, dtype=I8), x.new_empty((rows, 1), dtype=F32),
            x.new_empty(x.shape, dtype=I8), x.new_empty((rows, 1), dtype=F32))


@torch.library.custom_op("anima_flat_b200::gelu_int8_bwd", mutates_args=())
def _gelu_int8_bwd(dy: torch.Tensor, c: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    dx = torch.empty_like(dy)
    K = dy.shape[-1]
    call("afb_gelu_int8_bwd", dy.data_ptr(), c.data_ptr(), cs.data_ptr(), dx.data_ptr(), dy.numel() // K, K,
         HALF_TYPES[dy.dtype], _stream(dy))
    return dx


@_gelu_int8_bwd.register_fake
def _(dy, c, cs):
    return torch.empty_like(dy)


@torch.library.custom_op("anima_flat_b200::int8_restore", mutates_args=())
def _int8_restore(q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    y = torch.empty(q.shape, dtype=dtype, device=q.device)
    K = q.shape[-1]
    call("afb_int8_restore", q.data_ptr(), s.data_ptr(), y.data_ptr(), q.numel() // K, K, HALF_TYPES[dtype],
         _stream(q))
    return y


@_int8_restore.register_fake
def _(q, s, dtype):
    return q.new_empty(q.shape, dtype=dtype)


@torch.library.custom_op("anima_flat_b200::int8_wgrad", mutates_args=())
def _int8_wgrad(dy: torch.Tensor, q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    N, K = dy.shape[-1], q.shape[-1]
    dw = torch.empty((N, K), dtype=dy.dtype, device=dy.device)
    call("afb_int8_wgrad", dy.data_ptr(), q.data_ptr(), s.data_ptr(), dw.data_ptr(), q.numel() // K, N, K,
         HALF_TYPES[dy.dtype], _stream(dy))
    return dw


@_int8_wgrad.register_fake
def _(dy, q, s):
    return dy.new_empty((dy.shape[-1], q.shape[-1]))


# --------------------------------------------------------------------- checks --
def _check_cols(what: str, t: torch.Tensor, most: int = 16384) -> None:
    K = t.shape[-1] if t.ndim else 0
    if K < 16 or K % 16 or K > most:
        raise ValueError(f"the last dimension of {what} must be a multiple of 16 in [16, {most}], got {K}")


def _check_codes(q: torch.Tensor, s: torch.Tensor) -> None:
    if q.dtype != I8 or s.dtype != F32:
        raise ValueError(f"codes must be torch.int8 with torch.float32 scales, got {q.dtype} and {s.dtype}")
    _check_cols("the codes", q)
    if s.numel() * q.shape[-1] != q.numel():
        raise ValueError(f"one scale per row of the codes is needed: {list(q.shape)} and {list(s.shape)}")


def _check_weight(weight: Int8Weight, K: int) -> None:
    q, s, qt = weight
    if q.dtype != I8 or q.ndim != 2 or q.shape[1] != K or not q.shape[0]:
        raise ValueError(f"the weight's codes must be torch.int8 [N, {K}], got {q.dtype} {list(q.shape)}")
    if s.dtype != F32 or s.numel() != q.shape[0]:
        raise ValueError(f"the weight's scales must be torch.float32 [{q.shape[0]}], got {s.dtype} {list(s.shape)}")
    if qt is not None and (qt.dtype != I8 or qt.shape != (K, q.shape[0])):
        raise ValueError(f"the transposed codes must be torch.int8 [{K}, {q.shape[0]}]")


# --------------------------------------------------------------------- public --
def rowquant_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantize tokens to 8-bit integers with a scale per token.

    Args:
        x: Tokens, shape ``[..., K]`` bf16 or fp16, K a multiple of 16 up to 16384.

    Returns:
        ``(q, s)``: the codes, int8, shape of ``x``, and their float32 scales ``[rows, 1]``.

    Raises:
        ValueError: If ``x`` is not on CUDA or a dtype/shape is unsupported.
    """
    _check_same_device(x)
    _check_half("x", x)
    _check_cols("x", x)
    return _rowquant_int8(_dense(x))


def quantize_weight_int8(w: torch.Tensor, backward: bool = False) -> Int8Weight:
    """Quantize a weight ``[N, K]`` to 8-bit integers with a scale per output channel.

    Args:
        w: Weight, shape ``[N, K]`` bf16 or fp16, K a multiple of 16 up to 16384.
        backward: Keep the transposed codes too, for the input gradient (N a multiple of 16).

    Raises:
        ValueError: If ``w`` is not on CUDA or a dtype/shape is unsupported.
    """
    if w.ndim != 2:
        raise ValueError(f"expected a weight [N, K], got {list(w.shape)}")
    q, s = rowquant_int8(w.detach())
    if backward:
        _check_cols("the transposed weight", q.t())
    return Int8Weight(q, s.flatten(), q.t().contiguous() if backward else None)


def int8_linear(
    x: torch.Tensor | tuple[torch.Tensor, torch.Tensor],
    weight: Int8Weight,
    bias: torch.Tensor | None = None,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``x @ weight.T + bias`` in 8-bit integers, a scale per token and per output channel.

    Differentiable in ``x`` (given as a tensor) where the weight holds its
    transposed codes; weight and bias are constants.

    Args:
        x: Tokens ``[..., K]`` bf16 or fp16, quantized here, or the ``(q, s)`` of
            ``rowquant_int8``, ``gelu_int8`` or ``sandwich_norm_int8``.
        weight: The quantized weight ``[N, K]``.
        bias: Bias ``[N]`` of the output's type, or None.
        dtype: Output type where ``x`` is given as codes; that of ``x`` otherwise.

    Returns:
        ``[..., N]``.

    Raises:
        ValueError: On tensors off CUDA, unsupported dtypes or shapes, a bias that
            requires a gradient, or an ``x`` that does without transposed codes.
    """
    codes = not isinstance(x, torch.Tensor)
    first = x[0] if codes else x
    _check_same_device(first, *weight, bias)
    if codes:
        _check_codes(*x)
        if dtype not in HALF_TYPES:
            raise ValueError(f"dtype must be torch.bfloat16 or torch.float16, got {dtype}")
        _check_same_device(first, x[1])
    else:
        _check_half("x", x)
        _check_cols("x", x)
        dtype = x.dtype
    _check_weight(weight, first.shape[-1])
    wq, ws, wqt = _dense(weight.q), weight.s.contiguous(), weight.qt
    if bias is not None:
        if bias.dtype != dtype or bias.numel() != wq.shape[0]:
            raise ValueError(f"bias must be {dtype} [{wq.shape[0]}], got {bias.dtype} {list(bias.shape)}")
        if bias.requires_grad and torch.is_grad_enabled():
            raise ValueError("bias is a constant here: it must not require a gradient")
        bias = bias.contiguous()
    if codes:
        return _int8_linear_codes(_dense(x[0]), x[1].contiguous(), wq, ws, bias, dtype)
    if torch.is_grad_enabled() and x.requires_grad:
        if wqt is None:
            raise ValueError("the input gradient needs quantize_weight_int8(w, backward=True)")
        _check_cols("the transposed weight", wqt)
        wqt, ws = _dense(wqt), _dense(ws)
    return _int8_linear(_dense(x), wq, ws, wqt, bias)


def gelu_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """GELU (the erf form) in 8 bits, with its input's 8-bit checkpoint.

    Args:
        x: Tokens, shape ``[..., K]`` bf16 or fp16, K a multiple of 16 up to 16384.

    Returns:
        ``(q, s, c, cs)``: codes and scales of GELU(x), as ``int8_linear`` takes
        them, and codes and scales of ``x``, as ``gelu_int8_bwd`` takes them.

    Raises:
        ValueError: If ``x`` is not on CUDA or a dtype/shape is unsupported.
    """
    _check_same_device(x)
    _check_half("x", x)
    _check_cols("x", x)
    return _gelu_int8(_dense(x))


def gelu_int8_bwd(dy: torch.Tensor, c: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    """Gradient of GELU at the input whose codes are kept: ``dy * GELU'(c * cs)``.

    Args:
        dy: Gradient of GELU(x), shape ``[..., K]`` bf16 or fp16.
        c: Codes of ``x``, int8, same shape.
        cs: Their scales, one per row.

    Raises:
        ValueError: On tensors off CUDA or unsupported dtypes or shapes.
    """
    _check_same_device(dy, c, cs)
    _check_half("dy", dy)
    _check_codes(c, cs)
    if dy.shape != c.shape:
        raise ValueError(f"dy and the codes must match, got {list(dy.shape)} and {list(c.shape)}")
    return _gelu_int8_bwd(_dense(dy), _dense(c), cs.contiguous())


def int8_restore(q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that codes stand for: ``q * s`` in ``dtype`` (bf16 or fp16).

    Raises:
        ValueError: On tensors off CUDA or unsupported dtypes or shapes.
    """
    _check_same_device(q, s)
    _check_codes(q, s)
    if dtype not in HALF_TYPES:
        raise ValueError(f"dtype must be torch.bfloat16 or torch.float16, got {dtype}")
    return _int8_restore(_dense(q), s.contiguous(), dtype)


def int8_wgrad(dy: torch.Tensor, q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """Weight gradient ``dy.T @ x`` over all tokens, with ``x`` kept as 8-bit codes.

    Args:
        dy: Gradient at the layer's output, shape ``[..., N]`` bf16 or fp16 (for a
            low-rank adapter, at its first factor's output: N is the rank).
        q: Codes of the layer's input, int8 ``[..., K]``, same leading sizes.
        s: Their scales, one per token.

    Returns:
        ``[N, K]``, dtype of ``dy``, summed in fp32.

    Raises:
        ValueError: On tensors off CUDA or unsupported dtypes or shapes.
    """
    _check_same_device(dy, q, s)
    _check_half("dy", dy)
    _check_codes(q, s)
    if dy.shape[:-1] != q.shape[:-1] or not dy.shape[-1]:
        raise ValueError(f"dy and the codes must have the same tokens, got {list(dy.shape)} and {list(q.shape)}")
    N = dy.shape[-1]
    if N % 8:  # the kernel's copies of dy need rows of a multiple of 16 bytes
        dy = torch.nn.functional.pad(dy, (0, -N % 8))
    return _int8_wgrad(_dense(dy), _dense(q), s.contiguous())[:N]

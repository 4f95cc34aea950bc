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

``int8_linear`` of a tensor is differentiable in it.  The other functions have no
gradient: results of inputs that require one raise an error in a backward pass.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .._lib import load
from .common import HALF_TYPES, _check_half, _check_same_device, _dense, _direct, _launch, _plain, _registered

__all__ = [
    "Int8Weight",
    "gelu_int8",
    "gelu_int8_bwd",
    "int8_linear",
    "int8_linear_dx",
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
def _quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    K = x.shape[-1]
    rows = x.numel() // K
    q, s = torch.empty_like(x, dtype=I8), x.new_empty((rows, 1), dtype=F32)
    _launch("afb_rowquant_int8", x, x.data_ptr(), None, q.data_ptr(), s.data_ptr(), rows, K, HALF_TYPES[x.dtype])
    return q, s


def _product(q, s, wq, ws, bias, dtype):
    K, N = q.shape[-1], wq.shape[0]
    y = q.new_empty((*q.shape[:-1], N), dtype=dtype)
    _launch("afb_int8_linear", q, q.data_ptr(), s.data_ptr(), wq.data_ptr(), ws.data_ptr(),
            None if bias is None else bias.data_ptr(), y.data_ptr(), q.numel() // K, N, K, HALF_TYPES[dtype])
    return y


def _quant_product(x, cols, wq, ws, bias):
    """Quantize x, or x * cols, and multiply: one call, its codes in a workspace."""
    K, N = x.shape[-1], wq.shape[0]
    rows = x.numel() // K
    y = x.new_empty((rows, N) if x.ndim == 2 else (*x.shape[:-1], N))
    nbytes = load().afb_int8_linear_x_workspace(rows, N, K)
    work = x.new_empty(nbytes, dtype=I8) if nbytes else None
    _launch("afb_int8_linear_x", x, x.data_ptr(), None if cols is None else cols.data_ptr(), wq.data_ptr(),
            None if ws is None else ws.data_ptr(), None if bias is None else bias.data_ptr(), y.data_ptr(), rows, N, K,
            HALF_TYPES[x.dtype], None if work is None else work.data_ptr(), nbytes)
    return y


def _linear(x, wq, ws, wqt, bias):
    return _quant_product(x, None, wq, ws, bias)


def _linear_bwd(dy, ws, wqt):
    return _quant_product(_dense(dy), ws, wqt, None, None)


def _gelu(x):
    K = x.shape[-1]
    rows = x.numel() // K
    q, c = torch.empty_like(x, dtype=I8), torch.empty_like(x, dtype=I8)
    s, cs = x.new_empty((rows, 1), dtype=F32), x.new_empty((rows, 1), dtype=F32)
    _launch("afb_gelu_int8", x, x.data_ptr(), q.data_ptr(), s.data_ptr(), c.data_ptr(), cs.data_ptr(), rows, K,
            HALF_TYPES[x.dtype])
    return q, s, c, cs


def _gelu_bwd(dy, c, cs):
    dx = torch.empty_like(dy)
    K = dy.shape[-1]
    _launch("afb_gelu_int8_bwd", dy, dy.data_ptr(), c.data_ptr(), cs.data_ptr(), dx.data_ptr(), dy.numel() // K, K,
            HALF_TYPES[dy.dtype])
    return dx


def _restore(q, s, dtype):
    y = torch.empty_like(q, dtype=dtype)
    K = q.shape[-1]
    _launch("afb_int8_restore", q, q.data_ptr(), s.data_ptr(), y.data_ptr(), q.numel() // K, K, HALF_TYPES[dtype])
    return y


def _wgrad(dy, q, s):
    N, K = dy.shape[-1], q.shape[-1]
    rows = q.numel() // K
    dw = dy.new_empty((N, K))
    nbytes = load().afb_int8_wgrad_workspace(rows, N, K) if N % 8 else 0
    work = dy.new_empty(nbytes, dtype=I8) if nbytes else None
    _launch("afb_int8_wgrad", dy, dy.data_ptr(), q.data_ptr(), s.data_ptr(), dw.data_ptr(), rows, N, K,
            HALF_TYPES[dy.dtype], None if work is None else work.data_ptr(), nbytes)
    return dw


class _LinearFn(torch.autograd.Function):
    """int8_linear's gradient where the launches are called directly."""

    @staticmethod
    def forward(ctx, x, wq, ws, wqt, bias):
        ctx.save_for_backward(ws, wqt)
        return _linear(x, wq, ws, wqt, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ws, wqt = ctx.saved_tensors
        dx = _linear_bwd(dy, ws, wqt) if _plain(dy) else _registered(_int8_linear_bwd, dy, ws, wqt)
        return dx, None, None, None, None


# ----------------------------------------------------------------- custom ops --
@torch.library.custom_op("anima_flat_b200::rowquant_int8", mutates_args=())
def _rowquant_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _quant(_dense(x))


@_rowquant_int8.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=I8), x.new_empty((x.numel() // x.shape[-1], 1), dtype=F32)


@torch.library.custom_op("anima_flat_b200::int8_linear_codes", mutates_args=())
def _int8_linear_codes(
    q: torch.Tensor, s: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, bias: torch.Tensor | None,
    dtype: torch.dtype,
) -> torch.Tensor:
    return _product(_dense(q), _dense(s), _dense(wq), _dense(ws), bias, dtype)


@_int8_linear_codes.register_fake
def _(q, s, wq, ws, bias, dtype):
    return q.new_empty((*q.shape[:-1], wq.shape[0]), dtype=dtype)


@torch.library.custom_op("anima_flat_b200::int8_linear", mutates_args=())
def _int8_linear(
    x: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, wqt: torch.Tensor | None,
    bias: torch.Tensor | None,
) -> torch.Tensor:
    return _linear(_dense(x), _dense(wq), _dense(ws), wqt, bias)


@_int8_linear.register_fake
def _(x, wq, ws, wqt, bias):
    return x.new_empty((*x.shape[:-1], wq.shape[0]))


@torch.library.custom_op("anima_flat_b200::int8_linear_bwd", mutates_args=())
def _int8_linear_bwd(dy: torch.Tensor, ws: torch.Tensor, wqt: torch.Tensor) -> torch.Tensor:
    return _linear_bwd(dy, _dense(ws), _dense(wqt))


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
    return _gelu(_dense(x))


@_gelu_int8.register_fake
def _(x):
    rows = x.numel() // x.shape[-1]
    return (x.new_empty(x.shape, dtype=I8), x.new_empty((rows, 1), dtype=F32),
            x.new_empty(x.shape, dtype=I8), x.new_empty((rows, 1), dtype=F32))


@torch.library.custom_op("anima_flat_b200::gelu_int8_bwd", mutates_args=())
def _gelu_int8_bwd(dy: torch.Tensor, c: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    return _gelu_bwd(_dense(dy), _dense(c), _dense(cs))


@_gelu_int8_bwd.register_fake
def _(dy, c, cs):
    return dy.new_empty(dy.shape)


@torch.library.custom_op("anima_flat_b200::int8_restore", mutates_args=())
def _int8_restore(q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return _restore(_dense(q), _dense(s), dtype)


@_int8_restore.register_fake
def _(q, s, dtype):
    return q.new_empty(q.shape, dtype=dtype)


@torch.library.custom_op("anima_flat_b200::int8_wgrad", mutates_args=())
def _int8_wgrad(dy: torch.Tensor, q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return _wgrad(_dense(dy), _dense(q), _dense(s))


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


def _check_weight(wq, ws, bias, K: int, dtype: torch.dtype) -> torch.Tensor | None:
    if wq.dtype != I8 or wq.ndim != 2 or wq.shape[1] != K or not wq.shape[0]:
        raise ValueError(f"the weight's codes must be torch.int8 [N, {K}], got {wq.dtype} {list(wq.shape)}")
    N = wq.shape[0]
    if ws.dtype != F32 or ws.numel() != N:
        raise ValueError(f"the weight's scales must be torch.float32 [{N}], got {ws.dtype} {list(ws.shape)}")
    if ws.requires_grad and torch.is_grad_enabled():
        raise ValueError("the weight's scales are constants here: they must not require a gradient")
    if bias is None:
        return None
    if bias.dtype != dtype or bias.numel() != N:
        raise ValueError(f"bias must be {dtype} [{N}], got {bias.dtype} {list(bias.shape)}")
    if bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("bias is a constant here: it must not require a gradient")
    return bias.contiguous()


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
    return _quant(_dense(x)) if _direct(x) else _registered(_rowquant_int8, x)


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
        ValueError: On tensors off CUDA, unsupported dtypes or shapes, a bias or
            scales of the weight that require a gradient, or an ``x`` that does without transposed codes.
    """
    wq, ws, wqt = weight
    if not isinstance(x, torch.Tensor):
        q, s = x
        _check_same_device(q, s, wq, ws, bias)
        _check_codes(q, s)
        if dtype not in HALF_TYPES:
            raise ValueError(f"dtype must be torch.bfloat16 or torch.float16, got {dtype}")
        bias = _check_weight(wq, ws, bias, q.shape[-1], dtype)
        if not _direct(q, s, wq, ws, bias):
            return _registered(_int8_linear_codes, q, s, wq, ws, bias, dtype)
        return _product(_dense(q), _dense(s), _dense(wq), _dense(ws), bias, dtype)
    _check_same_device(x, wq, ws, wqt, bias)
    _check_half("x", x)
    _check_cols("x", x)
    bias = _check_weight(wq, ws, bias, x.shape[-1], x.dtype)
    grad = x.requires_grad and torch.is_grad_enabled()
    if grad:
        if wqt is None:
            raise ValueError("the input gradient needs quantize_weight_int8(w, backward=True)")
        if wqt.dtype != I8 or wqt.shape != (x.shape[-1], wq.shape[0]):
            raise ValueError(f"the transposed codes must be torch.int8 [{x.shape[-1]}, {wq.shape[0]}]")
        _check_cols("the transposed weight", wqt)
    if not _plain(x, wq, ws, wqt, bias):
        return _registered(_int8_linear, x, wq, ws, wqt, bias)
    x, wq, ws = _dense(x), _dense(wq), _dense(ws)
    return _LinearFn.apply(x, wq, ws, _dense(wqt), bias) if grad else _linear(x, wq, ws, wqt, bias)


def int8_linear_dx(dy: torch.Tensor, weight: Int8Weight) -> torch.Tensor:
    """Input gradient of ``int8_linear``: ``dy @ weight`` in 8-bit integers.

    ``dy`` times the weight's scales is quantized per token and multiplied by
    the transposed codes.  For a caller that writes its own backward pass;
    ``int8_linear`` itself is differentiable.

    Args:
        dy: Gradient at the output, shape ``[..., N]`` bf16 or fp16, N a multiple of 16 up to 16384.
        weight: The quantized weight ``[N, K]`` with its transposed codes.

    Returns:
        ``[..., K]``, dtype of ``dy``.

    Raises:
        ValueError: On tensors off CUDA, a weight without transposed codes, or
            unsupported dtypes or shapes.
    """
    wq, ws, wqt = weight
    if wqt is None:
        raise ValueError("the input gradient needs quantize_weight_int8(w, backward=True)")
    _check_same_device(dy, ws, wqt)
    _check_half("dy", dy)
    _check_cols("dy", dy)
    N = dy.shape[-1]
    if wqt.dtype != I8 or wqt.ndim != 2 or wqt.shape[1] != N or ws.dtype != F32 or ws.numel() != N:
        raise ValueError(f"the transposed codes must be torch.int8 [K, {N}] with torch.float32 scales [{N}]")
    if not _direct(dy, ws, wqt):
        return _registered(_int8_linear_bwd, dy, ws, wqt)
    return _linear_bwd(dy, _dense(ws), _dense(wqt))


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
    return _gelu(_dense(x)) if _direct(x) else _registered(_gelu_int8, x)


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
    if not _direct(dy, c, cs):
        return _registered(_gelu_int8_bwd, dy, c, cs)
    return _gelu_bwd(_dense(dy), _dense(c), _dense(cs))


def int8_restore(q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that codes stand for: ``q * s`` in ``dtype`` (bf16 or fp16).

    Raises:
        ValueError: On tensors off CUDA or unsupported dtypes or shapes.
    """
    _check_same_device(q, s)
    _check_codes(q, s)
    if dtype not in HALF_TYPES:
        raise ValueError(f"dtype must be torch.bfloat16 or torch.float16, got {dtype}")
    return _restore(_dense(q), _dense(s), dtype) if _direct(q, s) else _registered(_int8_restore, q, s, dtype)


def int8_wgrad(dy: torch.Tensor, q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """Weight gradient ``dy.T @ x`` over all tokens, with ``x`` kept as 8-bit codes.

    Args:
        dy: Gradient at the layer's output, shape ``[..., N]`` bf16 or fp16 (for a
            low-rank adapter, at its first factor's output: N is the rank), N at most 2^20.
        q: Codes of the layer's input, int8 ``[..., K]``, same leading sizes.
        s: Their scales, one per token.

    Returns:
        ``[N, K]``, dtype of ``dy``: an fp32 sum, rounded once.  The codes may stand for
        values that this type does not hold (those of a bf16 row with an fp16 ``dy``).

    Raises:
        ValueError: On tensors off CUDA or unsupported dtypes or shapes.
    """
    _check_same_device(dy, q, s)
    _check_half("dy", dy)
    _check_codes(q, s)
    if dy.shape[:-1] != q.shape[:-1] or not dy.shape[-1]:
        raise ValueError(f"dy and the codes must have the same tokens, got {list(dy.shape)} and {list(q.shape)}")
    if dy.shape[-1] > 2**20:
        raise ValueError(f"the last dimension of dy must be at most 2^20, got {dy.shape[-1]}")
    return _wgrad(_dense(dy), _dense(q), _dense(s)) if _direct(dy, q, s) else _registered(_int8_wgrad, dy, q, s)

"""Norms before and after a block, fused with its gate and residual scale.

No counterpart in the reference, whose blocks have one norm each
(``residual_adaln``).  For models that also normalise a block's output:

    z = a * residual + gate[b] * (rms(x) * post_weight)
    h = rms(z) * pre_weight * scale[b] + shift[b]

with ``rms(v) = v / sqrt(mean(v^2) + eps)``, x the block's output, z the
residual stream and h the next block's input.  z is rounded to its type before
h is formed from it.  ``scale`` already includes the +1, as for ``adaln``.
"""

from __future__ import annotations

import torch

from .._lib import load
from .common import HALF_TYPES, _check_half, _check_same_device, _check_vec, _dense, _direct, _launch, _plain, _registered

__all__ = ["sandwich_norm", "sandwich_norm_bwd", "sandwich_norm_int8"]

F32 = torch.float32


def _dense_all(*ts: torch.Tensor | None):
    return (None if t is None else _dense(t) for t in ts)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------ launches --
def _fwd(x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps):
    B, S, D = x.shape
    h, z = torch.empty_like(x), torch.empty_like(x)
    _launch("afb_sandwich_norm", x, x.data_ptr(), residual.data_ptr(), _ptr(gate), post_weight.data_ptr(),
            pre_weight.data_ptr(), _ptr(shift), _ptr(scale), h.data_ptr(), z.data_ptr(), B, S, D,
            residual_scale, eps, HALF_TYPES[x.dtype])
    return h, z


def _fwd_int8(x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps):
    B, S, D = x.shape
    z = torch.empty_like(x)
    q, s = torch.empty_like(x, dtype=torch.int8), x.new_empty((B * S, 1), dtype=F32)
    _launch("afb_sandwich_norm_int8", x, x.data_ptr(), residual.data_ptr(), _ptr(gate), post_weight.data_ptr(),
            pre_weight.data_ptr(), _ptr(shift), _ptr(scale), q.data_ptr(), s.data_ptr(), z.data_ptr(), B, S, D,
            residual_scale, eps, HALF_TYPES[x.dtype])
    return q, s, z


def _bwd(gh, gz, z, x, gate, post_weight, pre_weight, scale, residual_scale, eps):
    B, S, D = z.shape
    dx, dres = torch.empty_like(x), torch.empty_like(z)
    vec = gate if gate is not None else scale
    if vec is None:
        vec = z.new_empty((B, D))
    dgate, dshift, dscale = torch.empty_like(vec), torch.empty_like(vec), torch.empty_like(vec)
    dpost, dpre = torch.empty_like(post_weight), torch.empty_like(pre_weight)
    if z.numel() == 0:
        for t in (dgate, dshift, dscale, dpost, dpre):
            t.zero_()
        return dx, dres, dgate, dpost, dpre, dshift, dscale
    nbytes = load().afb_sandwich_norm_bwd_workspace(B, S, D)
    ws = z.new_empty(nbytes, dtype=torch.int8)
    _launch("afb_sandwich_norm_bwd", z, gh.data_ptr(), _ptr(gz), z.data_ptr(), x.data_ptr(), _ptr(gate),
            post_weight.data_ptr(), pre_weight.data_ptr(), _ptr(scale), dx.data_ptr(), dres.data_ptr(),
            dgate.data_ptr(), dpost.data_ptr(), dpre.data_ptr(), dshift.data_ptr(), dscale.data_ptr(),
            B, S, D, residual_scale, eps, HALF_TYPES[z.dtype], ws.data_ptr(), nbytes)
    return dx, dres, dgate, dpost, dpre, dshift, dscale


def _saved(ctx, x, gate, post_weight, pre_weight, shift, scale, z, residual_scale, eps):
    ctx.save_for_backward(x, gate, post_weight, pre_weight, scale, z)
    ctx.has_shift = shift is not None
    ctx.residual_scale = residual_scale
    ctx.eps = eps


def _grads(ctx, bwd, gh, gz):
    x, gate, post_weight, pre_weight, scale, z = ctx.saved_tensors
    dx, dres, dgate, dpost, dpre, dshift, dscale = bwd(
        gh, gz, z, x, gate, post_weight, pre_weight, scale, ctx.residual_scale, ctx.eps)
    return (dx, dres, dgate if gate is not None else None, dpost, dpre, dshift if ctx.has_shift else None,
            dscale if scale is not None else None, None, None)


class _SandwichFn(torch.autograd.Function):
    """sandwich_norm's gradient where the launches are called directly."""

    @staticmethod
    def forward(ctx, x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps):
        h, z = _fwd(x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps)
        _saved(ctx, x, gate, post_weight, pre_weight, shift, scale, z, residual_scale, eps)
        return h, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gh, gz):
        if not _plain(gh, gz):
            return _grads(ctx, lambda *args: _registered(_sandwich_norm_bwd, *args), gh, gz)
        return _grads(ctx, _bwd, *_dense_all(gh, gz))


# ----------------------------------------------------------------- custom ops --
@torch.library.custom_op("anima_flat_b200::sandwich_norm", mutates_args=())
def _sandwich_norm(
    x: torch.Tensor, residual: torch.Tensor, gate: torch.Tensor | None, post_weight: torch.Tensor,
    pre_weight: torch.Tensor, shift: torch.Tensor | None, scale: torch.Tensor | None,
    residual_scale: float, eps: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    return _fwd(*_dense_all(x, residual, gate, post_weight, pre_weight, shift, scale), residual_scale, eps)


@_sandwich_norm.register_fake
def _(x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape)


@torch.library.custom_op("anima_flat_b200::sandwich_norm_int8", mutates_args=())
def _sandwich_norm_int8(
    x: torch.Tensor, residual: torch.Tensor, gate: torch.Tensor | None, post_weight: torch.Tensor,
    pre_weight: torch.Tensor, shift: torch.Tensor | None, scale: torch.Tensor | None,
    residual_scale: float, eps: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _fwd_int8(*_dense_all(x, residual, gate, post_weight, pre_weight, shift, scale), residual_scale, eps)


@_sandwich_norm_int8.register_fake
def _(x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps):
    B, S, _ = x.shape
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty((B * S, 1), dtype=F32), x.new_empty(x.shape)


@torch.library.custom_op("anima_flat_b200::sandwich_norm_bwd", mutates_args=())
def _sandwich_norm_bwd(
    gh: torch.Tensor, gz: torch.Tensor | None, z: torch.Tensor, x: torch.Tensor, gate: torch.Tensor | None,
    post_weight: torch.Tensor, pre_weight: torch.Tensor, scale: torch.Tensor | None,
    residual_scale: float, eps: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _bwd(*_dense_all(gh, gz, z, x, gate, post_weight, pre_weight, scale), residual_scale, eps)


@_sandwich_norm_bwd.register_fake
def _(gh, gz, z, x, gate, post_weight, pre_weight, scale, residual_scale, eps):
    B, _, D = z.shape
    vec = [z.new_empty((B, D)) for _ in range(3)]
    w = [z.new_empty(D, dtype=F32) for _ in range(2)]
    return x.new_empty(x.shape), z.new_empty(z.shape), vec[0], w[0], w[1], vec[1], vec[2]


def _setup(ctx, inputs, output):
    x, _, gate, post_weight, pre_weight, shift, scale, residual_scale, eps = inputs
    _saved(ctx, x, gate, post_weight, pre_weight, shift, scale, output[1], residual_scale, eps)


def _backward(ctx, gh, gz):
    return _grads(ctx, _sandwich_norm_bwd, gh, gz)


torch.library.register_autograd("anima_flat_b200::sandwich_norm", _backward, setup_context=_setup)


# --------------------------------------------------------------------- public --
def _weight(w: torch.Tensor, D: int, name: str) -> torch.Tensor:
    if w.dtype is F32 and w.shape == (D,):
        return w
    if w.numel() != D:
        raise ValueError(f"{name} must be [{D}], got {list(w.shape)}")
    return w.to(F32).reshape(D)


def _vec(v: torch.Tensor | None, shape: tuple[int, int], dtype: torch.dtype, name: str) -> torch.Tensor | None:
    if v is None:
        return None
    if v.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {v.dtype}")
    if v.shape == shape:
        return v
    _check_vec(v, *shape, name)
    return v.reshape(shape)


def _check_rows(x: torch.Tensor, *like: tuple[str, torch.Tensor | None]) -> tuple[int, int]:
    _check_half("activations", x)
    shape = x.shape
    if len(shape) != 3:
        raise ValueError(f"expected [B, S, D] activations, got {list(shape)}")
    D = shape[2]
    if D < 8 or D % 8 or D > 4096:
        raise ValueError(f"D must be a multiple of 8 in [8, 4096], got {D}")
    if shape[0] > 65535 or shape[0] * shape[1] >= 2**31:
        raise ValueError(f"B must be at most 65535 and B * S below 2^31, got {list(shape)}")
    for name, t in like:
        if t is not None and (t.shape != shape or t.dtype is not x.dtype):
            raise ValueError(f"{name} must be {x.dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
    return shape[0], D


def _args(x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps):
    _check_same_device(x, residual, gate, post_weight, pre_weight, shift, scale)
    vec, dtype = _check_rows(x, ("residual", residual)), x.dtype
    return (x, residual, _vec(gate, vec, dtype, "gate"), _weight(post_weight, vec[1], "post_weight"),
            _weight(pre_weight, vec[1], "pre_weight"), _vec(shift, vec, dtype, "shift"),
            _vec(scale, vec, dtype, "scale"), float(residual_scale), float(eps))


def sandwich_norm(x, residual, gate, post_weight, pre_weight, shift=None, scale=None, residual_scale=1.0, eps=1e-6):
    """RMSNorm of a block's output, gated residual add, RMSNorm and modulation for the next block.

    Differentiable in every tensor.

    Args:
        x: The block's output, shape ``[B, S, D]`` bf16 or fp16, D a multiple of 8 up to 4096,
            B at most 65535.
        residual: Residual stream, same shape and dtype as ``x``.
        gate: Gate, shape ``[B, D]``, or None for one.
        post_weight: Weight ``[D]`` of the norm after the block.
        pre_weight: Weight ``[D]`` of the norm before the next one.
        shift: Shift, shape ``[B, D]``, or None for zero.
        scale: Scale (already including the +1), shape ``[B, D]``, or None for one.
        residual_scale: Factor of the residual stream.
        eps: Epsilon of both norms.

    Returns:
        ``(h, z)``: the next block's input and the updated residual stream.

    Raises:
        ValueError: On tensors off CUDA or unsupported dtypes or shapes.
    """
    args = _args(x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps)
    if not _plain(*args[:7]):
        return _registered(_sandwich_norm, *args)
    args = (*_dense_all(*args[:7]), *args[7:])
    if torch.is_grad_enabled():
        for t in args[:7]:
            if t is not None and t.requires_grad:
                return _SandwichFn.apply(*args)
    return _fwd(*args)


def sandwich_norm_int8(x, residual, gate, post_weight, pre_weight, shift=None, scale=None, residual_scale=1.0,
                       eps=1e-6):
    """``sandwich_norm`` whose output h is returned as 8-bit codes with a scale per token.

    Arguments as for ``sandwich_norm``; not differentiable: a backward pass through
    its results raises an error (``sandwich_norm_bwd`` takes its z).

    Returns:
        ``(q, s, z)``: codes ``[B, S, D]`` int8 and scales ``[B * S, 1]`` float32 of
        h before it is rounded, as ``int8_linear`` takes them, and z.

    Raises:
        ValueError: On tensors off CUDA or unsupported dtypes or shapes.
    """
    args = _args(x, residual, gate, post_weight, pre_weight, shift, scale, residual_scale, eps)
    if not _direct(*args[:7]):
        return _registered(_sandwich_norm_int8, *args)
    return _fwd_int8(*_dense_all(*args[:7]), *args[7:])


def sandwich_norm_bwd(gh, gz, z, x, gate, post_weight, pre_weight, scale=None, residual_scale=1.0, eps=1e-6):
    """Gradients of ``sandwich_norm`` from its output z and input x.

    For a caller that writes its own backward pass (with z or x restored from
    8-bit checkpoints, for instance); ``sandwich_norm`` itself is differentiable.

    Args:
        gh: Gradient of h, shape ``[B, S, D]``.
        gz: Gradient of z, same shape, or None for zero.
        z: The residual stream that ``sandwich_norm`` returned.
        x: The block's output that it was given.
        gate, post_weight, pre_weight, scale, residual_scale, eps: As it was given them.

    Returns:
        ``(dx, dresidual, dgate, dpost_weight, dpre_weight, dshift, dscale)``: the
        vectors of the activations' type, the weights' gradients float32.

    Raises:
        ValueError: On tensors off CUDA or unsupported dtypes or shapes.
    """
    _check_same_device(gh, gz, z, x, gate, post_weight, pre_weight, scale)
    vec, dtype = _check_rows(z, ("x", x), ("gh", gh), ("gz", gz)), z.dtype
    args = (gh, gz, z, x, _vec(gate, vec, dtype, "gate"),
            _weight(post_weight, vec[1], "post_weight"), _weight(pre_weight, vec[1], "pre_weight"),
            _vec(scale, vec, dtype, "scale"), float(residual_scale), float(eps))
    if not _direct(*args[:8]):
        return _registered(_sandwich_norm_bwd, *args)
    return _bwd(*_dense_all(*args[:8]), *args[8:])

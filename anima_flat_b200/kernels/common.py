"""Argument checks and launch plumbing shared by the op modules.

Mirrors src/kernels/common.py:6-9 (``_check``).  The reference's run-time
autotuner (``tuned_rows``, common.py:12-34) has no counterpart: every launch
shape here is fixed by the tensor shapes, so results never depend on timing.
"""

from __future__ import annotations

import torch

from .._lib import load

BF16 = torch.bfloat16


def _check(*ts: torch.Tensor) -> None:
    """Raise ValueError unless every tensor is on CUDA (common.py:6-9)."""
    for t in ts:
        if not t.is_cuda:
            raise ValueError("CUDA tensors required")


def _check_dtype(dtype: torch.dtype, what: str, *ts: torch.Tensor) -> None:
    for t in ts:
        if t.dtype != dtype:
            raise ValueError(f"{what} must be {dtype}, got {t.dtype}")


def _check_vec(t: torch.Tensor, batch: int, dim: int, name: str) -> None:
    """Per-sample modulation vectors are [batch, dim] (adaln.py:34, :44-45)."""
    if t.numel() != batch * dim or t.shape[-1] != dim:
        raise ValueError(f"{name} must be [batch, dim] = [{batch}, {dim}], got {list(t.shape)}")


def _stream(t: torch.Tensor) -> int:
    """Handle of the current CUDA stream on the tensor's device."""
    return torch.cuda.current_stream(t.device).cuda_stream


# dtype codes of the C ABI's entry points that take both 16-bit types.
HALF_TYPES = {torch.bfloat16: 0, torch.float16: 1}


def _check_half(what: str, t: torch.Tensor) -> None:
    if t.dtype not in HALF_TYPES:
        raise ValueError(f"{what} must be torch.bfloat16 or torch.float16, got {t.dtype}")


def _check_same_device(*ts: torch.Tensor | None) -> None:
    """Raise ValueError unless all tensors are on one CUDA device."""
    device = None
    for t in ts:
        if t is None:
            continue
        d = t.get_device()
        if d != device:
            if d < 0 or not t.is_cuda:
                raise ValueError("CUDA tensors required")
            if device is not None:
                raise ValueError(f"tensors are on devices {device} and {d}")
            device = d


def _dense(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned: a copy only where `t` is not.

    It reads the tensor's address, so a public function calls it once `_plain`
    has said that there is one; the registered ops call it on what they are given.
    """
    if t.is_contiguous():
        return t if not t.data_ptr() & 15 else t.clone()
    return t.contiguous()


_Tensor, _Parameter = torch.Tensor, torch.nn.Parameter


def _plain(*ts: torch.Tensor | None) -> bool:
    """True where the launches may be called directly, without torch's dispatcher.

    That is: ordinary tensors, outside compilation, ``torch.jit.trace``, dispatch
    modes (fake tensors, graph capture), function transforms and forward-mode
    differentiation, all of which need the registered op: none of them sees a
    launch that goes by addresses.  A Python custom op costs about 40 us a call; a
    direct call takes 9 to 17 us in all.
    """
    if (
        torch.compiler.is_compiling()
        or torch._C._is_tracing()
        or torch._C._len_torch_dispatch_stack()
        or torch._C._functorch.peek_interpreter_stack() is not None
        or torch.autograd.forward_ad._current_level >= 0
    ):
        return False
    for t in ts:
        if t is not None and type(t) is not _Tensor and type(t) is not _Parameter:
            return False
    return True


def _direct(*ts: torch.Tensor | None) -> bool:
    """`_plain` for the ops without a gradient: false where one is asked of them too.

    The registered op then keeps the graph, and the backward pass raises an error
    where the direct call would have cut the gradient off in silence.
    """
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return False
    return _plain(*ts)


def _registered(op, *args):
    """Call a registered op where `_plain` has ruled the direct launch out.

    The ops have no forward-mode derivative, which the dispatcher would leave
    out in silence, and none under ``torch.func``'s gradients: both are refused.
    """
    if not torch.compiler.is_compiling():
        ts = [a for a in args if isinstance(a, torch.Tensor) and a.is_floating_point()]
        forward_ad = torch.autograd.forward_ad
        if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
            raise RuntimeError(f"{op._qualname} has no forward-mode derivative")
        if torch._C._functorch.peek_interpreter_stack() is not None and any(t.requires_grad for t in ts):
            raise RuntimeError(f"{op._qualname} has no gradient under torch.func transforms: use torch.autograd")
    return op(*args)


_entries: dict[str, object] = {}


def _launch(name: str, t: torch.Tensor, *args) -> None:
    """Call entry point `name` on the current stream of the device of `t`."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(load(), name)
    device = t.get_device()
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        raise RuntimeError(f"{name} failed with status {rc}: {load().afb_last_error().decode(errors='replace')}")

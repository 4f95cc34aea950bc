"""Which calls of the 8-bit and sandwich-norm ops go past torch's dispatcher (CPU only)."""

from __future__ import annotations

import warnings

import pytest
import torch

import anima_flat_b200 as afb
from anima_flat_b200.kernels.common import _plain


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_tracing_takes_the_registered_ops():
    seen = []
    x = torch.zeros(2, 16)
    torch.jit.trace(lambda t: (seen.append(_plain(t)), t + 1)[1], (x,), check_trace=False)
    assert seen == [False] and _plain(x)


def test_fake_tensors_have_no_address_that_is_read():
    """The public functions under FakeTensorMode, on fake CUDA tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    bf, f32, i8 = torch.bfloat16, torch.float32, torch.int8
    with FakeTensorMode(), warnings.catch_warnings():
        warnings.simplefilter("error")
        e = lambda *s, d=bf: torch.empty(*s, dtype=d, device="cuda")  # noqa: E731
        x, dy, q, s = e(2, 6, 64), e(2, 6, 48), e(2, 6, 64, d=i8), e(12, 1, d=f32)
        up = afb.Int8Weight(e(48, 64, d=i8), e(48, d=f32), e(64, 48, d=i8))
        down = afb.Int8Weight(e(64, 48, d=i8), e(64, d=f32), e(48, 64, d=i8))
        w, g = e(64, d=f32), e(2, 64)
        shapes = [tuple(t.shape) for t in (
            *afb.rowquant_int8(x), afb.int8_linear(x, up), afb.int8_linear((q, s), up), afb.int8_linear_dx(dy, up),
            *afb.gelu_int8(x), afb.gelu_int8_bwd(x, q, s), afb.int8_restore(q, s), afb.int8_wgrad(dy, q, s),
            *afb.sandwich_norm(x, x, g, w, w), *afb.sandwich_norm_int8(x, x, g, w, w),
            *afb.sandwich_norm_bwd(x, None, x, x, g, w, w),
            afb.int8_lora_mlp(x, up, down, afb.LoRA(e(4, 64), e(48, 4)), afb.LoRA(e(4, 48), e(64, 4))))]
    rows, x, y = (12, 1), (2, 6, 64), (2, 6, 48)
    assert shapes == [x, rows, y, y, x, x, rows, x, rows, x, x, (48, 64), x, x, x, rows, x,
                      x, x, (2, 64), (64,), (64,), (2, 64), (2, 64), x]


def test_outputs_are_contiguous_whatever_the_inputs_are():
    """As the launches write them: what is compiled from the registered ops relies on their strides."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.anima_flat_b200
    with FakeTensorMode():
        e = lambda *s, d=torch.bfloat16: torch.empty(*s, dtype=d, device="cuda").transpose(0, 1)  # noqa: E731
        x, q, s, w = e(6, 2, 64), e(6, 2, 64, d=torch.int8), e(1, 12, d=torch.float32), torch.empty(64, device="cuda")
        assert not x.is_contiguous()
        wq, ws = e(64, 48, d=torch.int8), torch.empty(48, device="cuda")
        outs = (*ops.rowquant_int8(x), ops.int8_linear(x, wq, ws, None, None), ops.int8_linear_codes(q, s, wq, ws, None, x.dtype),
                ops.int8_linear_bwd(x, w, wq), *ops.gelu_int8(x), ops.gelu_int8_bwd(x, q, s), ops.int8_restore(q, s, x.dtype),
                ops.int8_wgrad(x, q, s), *ops.sandwich_norm(x, x, None, w, w, None, None, 1.0, 1e-6),
                *ops.sandwich_norm_int8(x, x, None, w, w, None, None, 1.0, 1e-6),
                *ops.sandwich_norm_bwd(x, None, x, x, None, w, w, None, 1.0, 1e-6))
        assert len(outs) == 24 and all(t.is_contiguous() for t in outs)


def test_sizes_beyond_the_launches_are_refused():
    """With a ValueError, like every other size, on fake CUDA tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        e = lambda *s, d=torch.bfloat16: torch.empty(*s, dtype=d, device="cuda")  # noqa: E731
        w = e(16, d=torch.float32)
        for x in (e(65536, 1, 16), e(4, 2**29, 16)):
            for call in (lambda: afb.sandwich_norm(x, x, None, w, w), lambda: afb.sandwich_norm_int8(x, x, None, w, w),
                         lambda: afb.sandwich_norm_bwd(x, None, x, x, None, w, w)):
                with pytest.raises(ValueError, match="65535"):
                    call()
        with pytest.raises(ValueError, match="2\\^20"):
            afb.int8_wgrad(e(2, 2**20 + 8), e(2, 16, d=torch.int8), e(2, 1, d=torch.float32))

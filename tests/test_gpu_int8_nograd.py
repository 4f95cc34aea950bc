"""The 8-bit and sandwich-norm functions without a gradient do not cut one off in silence."""

from __future__ import annotations

import pytest
import torch

import anima_flat_b200 as afb
from tests.test_gpu_int8_tracing import CALLS, _inputs, _list

pytestmark = pytest.mark.gpu

# function, and which of its arguments require a gradient in turn
FORMS = [("rowquant_int8", 0), ("int8_linear codes", 1), ("int8_linear_dx", 0), ("gelu_int8", 0), ("gelu_int8_bwd", 0),
         ("gelu_int8_bwd", 2), ("int8_restore", 1), ("int8_wgrad", 0), ("int8_wgrad", 2), ("sandwich_norm_int8", 0),
         ("sandwich_norm_int8", 1), ("sandwich_norm_int8", 3), ("sandwich_norm_bwd", 0), ("sandwich_norm_bwd", 4)]


@pytest.mark.parametrize("name,k", FORMS)
def test_backward_through_it_raises(name, k, cuda_dev):
    fn, args = CALLS[name]
    args = list(args(_inputs(7)))
    want = _list(fn(*args))
    args[k] = args[k].clone().requires_grad_(True)
    out = _list(fn(*args))
    assert all(torch.equal(a, b) for a, b in zip(out, want, strict=True))
    floats = [t for t in out if t.is_floating_point()]
    assert floats and all(t.requires_grad for t in floats)
    with pytest.raises(RuntimeError, match="autograd"):
        sum(t.float().sum() for t in floats).backward()
    with torch.no_grad():
        assert not any(t.requires_grad for t in _list(fn(*args)))


def test_scales_of_a_weight_are_constants(cuda_dev):
    c = _inputs(8)
    w = afb.Int8Weight(c["up"].q, c["up"].s.clone().requires_grad_(True), c["up"].qt)
    for x in (c["x"], (c["q"], c["s"])):
        with pytest.raises(ValueError, match="scales are constants"):
            afb.int8_linear(x, w)
    with pytest.raises(ValueError, match="scales are constants"):
        afb.int8_lora_mlp(c["x"], w, c["down"], afb.LoRA(*c["lora"][:2]), afb.LoRA(*c["lora"][2:]))
    with torch.no_grad():
        assert torch.equal(afb.int8_linear(c["x"], w), afb.int8_linear(c["x"], c["up"]))


def test_a_residual_stream_through_the_codes_is_not_cut_off(cuda_dev):
    """A block whose next input is quantised: the stream z must not lose its gradient unnoticed."""
    c = _inputs(9)
    r = c["r"].requires_grad_(True)
    q, s, z = afb.sandwich_norm_int8(c["y"], r, c["gate"], c["w"], c["w"])
    with pytest.raises(RuntimeError, match="autograd"):
        (z.float() + afb.int8_restore(q, s).float()).sum().backward()

"""torch.jit.trace through the public functions: the traced code launches what eager code does."""

from __future__ import annotations

import pytest
import torch

import anima_flat_b200 as afb

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    up = afb.quantize_weight_int8(rn(96, 64).to(BF), backward=True)
    down = afb.quantize_weight_int8(rn(64, 96).to(BF), backward=True)
    q, s = afb.rowquant_int8(rn(40, 64).to(BF))
    return dict(x=rn(40, 64).to(BF), dy=rn(40, 96).to(BF), q=q, s=s, up=up, down=down,
                y=rn(2, 20, 64).to(BF), r=rn(2, 20, 64).to(BF), gate=rn(2, 64).to(BF), w=1 + 0.1 * rn(64),
                lora=[(0.1 * rn(*s)).to(BF) for s in ((4, 64), (96, 4), (4, 96), (64, 4))])


# name -> function of tensors, and the tensors it is called with
CALLS = {
    "rowquant_int8": (afb.rowquant_int8, lambda c: (c["x"],)),
    "int8_linear": (lambda x, wq, ws: afb.int8_linear(x, afb.Int8Weight(wq, ws)), lambda c: (c["x"], *c["up"][:2])),
    "int8_linear codes": (lambda q, s, wq, ws: afb.int8_linear((q, s), afb.Int8Weight(wq, ws)),
                          lambda c: (c["q"], c["s"], *c["up"][:2])),
    "int8_linear_dx": (lambda dy, *w: afb.int8_linear_dx(dy, afb.Int8Weight(*w)), lambda c: (c["dy"], *c["up"])),
    "gelu_int8": (afb.gelu_int8, lambda c: (c["x"],)),
    "gelu_int8_bwd": (afb.gelu_int8_bwd, lambda c: (c["x"], c["q"], c["s"])),
    "int8_restore": (lambda q, s: afb.int8_restore(q, s), lambda c: (c["q"], c["s"])),
    "int8_wgrad": (afb.int8_wgrad, lambda c: (c["dy"], c["q"], c["s"])),
    "sandwich_norm": (lambda *t: afb.sandwich_norm(*t), lambda c: (c["y"], c["r"], c["gate"], c["w"], c["w"])),
    "sandwich_norm_int8": (lambda *t: afb.sandwich_norm_int8(*t), lambda c: (c["y"], c["r"], c["gate"], c["w"], c["w"])),
    "sandwich_norm_bwd": (lambda *t: afb.sandwich_norm_bwd(*t), lambda c: (c["y"], c["r"], c["y"], c["r"], c["gate"], c["w"], c["w"])),
    "int8_lora_mlp": (lambda x, a1, b1, a2, b2, *w: afb.int8_lora_mlp(
        x, afb.Int8Weight(*w[:3]), afb.Int8Weight(*w[3:]), afb.LoRA(a1, b1), afb.LoRA(a2, b2)),
        lambda c: (c["x"], *c["lora"], *c["up"], *c["down"])),
}


def _list(out):
    return [out] if isinstance(out, torch.Tensor) else list(out)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("name", list(CALLS))
def test_traced_code_gives_the_eager_result(name, cuda_dev):
    fn, args = CALLS[name]
    first, second = args(_inputs(1)), args(_inputs(2))
    traced = torch.jit.trace(fn, first, check_trace=False)
    assert all(torch.equal(a, b) for a, b in zip(_list(traced(*second)), _list(fn(*second)), strict=True))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_a_traced_backward_pass(cuda_dev):
    c, d = _inputs(3), _inputs(4)
    linear = lambda x, *w: afb.int8_linear(x, afb.Int8Weight(*w))  # noqa: E731
    traced = torch.jit.trace(linear, (c["x"].requires_grad_(True), *c["up"]), check_trace=False)
    x = d["x"].requires_grad_(True)
    (got,), (want,) = (torch.autograd.grad(f(x, *d["up"]), x, d["dy"]) for f in (traced, linear))
    assert torch.equal(got, want)
    fn, args = CALLS["int8_lora_mlp"]
    with pytest.raises(RuntimeError, match="no traced backward pass"):
        torch.jit.trace(fn, args(c), check_trace=False)

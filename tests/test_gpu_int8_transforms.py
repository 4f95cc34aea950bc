"""Graph capture, function transforms and saved-tensor hooks through the public functions.

No address of a tensor is read before it is known to be an ordinary one: the
rest takes the registered ops, and gives the eager result or a clear error.
"""

from __future__ import annotations

import warnings

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import anima_flat_b200 as afb
from tests.test_gpu_int8_tracing import CALLS, _inputs, _list

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("name", list(CALLS))
def test_make_fx(name, mode, cuda_dev):
    fn, args = CALLS[name]
    first, second = args(_inputs(1)), args(_inputs(2))
    with warnings.catch_warnings():
        warnings.filterwarnings("error", message="Accessing the data pointer")
        graph = make_fx(fn, tracing_mode=mode)(*first)
    assert all(torch.equal(a, b) for a, b in zip(_list(graph(*second)), _list(fn(*second)), strict=True))


def test_gradient_transforms_are_refused(cuda_dev):
    c = _inputs(3)
    calls = [(lambda x: afb.int8_linear(x, c["up"]), c["x"]), (afb.gelu_int8, c["x"]),
             (lambda y: afb.sandwich_norm(y, c["r"], c["gate"], c["w"], c["w"]), c["y"])]
    for fn, at in calls:
        with pytest.raises(RuntimeError, match="no gradient under torch.func transforms"):
            torch.func.grad(lambda t: _list(fn(t))[0].float().sum())(at)


@pytest.mark.parametrize("name", list(CALLS))
def test_vmap(name, cuda_dev):
    """Over samples of their own, or refused."""
    fn, args = CALLS[name]
    calls = [args(_inputs(s)) for s in (1, 2, 3)]
    stacked = [torch.stack(ts) for ts in zip(*calls)]
    try:
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            got = _list(torch.vmap(fn)(*stacked))
    except (RuntimeError, NotImplementedError) as e:
        print("refused:", e)
        assert "vmap" in str(e) or "functorch" in str(e), e
        return
    for k, c in enumerate(calls):
        assert all(torch.equal(a[k], b) for a, b in zip(got, _list(fn(*c)), strict=True))


@pytest.mark.parametrize("name", ["rowquant_int8", "int8_linear", "gelu_int8", "int8_wgrad", "sandwich_norm", "sandwich_norm_int8"])
def test_forward_mode_is_refused(name, cuda_dev):
    """Its tangents would be left out in silence."""
    fn, args = CALLS[name]
    t = args(_inputs(4))
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda x: fn(x, *t[1:]), t[:1], (torch.ones_like(t[0]),))
    with torch.autograd.forward_ad.dual_level():
        fn(*t)  # no tangents
        x = torch.autograd.forward_ad.make_dual(t[0], torch.ones_like(t[0]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            fn(x, *t[1:])


def test_batched_gradients_are_refused(cuda_dev):
    c = _inputs(6)
    x = c["x"].requires_grad_(True)
    y = afb.int8_linear(x, c["up"])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, torch.stack([c["dy"], 2 * c["dy"]]), is_grads_batched=True)


def test_saved_tensors_on_the_host(cuda_dev):
    c = _inputs(5)
    up, down = c["up"], c["down"]
    calls = [
        (lambda x: afb.int8_linear(x, up), [c["x"]]),
        (lambda y, r, g, w: afb.sandwich_norm(y, r, g, w, w)[0], [c["y"], c["r"], c["gate"], c["w"]]),
        (lambda x, a, b, d, e: afb.int8_lora_mlp(x, up, down, afb.LoRA(a, b), afb.LoRA(d, e)), [c["x"], *c["lora"]]),
    ]
    for fn, at in calls:
        leaves = [t.clone().requires_grad_(True) for t in at]
        out = fn(*leaves)
        g = torch.randn_like(out)
        want = torch.autograd.grad(out, leaves, g)
        with torch.autograd.graph.save_on_cpu():
            out = fn(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, g), want, strict=True))


@pytest.mark.parametrize("name", ["rowquant_int8", "int8_linear", "gelu_int8_bwd", "int8_wgrad", "sandwich_norm", "sandwich_norm_int8",
                                  "sandwich_norm_bwd"])
def test_compiled_code_with_permuted_inputs(name, cuda_dev):
    """Strides and values of compiled code, the backward pass's too, on inputs that are not contiguous."""
    fn, args = CALLS[name]
    at = [t.transpose(0, 1).contiguous().transpose(0, 1) if t.ndim > 1 else t for t in args(_inputs(8))]
    want = _list(fn(*at))
    got = _list(torch.compile(lambda *ts: [t + 0 for t in _list(fn(*ts))], backend="aot_eager", fullgraph=True)(*at))
    assert all(torch.equal(a, b) and a.stride() == b.stride() for a, b in zip(got, want, strict=True))
    if name == "sandwich_norm":
        grads = []
        for f in (fn, torch.compile(fn, backend="aot_eager", fullgraph=True)):
            leaves = [t.detach().requires_grad_(True) for t in at]
            h, z = f(*leaves)
            grads.append(torch.autograd.grad((h.float() * z.float()).sum(), leaves))
        assert all(torch.equal(a, b) for a, b in zip(*grads))

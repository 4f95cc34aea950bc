"""What the 8-bit linear, the 8-bit checkpoints and the sandwich norm refuse (CPU only)."""

from __future__ import annotations

import pytest
import torch

import anima_flat_b200 as afb
from anima_flat_b200 import _lib

FAKE = 4096  # a 16-byte aligned non-null address; validation rejects before any use
BF = torch.bfloat16


def _status(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.afb_last_error().decode()


@pytest.mark.parametrize("name,args,msg", [
    ("afb_rowquant_int8", (FAKE, None, FAKE, FAKE, 4, 24, 0, None), "K must be"),
    ("afb_rowquant_int8", (FAKE, None, FAKE, FAKE, 4, 16400, 0, None), "K must be"),
    ("afb_rowquant_int8", (FAKE, None, FAKE, FAKE, -1, 32, 0, None), "rows must be"),
    ("afb_rowquant_int8", (FAKE, None, FAKE, FAKE, 4, 32, 2, None), "dtype must be"),
    ("afb_rowquant_int8", (FAKE + 2, None, FAKE, FAKE, 4, 32, 0, None), "x is not 16-byte aligned"),
    ("afb_rowquant_int8", (FAKE, FAKE + 4, FAKE, FAKE, 4, 32, 0, None), "cols is not 16-byte aligned"),
    ("afb_gelu_int8", (FAKE, FAKE, FAKE, None, FAKE, 4, 32, 0, None), "c is null"),
    ("afb_gelu_int8_bwd", (None, FAKE, FAKE, FAKE, 4, 32, 0, None), "dy is null"),
    ("afb_int8_restore", (FAKE, FAKE + 2, FAKE, 4, 32, 0, None), "s is not 4-byte aligned"),
    ("afb_int8_linear", (FAKE, FAKE, FAKE, FAKE, None, FAKE, 4, 8, 24, 0, None), "K must be"),
    ("afb_int8_linear", (FAKE, FAKE, FAKE, FAKE, None, FAKE, 4, 8, 131088, 0, None), "K must be"),
    ("afb_int8_linear", (FAKE, FAKE, FAKE, FAKE, None, FAKE, 4, 0, 32, 0, None), "N must be"),
    ("afb_int8_linear", (FAKE, FAKE, FAKE, FAKE, FAKE + 1, FAKE, 4, 8, 32, 0, None), "bias is not"),
    ("afb_int8_linear", (FAKE + 8, FAKE, FAKE, FAKE, None, FAKE, 4, 8, 32, 0, None), "q is not 16-byte aligned"),
    ("afb_int8_wgrad", (FAKE, FAKE, FAKE, FAKE, 4, 0, 32, 0, None, 0, None), "N must be"),
    ("afb_int8_wgrad", (FAKE, FAKE, FAKE, FAKE, 4, 12, 32, 0, FAKE, 127, None), "workspace too small"),
    ("afb_int8_wgrad", (FAKE, FAKE, FAKE, FAKE, 4, 16, 40, 0, None, 0, None), "K must be"),
    ("afb_int8_wgrad", (FAKE, None, FAKE, FAKE, 4, 16, 32, 0, None, 0, None), "q is null"),
    ("afb_sandwich_norm", (*([FAKE] * 9), 1, 4, 20, 1.0, 1e-6, 0, None), "dim must be"),
    ("afb_sandwich_norm", (*([FAKE] * 9), 1, 4, 4104, 1.0, 1e-6, 0, None), "dim must be"),
    ("afb_sandwich_norm", (*([FAKE] * 7), None, FAKE, 1, 4, 64, 1.0, 1e-6, 0, None), "h is null"),
    ("afb_sandwich_norm", (FAKE, FAKE, FAKE + 2, *([FAKE] * 6), 1, 4, 64, 1.0, 1e-6, 0, None), "gate is not"),
    ("afb_sandwich_norm_int8", (*([FAKE] * 10), 65536, 4, 64, 1.0, 1e-6, 0, None), "batch must be"),
])
def test_c_entry_points_reject(name, args, msg):
    rc, said = _status(name, *args)
    assert rc == 1 and said.startswith(name) and msg in said


def test_backward_rejects_a_small_workspace():
    need = int(_lib.load().afb_sandwich_norm_bwd_workspace(2, 100, 64))
    assert need > 0 and need % (3 * 64 * 4) == 0
    rc, said = _status("afb_sandwich_norm_bwd", *([FAKE] * 15), 2, 100, 64, 1.0, 1e-6, 0, FAKE, need - 1, None)
    assert rc == 1 and "workspace too small" in said
    assert int(_lib.load().afb_sandwich_norm_bwd_workspace(2**40, 2**40, 64)) == 2**64 - 1


@pytest.mark.parametrize("name,args", [
    ("afb_rowquant_int8", (None, None, None, None, 0, 32, 0, None)),
    ("afb_gelu_int8", (None, None, None, None, None, 0, 32, 0, None)),
    ("afb_int8_linear", (None, None, None, None, None, None, 0, 8, 32, 0, None)),
    ("afb_sandwich_norm", (*([None] * 9), 0, 4, 64, 1.0, 1e-6, 0, None)),
    ("afb_sandwich_norm", (*([None] * 9), 4, 0, 64, 1.0, 1e-6, 0, None)),
])
def test_nothing_to_do(name, args):
    assert _status(name, *args)[0] == 0


def test_cpu_tensors_are_refused():
    x, q, s = torch.zeros(4, 32, dtype=BF), torch.zeros(4, 32, dtype=torch.int8), torch.ones(4, 1)
    w = afb.Int8Weight(torch.zeros(8, 32, dtype=torch.int8), torch.ones(8))
    y, f = torch.zeros(1, 4, 64, dtype=BF), torch.ones(64)
    for call in (lambda: afb.rowquant_int8(x), lambda: afb.int8_linear(x, w), lambda: afb.int8_linear((q, s), w),
                 lambda: afb.gelu_int8(x), lambda: afb.gelu_int8_bwd(x, q, s), lambda: afb.int8_restore(q, s),
                 lambda: afb.int8_wgrad(x, q, s), lambda: afb.sandwich_norm(y, y, None, f, f),
                 lambda: afb.sandwich_norm_int8(y, y, None, f, f), lambda: afb.sandwich_norm_bwd(y, None, y, y, None, f, f)):
        with pytest.raises(ValueError, match="CUDA tensors required"):
            call()


def test_fake_impls():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.anima_flat_b200
    with FakeTensorMode():
        x = torch.empty(2, 6, 64, dtype=BF, device="meta")
        wq, ws = torch.empty(40, 64, dtype=torch.int8, device="meta"), torch.empty(40, device="meta")
        q, s = ops.rowquant_int8(x)
        y = ops.int8_linear(x, wq, ws, None, None)
        yc = ops.int8_linear_codes(q, s, wq, ws, None, torch.float16)
        g = ops.gelu_int8(x)
        dx = ops.gelu_int8_bwd(x, g[2], g[3])
        r = ops.int8_restore(q, s, torch.float16)
        dw = ops.int8_wgrad(y, q, s)
        f = torch.empty(64, device="meta")
        h, z = ops.sandwich_norm(x, x, None, f, f, None, None, 1.0, 1e-6)
        hq, hs, _ = ops.sandwich_norm_int8(x, x, None, f, f, None, None, 1.0, 1e-6)
        b = ops.sandwich_norm_bwd(h, None, z, x, None, f, f, None, 1.0, 1e-6)
    assert q.shape == (2, 6, 64) and q.dtype == torch.int8 and s.shape == (12, 1)
    assert y.shape == yc.shape == (2, 6, 40) and y.dtype == BF and yc.dtype == torch.float16
    assert g[0].shape == g[2].shape == dx.shape == r.shape == (2, 6, 64) and g[3].shape == (12, 1)
    assert dw.shape == (40, 64) and dw.dtype == BF
    assert h.shape == z.shape == hq.shape == (2, 6, 64) and hs.shape == (12, 1)
    assert [tuple(t.shape) for t in b] == [(2, 6, 64)] * 2 + [(2, 64), (64,), (64,), (2, 64), (2, 64)]


@pytest.mark.gpu
def test_arguments_are_checked(cuda_dev):
    z = lambda *s, d=BF: torch.zeros(*s, dtype=d, device=cuda_dev)  # noqa: E731
    x, q, s = z(4, 32), z(4, 32, d=torch.int8), z(4, 1, d=torch.float32)
    w = afb.Int8Weight(z(8, 32, d=torch.int8), z(8, d=torch.float32))
    y, f = z(2, 4, 64), z(64, d=torch.float32)
    refused = [
        lambda: afb.rowquant_int8(x.float()), lambda: afb.rowquant_int8(z(4, 24)), lambda: afb.rowquant_int8(z(1, 16400)),
        lambda: afb.int8_linear(z(4, 48), w), lambda: afb.int8_linear(x, afb.Int8Weight(w.q.float(), w.s)),
        lambda: afb.int8_linear(x, afb.Int8Weight(w.q, w.s[:7])), lambda: afb.int8_linear(x, w, z(7)),
        lambda: afb.int8_linear(x, w, z(8, d=torch.float16)), lambda: afb.int8_linear((q, s[:3]), w),
        lambda: afb.int8_linear((q, s), w, dtype=torch.float32), lambda: afb.int8_linear((x, s), w),
        lambda: afb.int8_linear(x.clone().requires_grad_(True), w), lambda: afb.int8_linear(x, w, z(8).requires_grad_(True)),
        lambda: afb.quantize_weight_int8(z(8, 32), backward=True), lambda: afb.quantize_weight_int8(z(1, 8, 32)),
        lambda: afb.gelu_int8_bwd(z(4, 48), q, s), lambda: afb.int8_restore(q, s, torch.float32),
        lambda: afb.int8_wgrad(z(5, 8), q, s), lambda: afb.int8_wgrad(z(4, 8, d=torch.float32), q, s),
        lambda: afb.sandwich_norm(y, z(2, 4, 32), None, f, f), lambda: afb.sandwich_norm(y, y.half(), None, f, f),
        lambda: afb.sandwich_norm(y, y, z(2, 32), f, f), lambda: afb.sandwich_norm(y, y, None, f[:63], f),
        lambda: afb.sandwich_norm(y, y, z(2, 64, d=torch.float32), f, f), lambda: afb.sandwich_norm(y[0], y[0], None, f, f),
        lambda: afb.sandwich_norm(z(1, 1, 20), z(1, 1, 20), None, z(20), z(20)),
        lambda: afb.sandwich_norm_bwd(y, y[:1], y, y, None, f, f),
        lambda: afb.rowquant_int8(x.cpu()), lambda: afb.int8_linear(x, afb.Int8Weight(w.q.cpu(), w.s)),
    ]
    for k, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {k} was not refused")

"""Which calls of the 8-bit and sandwich-norm ops go past torch's dispatcher (CPU only)."""

from __future__ import annotations

import pytest
import torch

from anima_flat_b200.kernels.common import _plain


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_tracing_takes_the_registered_ops():
    seen = []
    x = torch.zeros(2, 16)
    torch.jit.trace(lambda t: (seen.append(_plain(t)), t + 1)[1], (x,), check_trace=False)
    assert seen == [False] and _plain(x)

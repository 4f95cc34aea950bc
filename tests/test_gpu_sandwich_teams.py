"""sandwich_norm's forward on either side of the choice between groups of warps and teams, and with every number of teams.

The bounds are those of the other sandwich tests.
"""

from __future__ import annotations

import pytest
import torch

import anima_flat_b200 as afb
from tests.test_gpu_sandwich import BF, HF, TINY, U, _call, _case, _h64, _within, _z64

pytestmark = pytest.mark.gpu

# (samples, rows, columns): 8 teams of short rows, idle lanes in several teams, 5 to 2
# teams and one; one block a sample, and more samples than multiprocessors with
# one row, a few, and many each.
SHAPES = [(1, 8192, 512), (1, 8189, 520), (3, 5501, 264), (1, 70001, 64), (2, 2700, 776), (2, 601, 1024), (1, 701, 1032),
          (1, 411, 1288), (1, 300, 1800), (5, 77, 2040), (1, 131, 4088), (100, 41, 1024), (140, 31, 2048), (200, 3, 1024),
          (149, 30, 2048), (256, 16, 1152), (256, 64, 1032), (300, 25, 2048), (300, 23, 4096), (1024, 1, 2048),
          (2100, 1, 520), (1024, 17, 264), (1030, 33, 512)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("B,S,D", SHAPES)
def test_forward(B, S, D, dt, cuda_dev):
    c = _case(B, S, D, dt, B + S + D)
    h, z = _call(c)
    a, b = _z64(c)
    _within(z, a + b, U[dt] * (a + b).abs() + 2.0**-18 * (a.abs() + b.abs()) + TINY[dt])
    a, b = _h64(c, z)
    _within(h, a + b, U[dt] * (a + b).abs() + 2.0**-18 * (a.abs() + b.abs()) + TINY[dt])


@pytest.mark.parametrize("B,S,D", SHAPES)
def test_codes(B, S, D, cuda_dev):
    c = _case(B, S, D, BF, 7 + D)
    q, s, z = _call(c, afb.sandwich_norm_int8)
    a, b = _z64(c)
    _within(z, a + b, U[BF] * (a + b).abs() + 2.0**-18 * (a.abs() + b.abs()) + TINY[BF])
    a, b = _h64(c, z)
    h, err = (a + b).view(-1, D), 2.0**-18 * (a.abs() + b.abs()).view(-1, D)
    top = h.abs().amax(1, keepdim=True)
    _within(s, top / 127.0, err.amax(1, keepdim=True) / 127.0 + 2.0**-23 * top)
    _within(q.view(-1, D).double() * s.double(), h, 0.5001 * s.double() + 2 * err.amax(1, keepdim=True))


def _time(fn):
    """Milliseconds of 20 calls in a graph, the least of five."""
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        fn()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(20):
            fn()
    best = float("inf")
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("fn", [afb.sandwich_norm, afb.sandwich_norm_int8])
def test_short_samples_cost_what_their_rows_do(fn, cuda_dev):
    """4096 rows of 4096 samples read 1.75 times the bytes of 4096 rows of one: no 4 times the time."""
    times = [_time(lambda c=_case(B, S, 2048, BF, 1): _call(c, fn)) for B, S in ((1, 4096), (4096, 1))]
    assert times[1] <= 4 * times[0]

"""Order on the device: bounded steps planned, called, planned again and captured on several streams, whose
work waits long enough that a missing dependency would show. Results are compared bit for bit with the same
calls one after the other, or with the 64-bit oracle under the tolerances of test_gpu_bounded.py."""

from __future__ import annotations

import pytest

from gpu_util import torch_cuda
from test_gpu_bounded import Case

pytestmark = pytest.mark.gpu

SHAPES = [("bf16", 8, 2, 128, 16), ("fp32", 8, 2, 64, 16)]
BUSY = 40_000_000  # clocks that a stream is kept waiting: 20 ms and more


def _shape(s):
    return "-".join(map(str, s))


def _busy(stream):
    torch = torch_cuda()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(BUSY)


@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("shape", SHAPES, ids=_shape)
def test_the_first_call_on_another_stream_follows_the_tables(shape, weights):
    """The tables are uploaded on the stream that made the batch, behind what is queued there."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch

    c = Case(*shape, [100, 333, 40, 700], [1, 1, 80, 5], window=60, sinks=4, weights=weights)
    PagedBatch(c.pool, [t[::-1].copy() for t in c.tables], c.starts, c.new, window=60)  # leaves a handle with other tables
    planning, running = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    _busy(planning)
    with torch.cuda.stream(planning):
        b = c.batch()
    with torch.cuda.stream(running):
        out = b.write_and_attend(0, c.q, c.k, c.v)
    torch.cuda.synchronize()
    b.check()
    c.check(out)

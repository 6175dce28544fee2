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


@pytest.mark.parametrize("shape", SHAPES, ids=_shape)
def test_calls_of_one_batch_on_several_streams(shape):
    """They share scores, statistics, partials and counters: as one after the other, here with split keys,
    chunks and weights, the last call's in the end."""
    torch = torch_cuda()
    c = Case(*shape, [9000, 40, 700, 90], [1, 60, 5, 300], window=5000, sinks=4, weights="replace")
    b = c.batch()
    qs = [c.q] + [torch.randn_like(c.q) for _ in range(3)]
    want = []
    for q in qs:
        want.append(b.write_and_attend(0, q, c.k, c.v))
    weights = c.pool.weights.clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    _busy(streams[0])
    got = []
    for q, s in zip(qs, streams):
        with torch.cuda.stream(s):
            got.append(b.write_and_attend(0, q, c.k, c.v))
    torch.cuda.synchronize()
    b.check()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    assert torch.equal(c.pool.weights, weights)
    c.q = qs[-1]
    c.check(got[-1])


@pytest.mark.parametrize("shape", SHAPES, ids=_shape)
def test_a_new_plan_follows_the_calls_before_it(shape):
    """Other n_heads, and a recycled handle that is planned on a second stream and called on a third:
    calls that wait on the first stream still have their own tables, plan and scratch."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch

    c = Case(*shape, [9000, 40, 700], [1, 60, 5], window=5000, sinks=4, poison=False)
    q2 = torch.randn((c.q.shape[0], 2 * c.H, c.D), device="cuda", dtype=c.q.dtype)
    other = dict(starts=[300, 20], n_new=[3, 70], window=90, sinks=1)
    tables = [c.tables[0][-30:], c.tables[2]]
    q3 = torch.randn((73, c.H, c.D), device="cuda", dtype=c.q.dtype)

    def steps(streams):
        b = c.batch()
        b.attend(0, c.q)
        torch.cuda.synchronize()
        if streams[0] is not streams[1]:
            _busy(streams[0])
        outs = []
        for q, s in ((c.q, streams[0]), (q2, streams[1])):
            with torch.cuda.stream(s):
                outs.append(b.attend(0, q))
        del b  # its handle goes to the next batch
        with torch.cuda.stream(streams[2]):
            n = PagedBatch(c.pool, tables, **other)
        with torch.cuda.stream(streams[3]):
            outs.append(n.attend(0, q3))
        torch.cuda.synchronize()
        n.check()
        return outs

    c.run()
    now = torch.cuda.current_stream()
    want = steps([now] * 4)
    got = steps([torch.cuda.Stream() for _ in range(4)])
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("what", ["capture", "head_dim"])
def test_refused_evictions_leave_the_tables_alone(what):
    """What pool.evict refuses for good, evict_sequences refuses before the manager's tables change."""
    torch = torch_cuda()
    from gpu_util import Shape
    from pagellm_b200 import _lib
    from pagellm_b200.cache import BlockManager, PagedKVPool, evict_sequences

    pool = PagedKVPool(Shape(1, 1, 32 if what == "capture" else 513), 8, 16, track_weights=True)
    bm = BlockManager(8, 16, enable_prefix_caching=False)
    bm.allocate(1, list(range(100)))
    bm.fork(1, 2)
    before = bm.block_table(1), bm.block_table(2), bm.alloc.num_free
    with pytest.raises(_lib.PagedKVError, match="captured" if what == "capture" else "head_dim"):
        if what == "capture":
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                evict_sequences(pool, bm, [1, 2], [100, 100], 10)
        else:
            evict_sequences(pool, bm, [1, 2], [100, 100], 10)
    torch.cuda.synchronize()
    assert (bm.block_table(1), bm.block_table(2), bm.alloc.num_free) == before
    if what == "capture":
        bm.free(2)
        assert evict_sequences(pool, bm, [1], [100], 10).tolist() == [10]


def _until(condition):
    """A destroyed graph's end is counted a moment later, by a thread of CUDA's."""
    import time

    for _ in range(200):
        if condition():
            return True
        time.sleep(0.01)
    return False


@pytest.mark.parametrize("shape", SHAPES, ids=_shape)
def test_a_live_graph_keeps_the_plan_it_reads(shape):
    """A graph holds addresses of its batch's tables, plan and scratch: they stay until it is gone, whether
    the batch lives on, is asked for other heads, or is dropped and others are made."""
    torch = torch_cuda()
    from pagellm_b200 import _lib
    from pagellm_b200.cache import PagedBatch

    c = Case(*shape, [4000, 40, 300], [1, 60, 5], window=500, sinks=4, weights="replace")
    b = c.batch()
    want = c.run(b).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b.write_and_attend(0, c.q, c.k, c.v)
        got = b.write_and_attend(0, c.q, c.k, c.v)
    handle = b._b
    assert c.pool._graphs_of(handle) == 1
    q2 = torch.cat([c.q, c.q], 1)
    with pytest.raises(_lib.PagedKVError, match="graph"):
        b.attend(0, q2)
    assert torch.equal(c.run(b), want)  # the plan is as it was
    del b
    others = []
    for _ in range(3):  # none of them gets the graph's handle
        others.append(PagedBatch(c.pool, [c.tables[0]], [1000], [3], window=50))
        others[-1].attend(0, q2[:3])
    assert handle not in [o._b for o in others] and handle in c.pool._held_batches
    for _ in range(2):
        got.zero_()
        c.pool.weights.copy_(c.before)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        c.check(got)
    del graph
    assert _until(lambda: c.pool._graphs_of(handle) == 0)
    again = c.batch()
    assert not c.pool._held_batches
    c.check(again.write_and_attend(0, c.q, c.k, c.v))


def test_a_failed_capture_keeps_nothing():
    torch = torch_cuda()
    c = Case("bf16", 8, 2, 128, 16, [100], [1], window=40)
    b = c.batch()
    c.run(b)
    with pytest.raises(RuntimeError, match="on purpose"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.write_and_attend(0, c.q, c.k, c.v)
            raise RuntimeError("on purpose")
    torch.cuda.synchronize()
    assert _until(lambda: c.pool._graphs_of(b._b) == 0)
    q2 = torch.cat([c.q, c.q], 1)
    b.attend(0, q2)
    c.check(c.run(b))


@pytest.mark.parametrize("shape", SHAPES, ids=_shape)
def test_a_new_stream_under_a_destroyed_ones_handle(shape):
    """A destroyed stream's work goes on; the next stream may get its handle, not its place in the order."""
    torch = torch_cuda()
    import ctypes

    c = Case(*shape, [9000, 40], [1, 60], window=5000, sinks=4, weights="replace")
    b = c.batch()
    qs = [c.q, torch.randn_like(c.q)]
    want = [b.write_and_attend(0, q, c.k, c.v) for q in qs]
    torch.cuda.synchronize()
    rt = torch.cuda.cudart()

    def create():
        h = ctypes.c_void_p()
        assert int(rt.cudaStreamCreate(ctypes.addressof(h))) == 0
        return h.value

    for _ in range(4):
        first = create()
        with torch.cuda.stream(torch.cuda.ExternalStream(first)):
            torch.cuda._sleep(BUSY)
            got = [b.write_and_attend(0, qs[0], c.k, c.v)]
        assert int(rt.cudaStreamDestroy(first)) == 0
        second = create()
        with torch.cuda.stream(torch.cuda.ExternalStream(second)):
            got.append(b.write_and_attend(0, qs[1], c.k, c.v))
        torch.cuda.synchronize()
        assert int(rt.cudaStreamDestroy(second)) == 0
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        if second == first:
            break
    b.check()


def test_a_batch_is_made_before_a_capture():
    """The refusal leaves the handle fit: its events belong to no capture."""
    torch = torch_cuda()
    from pagellm_b200 import _lib
    from pagellm_b200.cache import PagedBatch

    c = Case("bf16", 8, 2, 128, 16, [100], [1], window=40)
    c.run()
    for kw in (dict(window=40), {}):  # the second: a plain step on a handle that ran a bounded one
        with pytest.raises(_lib.PagedKVError, match="capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                PagedBatch(c.pool, c.tables, c.starts, c.new, **kw)
        torch.cuda.synchronize()
        c.check(c.run())


def test_a_plain_graph_keeps_its_dropped_batch():
    """Plain steps too: a graph goes on replaying after its batch was dropped, others made and the pool trimmed."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch

    c = Case("bf16", 8, 2, 128, 16, [700, 300, 90], [1, 1, 80], window=40, poison=False)
    q, k, v = c.q.float(), c.k.float(), c.v.float()
    b = PagedBatch(c.pool, c.tables, c.starts, c.new)
    want = b.write_and_attend(0, q, k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b.write_and_attend(0, q, k, v)
    handle = b._b
    del b
    for kw in ({}, dict(window=33)):
        other = PagedBatch(c.pool, [c.tables[1], c.tables[0]], [200, 9], [1, 70], **kw)
        assert other._b != handle
        other.attend(0, q[:71])
        del other
    assert c.pool.trim() > 0 and c.pool._held_batches == [handle]
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del graph
    assert _until(lambda: c.pool._graphs_of(handle) == 0)
    again = PagedBatch(c.pool, c.tables, c.starts, c.new)
    assert again._b == handle and torch.equal(again.write_and_attend(0, q, k, v), want)


def test_prefix_sharing_does_not_unmake_a_bounded_plan():
    torch = torch_cuda()
    c = Case("bf16", 8, 2, 128, 16, [100, 40], [1, 5], window=40, sinks=2)
    b = c.batch()
    want = c.run(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b.write_and_attend(0, c.q, c.k, c.v)
    b.prefix_sharing = "off"
    assert torch.equal(c.run(b), want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_host_rows_follow_the_tables_too():
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch

    c = Case("fp32", 8, 2, 64, 16, [100, 333, 40], [1, 1, 80], window=60, sinks=4, weights="replace")
    PagedBatch(c.pool, [t[::-1].copy() for t in c.tables], c.starts, c.new, window=60)
    planning, running = torch.cuda.Stream(), torch.cuda.Stream()
    rows = [x.cpu().numpy() for x in (c.q, c.k, c.v)]
    torch.cuda.synchronize()
    _busy(planning)
    with torch.cuda.stream(planning):
        b = c.batch()
    with torch.cuda.stream(running):
        out = b.write_and_attend(0, *rows)
    b.check()
    c.check(torch.from_numpy(out))


@pytest.mark.parametrize("bounds, weights", [((60, 4), None), ((60, 4), "replace"), ((None, 0), "replace")])
@pytest.mark.parametrize("shape", SHAPES + [("bf16", 10, 2, 64, 16)], ids=_shape)
def test_the_head_exchange_takes_bounded_steps(shape, bounds, weights):
    """One rank, whose slice is the whole result: on the planning stream and on another."""
    torch = torch_cuda()
    import ctypes as C

    from pagellm_b200 import _lib
    from pagellm_b200.cache.paged import _CudaArray

    lib = _lib.load()
    c = Case(*shape, [100, 333, 40], [1, 1, 80], window=bounds[0], sinks=bounds[1], weights=weights, io="fp32")
    b = c.batch()
    want = c.run(b)
    gather, own, res = C.c_void_p(), C.create_string_buffer(64), C.c_void_p()
    _lib.check(lib.pk_peer_gather_create(0, 1, 0, 1 << 22, C.byref(gather)))
    try:
        _lib.check(lib.pk_peer_gather_handle(gather, own))
        _lib.check(lib.pk_peer_gather_open(gather, own.raw))
        for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
            torch.cuda.synchronize()
            if weights:
                c.pool.weights.copy_(c.before)
                torch.cuda.synchronize()
            _lib.check(lib.pk_peer_gather_write_and_attend(gather, b._b, 0, c.H, c.q.data_ptr(), c.k.data_ptr(),
                                                           c.v.data_ptr(), C.byref(res), stream.cuda_stream))
            _lib.check(lib.pk_peer_gather_check(gather, stream.cuda_stream))
            got = torch.as_tensor(_CudaArray(res.value, c.q.shape, "<f4", None), device="cuda")
            assert torch.equal(got, want)
            c.check(got, q_step=2.0 ** -8 if shape[0] == "bf16" else 0.0)
    finally:
        _lib.check(lib.pk_peer_gather_destroy(gather))

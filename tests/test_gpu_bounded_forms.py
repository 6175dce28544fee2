"""The forms that a bounded step takes besides the ordinary ones: register tiles on the CUDA cores,
split keys, long contexts with few KV heads, weights summed from many units, steps on several streams
and in captured graphs. Same oracle, same tolerances as the steps of test_gpu_bounded."""

from __future__ import annotations

import numpy as np
import pytest

from gpu_util import Shape, torch_cuda
from test_gpu_bounded import Case

pytestmark = pytest.mark.gpu


def _shape(s):
    return "-".join(map(str, s))


TILES = [("fp32", 16, 8, 128, 16), ("fp32", 64, 1, 32, 8), ("fp32", 33, 1, 64, 16), ("fp32", 6, 2, 96, 5),
         ("fp32", 4, 4, 256, 16), ("fp32", 8, 2, 100, 48), ("fp32", 4, 2, 4, 1), ("bf16", 8, 2, 48, 16),
         ("bf16", 9, 3, 132, 7), ("bf16", 16, 1, 252, 200)]


@pytest.mark.parametrize("bounds", [(None, 0), (50, 3), (64, 70), (1, 1)])
@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("shape", TILES, ids=_shape)
def test_chunks_in_register_tiles(shape, weights, bounds):
    """Sequences on both sides of the tiles' smallest size, beside rows alone and none."""
    c = Case(*shape, [0, 200, 77, 5, 64, 129], [100, 33, 0, 1, 64, 7], window=bounds[0], sinks=bounds[1], weights=weights)
    c.check(c.run())


@pytest.mark.parametrize("weights", [None, "replace"])
@pytest.mark.parametrize("shape", [("fp32", 65, 1, 64, 16), ("fp32", 4, 2, 260, 16), ("fp32", 3, 1, 17, 5),
                                   ("fp32", 2, 1, 512, 16), ("bf16", 5, 1, 33, 16)], ids=_shape)
def test_chunks_that_tiles_do_not_take(shape, weights):
    c = Case(*shape, [0, 90], [40, 21], window=60, sinks=3, weights=weights)
    c.check(c.run())


@pytest.mark.parametrize("rows_io", ["bf16", "fp32"])
def test_tiles_read_both_types_of_rows(rows_io):
    c = Case("bf16", 8, 2, 48, 16, [30, 300], [70, 20], window=90, sinks=2, weights="add", io=rows_io)
    c.check(c.run())


@pytest.mark.parametrize("bounds", [(None, 0), (5000, 4)])
@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("shape, starts, new", [
    (("fp32", 4, 1, 64, 16), [9000], [16]),            # tiles, keys split
    (("fp32", 4, 1, 64, 16), [0, 20], [700, 9]),       # the weights' columns dealt to several CTAs
    (("fp32", 4, 1, 64, 16), [9000, 3], [1, 1]),       # rows, keys split
    (("fp32", 16, 1, 128, 16), [9000], [1]),
    (("fp32", 4, 1, 64, 16), [9000, 4000], [16, 2]),   # both in one step
    (("bf16", 4, 2, 48, 16), [9000, 8000], [1, 30])], ids=str)
def test_long_contexts_on_the_cuda_cores(shape, starts, new, weights, bounds):
    c = Case(*shape, starts, new, window=bounds[0], sinks=bounds[1], weights=weights)
    c.check(c.run())


@pytest.mark.parametrize("bounds", [(None, 0), (20000, 4)])
@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("H, new", [(8, 33), (16, 129), (4, 300)])
def test_chunks_of_few_kv_heads_behind_long_contexts(H, new, weights, bounds):
    c = Case("bf16", H, 1, 128, 16, [30000], [new], window=bounds[0], sinks=bounds[1], weights=weights, poison=False)
    c.check(c.run())


@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("shape", [("bf16", 8, 2, 128, 128), ("bf16", 32, 1, 128, 16), ("bf16", 8, 8, 128, 32),
                                   ("bf16", 64, 2, 128, 64)], ids=_shape)
@pytest.mark.parametrize("bounds", [(None, 0), (130, 3), (1, 129)])
def test_chunks_beside_decodes(shape, weights, bounds):
    c = Case(*shape, [0, 500, 127, 128, 0, 3], [200, 1, 1, 300, 0, 5], window=bounds[0], sinks=bounds[1], weights=weights)
    c.check(c.run())


@pytest.mark.parametrize("mode", ["add", "replace"])
@pytest.mark.parametrize("shape", [("bf16", 16, 4, 64, 16), ("bf16", 24, 8, 128, 16), ("bf16", 10, 2, 128, 32)], ids=_shape)
def test_weights_of_sequences_in_many_units(shape, mode):
    c = Case(*shape, [0, 100, 7], [300, 40, 1], window=150, sinks=2, weights=mode)
    c.check(c.run())


def test_rows_of_every_magnitude():
    """Scores up to some hundreds either way: the softmax ends on few keys, and earlier maxima fade."""
    for dtype in ("fp32", "bf16"):
        c = Case(dtype, 8, 2, 128, 16, [40, 300], [80, 1], window=70, sinks=2, q_scale=30.0)
        c.check(c.run())


@pytest.mark.parametrize("shape", [("fp32", 4, 1, 64, 16), ("bf16", 8, 1, 128, 16)], ids=_shape)
def test_split_steps_captured_and_repeated(shape):
    """Counters and partials of split keys are ready again after each replay."""
    torch = torch_cuda()
    c = Case(*shape, [9000, 40], [40, 1], window=8000, sinks=4, weights="replace")
    b = c.batch()
    eager, weights = c.run(b).clone(), c.pool.weights.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b.write_and_attend(0, c.q, c.k, c.v)
    for _ in range(3):
        got.zero_()
        c.pool.weights.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        touched = c.pool.weights != 0
        assert torch.equal(c.pool.weights[touched], weights[touched])
        assert bool((~touched | (weights != 0)).all())
    b.check()
    # and the handle runs eagerly again
    c.pool.weights.copy_(c.before)
    c.check(c.run(b))


@pytest.mark.parametrize("shape", [("fp32", 8, 2, 128, 16), ("bf16", 8, 2, 128, 16)], ids=_shape)
def test_two_steps_of_one_pool_at_once(shape):
    """Two handles with sequences of their own, on two streams: as one after the other."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch

    c = Case(*shape, [3000, 1000, 40, 600], [1, 90, 60, 1], window=800, sinks=4, weights="add")
    c.check(c.run())
    halves = []
    for ids in ((0, 1), (2, 3)):
        rows = torch.cat([torch.arange(c.rows(i).start, c.rows(i).stop) for i in ids]).cuda()
        halves.append((PagedBatch(c.pool, [c.tables[i] for i in ids], c.starts[list(ids)], c.new[list(ids)], window=800,
                                  sinks=4, weights="add"), rows, [x[rows].contiguous() for x in (c.q, c.k, c.v)]))
    one, weights = [], []
    for turn in range(4):
        c.pool.weights.copy_(c.before)
        torch.cuda.synchronize()
        outs, streams = [], []
        for b, _, (q, k, v) in halves:
            s = torch.cuda.Stream() if turn else torch.cuda.current_stream()
            with torch.cuda.stream(s):
                outs.append(b.write_and_attend(0, q, k, v))
            streams.append(s)
        torch.cuda.synchronize()
        one.append(torch.cat(outs))
        weights.append(c.pool.weights.clone())
    for x in range(1, 4):
        assert torch.equal(one[x], one[0]) and torch.equal(weights[x], weights[0])
    order = torch.argsort(torch.cat([r for _, r, _ in halves]))
    c.pool.weights.copy_(weights[0])
    c.check(one[0][order])


def test_many_layers_share_a_plan():
    """One plan, a call per layer, each with its own weights."""
    torch = torch_cuda()
    c = Case("fp32", 8, 2, 64, 16, [700, 30], [40, 1], window=300, sinks=2, weights="add", layers=3, layer=1)
    b = c.batch()
    before = c.pool.weights.clone()
    c.check(c.run(b))
    assert torch.equal(c.pool.weights[0], before[0]) and torch.equal(c.pool.weights[2], before[2])
    for layer in (0, 2):
        c.layer, c.before = layer, c.pool.weights.clone()
        c.check(c.run(b))


def test_a_pool_of_numpy_rows_in_tiles():
    """Host rows go the same way."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    rng = np.random.default_rng(3)
    q = rng.standard_normal((50, 4, 32)).astype(np.float32)
    k, v = (rng.standard_normal((50, 2, 32)).astype(np.float32) for _ in range(2))
    pools = [PagedKVPool(Shape(1, 2, 32), 8, 8, track_weights=True) for _ in range(2)]
    outs = []
    for pool, rows in zip(pools, ((q, k, v), [torch.as_tensor(x).cuda() for x in (q, k, v)])):
        outs.append(PagedBatch(pool, [list(range(7))], [0], [50], window=20, sinks=1, weights="add").write_and_attend(0, *rows))
    assert isinstance(outs[0], np.ndarray) and np.array_equal(outs[0], outs[1].cpu().numpy())
    assert torch.equal(pools[0].weights, pools[1].weights)


def test_positions_near_the_end_of_32_bits_are_refused():
    """Kernels step through positions in 32 bits; the last 65536 of them are not given out."""
    from pagellm_b200 import _lib
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    pool = PagedKVPool(Shape(1, 1, 4), 1, 16, track_weights=True)
    for n in (2 ** 31 - 2, 2 ** 31 - 65536):
        with pytest.raises(_lib.PagedKVError, match="too long"):
            PagedBatch(pool, [[0]], [n - 1], [1], window=4)
        with pytest.raises(_lib.PagedKVError, match="too long"):
            pool.evict([[0]], [n], 4)


def _evictable(n=8, length=700, bs=16):
    from pagellm_b200.cache import PagedKVPool

    torch = torch_cuda()
    nb = -(-length // bs)
    pool = PagedKVPool(Shape(2, 2, 64), n * nb, bs, track_weights=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    for x in (pool.k, pool.v, pool.weights):
        x.normal_(generator=g)
    pool.weights.abs_()
    return pool, [list(range(i * nb, (i + 1) * nb)) for i in range(n)]


def test_evict_with_a_budget_beyond_every_sequence():
    torch = torch_cuda()
    pool, tables = _evictable()
    k, w = pool.k.clone(), pool.weights.clone()
    for budget in (700, 2 ** 31 - 1):
        assert pool.evict(tables, [700, 0, 1, 16, 333, 700, 699, 2], budget, sinks=4, recent=100).tolist() \
            == [700, 0, 1, 16, 333, 700, 699, 2]
        assert torch.equal(pool.k, k) and torch.equal(pool.weights, w)


def test_evictions_from_several_threads():
    """Each thread shortens its own sequences on its own stream, as one call after the other."""
    import threading

    torch = torch_cuda()
    pool, tables = _evictable(16)
    before = [x.clone() for x in (pool.k, pool.v, pool.weights)]
    for t in tables:
        pool.evict([t], [700], 100, sinks=2, recent=10)
    want = [x.clone() for x in (pool.k, pool.v, pool.weights)]
    for x, y in zip((pool.k, pool.v, pool.weights), before):
        x.copy_(y)
    torch.cuda.synchronize()

    def work(mine):
        with torch.cuda.stream(torch.cuda.Stream()):
            for t in mine:
                pool.evict([t], [700], 100, sinks=2, recent=10)

    threads = [threading.Thread(target=work, args=(tables[i::4],)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for x, y in zip((pool.k, pool.v, pool.weights), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("mode", ["add", "replace"])
@pytest.mark.parametrize("shape", [("fp32", 16, 8, 64, 8), ("fp32", 8, 1, 128, 16), ("fp32", 10, 2, 64, 16),
                                   ("bf16", 40, 8, 128, 64)], ids=_shape)
def test_weights_of_few_columns(shape, mode):
    """Rows on one kernel, their weights on another: by rows or in tiles, side by side in one step."""
    c = Case(*shape, [150, 90, 333, 0, 64], [7, 1, 1, 19, 4], window=120, sinks=2, weights=mode)
    c.check(c.run())


@pytest.mark.parametrize("dtype, D", [("bfloat16", 513), ("bfloat16", 2051), (np.float32, 1024), (np.float32, 2050)])
def test_head_sizes_beyond_the_kernels_are_refused(dtype, D):
    torch = torch_cuda()
    from pagellm_b200 import _lib
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    pool = PagedKVPool(Shape(1, 1, D), 2, 16, dtype, track_weights=True)
    with pytest.raises(_lib.PagedKVError, match="head_dim"):
        pool.evict([[0]], [9], 4)
    x = torch.zeros((1, 1, D), device="cuda")
    with pytest.raises(_lib.PagedKVError, match="head_dim"):
        PagedBatch(pool, [[0]], [3], [1], window=2).write_and_attend(0, x, x, x)
    assert not bool(pool.k.any())


@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("shape, new", [(("bf16", 8, 8, 128, 16), 33), (("bf16", 1, 1, 128, 128), 40),
                                        (("bf16", 128, 1, 128, 16), 1), (("bf16", 128, 1, 128, 32), 3)], ids=str)
def test_chunks_smaller_than_a_query_tile(shape, new, weights):
    """A step of fewer rows than one query tile has tokens, and one token that fills it."""
    c = Case(*shape, [100], [new], window=77, sinks=2, weights=weights)
    c.check(c.run())


@pytest.mark.parametrize("bounds", [(None, 0), (70, 3), (1, 40), (33, 100)])
@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("shape", [("bf16", 32, 8, 128, 32), ("bf16", 40, 8, 128, 64), ("bf16", 16, 4, 256, 32),
                                   ("bf16", 8, 8, 128, 128), ("bf16", 6, 2, 256, 64), ("bf16", 16, 8, 128, 256),
                                   ("bf16", 8, 8, 64, 96)], ids=_shape)
def test_blocks_too_large_for_two_stages(shape, weights, bounds):
    """The split-KV kernel takes such blocks in parts."""
    c = Case(*shape, [0, 31, 300, 129, 64, 500], [1, 3, 1, 60, 0, 9], window=bounds[0], sinks=bounds[1], weights=weights)
    c.check(c.run())
    d = Case(*shape, [0, 31, 300, 64, 255, 256, 700], [1] * 7, window=bounds[0], sinks=bounds[1], weights=weights, seed=1)
    b = d.batch()
    d.check(d.run(b))
    if bounds[0] or weights:  # (a plain step has them on the CUDA cores)
        assert b.stats()["generic_rows"] == 0


@pytest.mark.parametrize("shape", [("bf16", 32, 8, 128, 32), ("bf16", 16, 8, 128, 64), ("bf16", 16, 4, 256, 32)], ids=_shape)
def test_parts_of_blocks_with_float_rows_layers_and_graphs(shape):
    torch = torch_cuda()
    for new in ([1, 1, 1, 1], [1, 70, 2, 0]):
        c = Case(*shape, [300, 31, 64, 5], new, window=90, sinks=3, weights="add", io="fp32", layers=2, layer=1)
        b = c.batch()
        # q at bf16 where the kernel has no room for its low half
        c.check(c.run(b), q_step=2.0 ** -8)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = b.write_and_attend(1, c.q, c.k, c.v)
        for _ in range(2):
            c.pool.weights.copy_(c.before)
            graph.replay()
            torch.cuda.synchronize()
            c.check(got, q_step=2.0 ** -8)
        b.check()


def test_batches_give_their_memory_back():
    """Every scratch of a batch goes with it: here split keys of tiles, weights in parts, kept scores and chunks."""
    torch = torch_cuda()
    from pagellm_b200 import _lib
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    lib = _lib.load()
    bf16 = PagedKVPool(Shape(1, 8, 128), 1100, 16, "bfloat16", track_weights=True)
    fp32 = PagedKVPool(Shape(1, 8, 128), 550, 16, track_weights=True)

    def round_trip():
        for pool, H, starts, new in ((fp32, 32, [8000], [64]), (fp32, 8, [8000], [1]), (bf16, 32, [8000, 8000], [64, 1])):
            nb = 550
            b = PagedBatch(pool, [list(range(i * nb, (i + 1) * nb)) for i in range(len(starts))], starts, new, weights="add")
            rows = sum(new)
            q, k = (torch.randn((rows, h, 128), device="cuda") for h in (H, 8))
            b.write_and_attend(0, q, k, k)
            b.check()
            del b
            for h in pool._idle_batches:
                assert lib.pk_batch_destroy(h) == 0
            pool._idle_batches.clear()
            pool._batch_bounds.clear()

    round_trip()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(6):
        round_trip()
    torch.cuda.synchronize()
    # the device allocates 2 MB at a time; one split-key scratch alone is more than 8
    assert free - torch.cuda.mem_get_info()[0] <= 4 << 20


def test_trim_gives_back_what_idle_batches_and_evictions_hold():
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch

    c = Case("bf16", 40, 8, 64, 16, [3000, 40], [300, 1], weights="replace", poison=False)
    out = c.run()  # 300 rows x 5 heads in units: scores of some 240 MB
    live = PagedBatch(c.pool, c.tables, c.starts, c.new, weights="replace")
    live.write_and_attend(0, c.q, c.k, c.v)
    other = PagedBatch(c.pool, c.tables, c.starts, c.new, window=70, sinks=1)
    other.write_and_attend(0, c.q, c.k, c.v)
    held = live.scratch_nbytes
    assert held > 150 << 20
    c.pool.evict(c.tables, c.starts + c.new, 900)
    del other
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    first = c.pool.trim()
    assert first > 0 and live.scratch_nbytes == held
    del live
    assert c.pool.trim() == held and c.pool.trim() == 0
    assert torch.cuda.mem_get_info()[0] - free >= held - (8 << 20)
    again = Case("bf16", 40, 8, 64, 16, [3000, 40], [300, 1], weights="replace", poison=False)
    again.pool.trim()
    assert torch.equal(again.run(), out)
    # plain, windowed and evicting calls go on after it
    b = PagedBatch(c.pool, [c.tables[1]], [10], [1], window=4)
    b.write_and_attend(0, c.q[:1], c.k[:1], c.v[:1])
    b.check()
    c.pool.evict([c.tables[1]], [11], 5)
    del b
    assert c.pool.trim() > 0


def test_batches_may_outlive_their_pool():
    """A pool closed before its last batch is dropped: the batch's memory goes without the pool's."""
    torch = torch_cuda()
    import gc

    gc.collect()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(4):
        c = Case("bf16", 40, 8, 64, 16, [3000], [100], weights="replace", poison=False)
        b = c.batch()
        b.write_and_attend(0, c.q, c.k, c.v)
        b.check()
        assert b.scratch_nbytes > 32 << 20
        c.pool.close()
        del b, c
        gc.collect()
    assert free - torch.cuda.mem_get_info()[0] <= 24 << 20  # (torch keeps some of the inputs' memory)


@pytest.mark.parametrize("in_place", [True, False])
def test_evictions_of_many_positions_take_the_layers_in_groups(in_place):
    """The scratch of kept positions stays small (175 MB here in one piece): as with the caller's own."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedKVPool

    layers, KVH, bs, n, budget = 37, 8, 16, 33000, 31000
    nb = -(-n // bs)
    lens = [n, 40, n - 100, n, 0]
    tables = [np.arange(i * nb, (i + 1) * nb, dtype=np.int32) for i in range(4)] + [np.zeros(0, np.int32)]
    new = None if in_place else [t + 4 * nb for t in tables]
    pool = PagedKVPool(Shape(layers, KVH, 2), (4 if in_place else 8) * nb, bs, "bfloat16", track_weights=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    state = (pool.k, pool.v, pool.weights)
    for x in state:
        x.normal_(generator=g)
    before = [x.clone() for x in state]
    kept = pool.evict(tables, lens, budget, sinks=4, recent=1000, new_tables=new, return_kept=True)[1]
    assert kept.numel() * 4 > 128 << 20
    del kept
    want = [x.clone() for x in state]
    assert not torch.equal(want[0], before[0])
    for x, y in zip(state, before):
        x.copy_(y)
    del before
    pool.trim()
    assert pool.evict(tables, lens, budget, sinks=4, recent=1000, new_tables=new).tolist() == [budget, 40, budget, budget, 0]
    for x, y in zip(state, want):
        assert torch.equal(x, y)
    assert 0 < pool.trim() <= (128 << 20) * 5 // 4  # (reserved with a quarter more)

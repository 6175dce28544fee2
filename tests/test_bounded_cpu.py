"""Bounded caches without a GPU: which blocks a windowed step reads, the checks of an eviction,
the block manager's side of it, and the refusals of the Python entry points."""

from __future__ import annotations

import ctypes as C
import random

import numpy as np
import pytest

from oracle import bounded_oracle as bo
from pagellm_b200 import _lib
from pagellm_b200.cache import BlockManager, OutOfBlocks, PagedBatch, evict_sequences


# ------------------------------------------------------------------ visible blocks
def _visible(q0, ctx, window, sinks, bs):
    out = (C.c_int64 * 3)()
    rc = _lib.load().pk_plan_visible_blocks(q0, ctx, window, sinks, bs, out)
    return rc, list(out)


@pytest.mark.parametrize("bs", [1, 4, 16])
def test_visible_blocks_are_those_with_a_visible_key(bs):
    rnd = random.Random(bs)
    for _ in range(600):
        q0 = rnd.randrange(0, 90)
        ctx = q0 + rnd.randrange(1, 12)
        window, sinks = rnd.choice([(0, 0), (rnd.randrange(1, 100), rnd.choice([0, 1, 3, 17, 200]))])
        rc, (head, skip, count) = _visible(q0, ctx, window, sinks, bs)
        assert rc == 0
        got = [x if x < head else x + skip for x in range(count)]
        want = set()
        for p in range(q0, ctx):
            want |= {int(j) // bs for j in bo.visible(p, window or None, sinks)}
        assert got == sorted(want), (q0, ctx, window, sinks)


def test_visible_blocks_of_the_longest_context():
    big = 2 ** 31 - 1
    assert _visible(big - 1, big, big, big, 16) == (0, [0, 0, 2 ** 27])
    rc, (head, skip, count) = _visible(big - 1, big, 1, 1, 16)
    assert rc == 0 and head == 1 and count == 2 and head + skip == 2 ** 27 - 1


@pytest.mark.parametrize("args", [(-1, 4, 0, 0, 16), (4, 4, 0, 0, 16), (0, 2 ** 31, 0, 0, 16), (0, 4, -1, 0, 16),
                                  (0, 4, 0, 1, 16), (0, 4, 2, -1, 16), (0, 4, 2, 1, 0)])
def test_visible_blocks_refuses(args):
    assert _visible(*args)[0] == _lib.PK_ERR_INVALID_ARG


# ------------------------------------------------------------------ eviction's checks
def _csr(tables):
    ip = np.zeros(len(tables) + 1, np.int64)
    np.cumsum([len(t) for t in tables], out=ip[1:])
    return ip, np.array([b for t in tables for b in t] or [0], np.int32)


def _plan_evict(tables, lengths, new, budget, sinks=0, recent=0, blocks=64, bs=4):
    ip, ids = _csr(tables)
    nip, nids = _csr(new)
    ln = np.array(lengths, np.int64)
    n = C.c_int64(-1)
    rc = _lib.load().pk_plan_evict(blocks, bs, len(lengths), ip.ctypes.data, ids.ctypes.data, ln.ctypes.data,
                                   nip.ctypes.data, nids.ctypes.data, budget, sinks, recent, C.byref(n))
    return rc, n.value


def test_evict_accepts_fresh_and_own_blocks():
    assert _plan_evict([[0, 1, 2]], [10], [[5, 6]], 8) == (0, 1)
    assert _plan_evict([[0, 1, 2]], [10], [[0, 1]], 8) == (0, 1)       # in place
    assert _plan_evict([[0, 1, 2]], [10], [[7, 1]], 8) == (0, 1)       # the first one fresh
    assert _plan_evict([[0, 1], [0, 2]], [8, 8], [[5], [6]], 4) == (0, 2)  # a shared source
    assert _plan_evict([[0, 1], [2, 3]], [8, 3], [[0], [2]], 4) == (0, 2)
    assert _plan_evict([], [], [], 4) == (0, 0)
    assert _plan_evict([[], [1]], [0, 4], [[], [1]], 4) == (0, 1)
    # pieces of 256 rows when fresh, one when in place
    t = list(range(200))
    assert _plan_evict([t], [800], [list(range(200, 350))], 600, blocks=400) == (0, 3)
    assert _plan_evict([t], [800], [t[:150]], 600, blocks=400) == (0, 1)


@pytest.mark.parametrize("call, code", [
    (dict(tables=[[0, 1]], lengths=[8], new=[[1]], budget=4), _lib.PK_ERR_INVALID_ARG),        # own, other index
    (dict(tables=[[0, 1], [2]], lengths=[8, 4], new=[[2], [2]], budget=4), _lib.PK_ERR_INVALID_ARG),
    (dict(tables=[[0, 1], [0, 2]], lengths=[8, 8], new=[[0], [5]], budget=4), _lib.PK_ERR_INVALID_ARG),  # shared
    (dict(tables=[[0, 0]], lengths=[8], new=[[0]], budget=4), _lib.PK_ERR_INVALID_ARG),        # twice in one table
    (dict(tables=[[0, 1], [2, 3]], lengths=[8, 8], new=[[5], [5]], budget=4), _lib.PK_ERR_INVALID_ARG),
    (dict(tables=[[0, 1], [2, 3]], lengths=[8, 8], new=[[2], [5]], budget=4), _lib.PK_ERR_INVALID_ARG),
    (dict(tables=[[0, 64]], lengths=[8], new=[[5]], budget=4), _lib.PK_ERR_OUT_OF_RANGE),
    (dict(tables=[[0, -1]], lengths=[8], new=[[5]], budget=4), _lib.PK_ERR_OUT_OF_RANGE),
    (dict(tables=[[0, 1]], lengths=[8], new=[[64]], budget=4), _lib.PK_ERR_OUT_OF_RANGE),
    (dict(tables=[[0, 1]], lengths=[9], new=[[5]], budget=4), _lib.PK_ERR_OUT_OF_RANGE),       # table too short
    (dict(tables=[[0, 1]], lengths=[8], new=[[5]], budget=5), _lib.PK_ERR_OUT_OF_RANGE),       # new table too short
    (dict(tables=[[0, 1]], lengths=[-1], new=[[5]], budget=4), _lib.PK_ERR_INVALID_ARG),
    (dict(tables=[[0, 1]], lengths=[8], new=[[5]], budget=0), _lib.PK_ERR_INVALID_ARG),
    (dict(tables=[[0, 1]], lengths=[8], new=[[5]], budget=4, sinks=3, recent=2), _lib.PK_ERR_INVALID_ARG),
    (dict(tables=[[0, 1]], lengths=[8], new=[[5]], budget=4, sinks=-1), _lib.PK_ERR_INVALID_ARG),
    (dict(tables=[[0, 1]], lengths=[8], new=[[5]], budget=4, recent=2 ** 62, sinks=4), _lib.PK_ERR_INVALID_ARG),
    (dict(tables=[[0, 1]], lengths=[8], new=[[5]], budget=2 ** 40), _lib.PK_ERR_UNSUPPORTED),
])
def test_evict_refuses(call, code):
    assert _plan_evict(**call)[0] == code, _lib.last_error()


def test_null_arguments():
    lib = _lib.load()
    assert lib.pk_pool_track_weights(None, None) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_pool_evict(None, 0, None, None, None, None, None, 4, 0, 0, None, None) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_batch_set_bounds(None, 0, 0, 0) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_batch_write_and_attend_bf16(None, 0, 1, None, None, None, None, None) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_plan_evict(8, 4, 1, None, None, None, None, None, 4, 0, 0, None) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_plan_evict(0, 4, 0, None, None, None, None, None, 4, 0, 0, None) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_bm_compact(None, 0, 0, None, 0, None) == _lib.PK_ERR_INVALID_ARG


def test_scratch_calls_need_their_objects():
    n = C.c_int64(7)
    assert _lib.load().pk_batch_scratch(None, C.byref(n)) == _lib.PK_ERR_INVALID_ARG
    assert _lib.load().pk_pool_trim(None, C.byref(n)) == _lib.PK_ERR_INVALID_ARG and n.value == 7


def test_graph_count_needs_a_batch():
    n = C.c_int64(7)
    assert _lib.load().pk_batch_graphs(None, C.byref(n)) == _lib.PK_ERR_INVALID_ARG and n.value == 7


# ------------------------------------------------------------------ block manager
def test_compact_keeps_own_blocks_and_releases_the_rest():
    bm = BlockManager(16, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(22)))
    old = bm.block_table(1)
    free = bm.alloc.num_free
    assert bm.compact(1, 9) == (old, old[:3])
    assert bm.block_table(1) == old[:3]
    assert bm.alloc.num_free == free + 3
    assert [int(bm.alloc.ref[b]) for b in old] == [1, 1, 1, 0, 0, 0]
    assert bm.alloc.free[-3:] == [old[5], old[4], old[3]]  # last block first, as free does
    assert bm.compact(1, 0) == (old[:3], [])
    bm.free(1)
    assert bm.alloc.num_free == 16


def test_compact_exchanges_shared_blocks():
    bm = BlockManager(16, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(12)))
    bm.fork(1, 2)
    old, new = bm.compact(2, 8)
    assert old == bm.block_table(1) and len(new) == 2 and not set(new) & set(old)
    assert [int(bm.alloc.ref[b]) for b in old + new] == [1, 1, 1, 1, 1]
    old1, new1 = bm.compact(1, 8)  # now the last holder: in place
    assert new1 == old1[:2]


def test_compact_exchanges_published_blocks_and_publishes_nothing_afterwards():
    bm = BlockManager(16, 4)
    toks = list(range(12))
    bm.allocate(1, toks)
    bm.mark_computed(1, toks, 12)
    old, new = bm.compact(1, 6)
    assert not set(new) & set(old)
    assert list(bm.alloc.evictable) == [old[2], old[1], old[0]]  # still a cached prefix for others
    assert bm.allocate(2, toks) == 8
    bm.ensure_capacity(1, 16, 6)
    cached = bm.alloc.cached
    bm.mark_computed(1, list(range(100, 116)), 16)
    assert bm.alloc.cached == cached and bm.tables[1].hashes == []
    bm.fork(1, 3)
    bm.mark_computed(3, list(range(100, 116)), 16)
    assert bm.alloc.cached == cached
    bm.free(1)
    bm.allocate(1, toks + [7] * 8)  # a new sequence under the old id publishes again
    bm.mark_computed(1, toks + [7] * 8, 20)
    assert len(bm.alloc.cached) > len(cached)


def test_compacted_sequences_are_not_hashed_again(monkeypatch):
    from pagellm_b200.cache import block_manager

    calls = []
    real = block_manager.block_hash
    monkeypatch.setattr(block_manager, "block_hash", lambda *a: calls.append(a) or real(*a))
    bm = BlockManager(16, 4)
    toks = list(range(24))
    bm.allocate(1, toks)
    bm.mark_computed(1, toks, 24)
    assert len(calls) >= 6
    bm.compact(1, 12)
    bm.fork(1, 2)
    del calls[:]
    for n in (12, 16, 20):
        bm.ensure_capacity(1, n, n - 4)
        bm.mark_computed(1, toks, n)
        bm.mark_computed(2, toks, 12)
    assert not calls and bm.tables[1].hashes == []
    bm.free(1)
    bm.allocate(1, [7] * 8)  # the old id's next sequence is hashed
    bm.mark_computed(1, [7] * 8, 8)
    assert calls and len(bm.tables[1].hashes) == 2


def test_compact_refusals_change_nothing():
    bm = BlockManager(6, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(16)))
    bm.fork(1, 2)
    before = bm.block_table(1), bm.alloc.free, bm.alloc.ref.copy()
    for n in (-1, 17):
        with pytest.raises(ValueError):
            bm.compact(1, n)
    with pytest.raises(OutOfBlocks):
        bm.compact(1, 12)  # three shared blocks, two free
    with pytest.raises(KeyError):
        bm.compact(9, 1)
    assert (bm.block_table(1), bm.alloc.free) == before[:2] and np.array_equal(bm.alloc.ref, before[2])


# ------------------------------------------------------------------ Python refusals and grouping
class _FakePool:
    def __init__(self, weights=object()):
        self.weights, self.calls = weights, []

    def evict(self, tables, lengths, budget, *, sinks, recent, new_tables):
        ip, ids = [list(map(list, x)) for x in (tables, new_tables)]
        rc, _ = _plan_evict(ip, lengths, ids, budget, sinks, recent)
        assert rc == 0, _lib.last_error()
        self.calls.append((ip, list(lengths), ids))


def test_evict_sequences_splits_calls_that_would_read_a_new_block():
    bm = BlockManager(16, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(16)))
    bm.fork(1, 2)
    bm.allocate(3, list(range(16)))
    bm.allocate(4, list(range(5)))
    pool = _FakePool()
    got = evict_sequences(pool, bm, [1, 2, 3, 4], [16, 16, 16, 5], 8, sinks=1, recent=2)
    assert got.tolist() == [8, 8, 8, 5]
    # 1 takes fresh blocks, 2 is then the blocks' last holder and thins them out in place, so it
    # must wait until 1 has read them; 3 can go with 2; 4 is short enough
    assert [c[1] for c in pool.calls] == [[16], [16, 16]]
    assert all(len(bm.block_table(s)) == 2 for s in (1, 2, 3, 4))


def test_evict_sequences_runs_what_it_compacted_before_blocks_ran_out():
    bm = BlockManager(8, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(16)))
    bm.allocate(2, list(range(12)))
    bm.fork(2, 3)
    pool = _FakePool()
    with pytest.raises(OutOfBlocks):
        evict_sequences(pool, bm, [1, 2], [16, 12], 9)  # two free blocks by then; 2 shares three
    assert [c[1] for c in pool.calls] == [[16]]


def test_evict_sequences_tells_what_it_shortened_before_blocks_ran_out():
    bm = BlockManager(8, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(12)))  # keeps its three blocks: its table does not show that it was shortened
    bm.allocate(4, list(range(4)))
    bm.allocate(2, list(range(12)))
    bm.fork(2, 3)
    before = bm.block_table(1)
    with pytest.raises(OutOfBlocks) as e:
        evict_sequences(_FakePool(), bm, [1, 4, 2, 3], [12, 4, 12, 12], 9)
    assert bm.block_table(1) == before
    assert e.value.lengths.tolist() == [9, 4, 12, 12]


@pytest.mark.parametrize("ids, lens, kw", [
    ([1], [4, 4], dict(budget=2)), ([1, 1], [4, 4], dict(budget=2)), ([1], [4], dict(budget=0)),
    ([1], [4], dict(budget=2, sinks=2, recent=1)), ([1], [4], dict(budget=2, sinks=-1)), ([1], [99], dict(budget=2)),
    ([1], [-1], dict(budget=2))])
def test_evict_sequences_refuses(ids, lens, kw):
    bm = BlockManager(8, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(8)))
    pool = _FakePool()
    with pytest.raises(ValueError):
        evict_sequences(pool, bm, ids, lens, **kw)
    with pytest.raises(ValueError):
        evict_sequences(_FakePool(None), bm, [1], [8], 4)
    assert not pool.calls and len(bm.block_table(1)) == 2


def test_evict_sequences_checks_the_pool_before_it_compacts():
    bm = BlockManager(8, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(16)))
    for wrong in (dict(block_size=8, num_blocks=8), dict(block_size=4, num_blocks=7)):
        pool = _FakePool()
        pool.__dict__.update(wrong)
        with pytest.raises(ValueError, match="pool's"):
            evict_sequences(pool, bm, [1], [16], 4)
        assert not pool.calls and len(bm.block_table(1)) == 4


def test_evict_sequences_does_not_repeat_a_failed_call():
    class Broken(_FakePool):
        def evict(self, tables, lengths, budget, **kw):
            self.calls.append(lengths)
            raise RuntimeError("device")

    bm = BlockManager(8, 4, enable_prefix_caching=False)
    bm.allocate(1, list(range(16)))
    pool = Broken()
    with pytest.raises(RuntimeError, match="device"):
        evict_sequences(pool, bm, [1], [16], 4)
    assert pool.calls == [[16]]


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(sinks=1), dict(window=4, sinks=-1),
                                dict(weights="sum"), dict(weights="add")])
def test_paged_batch_refuses_bad_bounds(kw):
    pool = _FakePool(weights=None)
    with pytest.raises(ValueError):
        PagedBatch(pool, [[0]], [0], [1], **kw)


# ------------------------------------------------------------------ the oracle's own rules
def test_evict_keep_orders_ties_and_nan():
    w = [0.0, 5.0, 1.0, 5.0, float("nan"), 5.0, 0.0, -0.0]
    assert bo.evict_keep(w, 3, 0, 0).tolist() == [1, 3, 4]
    assert bo.evict_keep(w, 4, 1, 1).tolist() == [0, 1, 4, 7]
    assert bo.evict_keep(w, 2, 1, 1).tolist() == [0, 7]
    assert bo.evict_keep(w, 8, 1, 1).tolist() == list(range(8))
    assert bo.evict_keep([1.0, 0.0, -0.0, 0.0], 2, 0, 0).tolist() == [0, 1]


def test_block_ids_do_not_wrap_and_tables_do_not_run_out():
    from pagellm_b200.cache.paged import _csr

    for ids in ([2 ** 32], [-2 ** 31 - 1], [3, 2 ** 31]):
        for tables in ([ids], [np.array(ids, np.int64)], [np.array([1], np.int32), np.array(ids, np.int64)]):
            with pytest.raises(IndexError):
                _csr(tables)
    with pytest.raises(IndexError):
        _csr([np.array([2 ** 31], np.uint32)])
    with pytest.raises(ValueError):
        _csr((np.array([0, 2, 4], np.int64), np.array([0, 1, 2], np.int32)))
    for tables in ([[5, 0], [7]], [np.array([5, 0]), np.array([7])], [np.array([5, 0], np.int32), np.array([7], np.uint8)],
                   (np.array([0, 2, 3], np.int64), np.array([5, 0, 7], np.int32))):
        indptr, ids = _csr(tables)
        assert indptr.tolist() == [0, 2, 3] and ids.tolist() == [5, 0, 7] and ids.dtype == np.int32


def test_handles_survive_other_threads_between_two_operations(monkeypatch):
    """What another thread gives or takes while a handle is looked at is neither lost nor handed out twice."""
    from pagellm_b200.cache import PagedKVPool

    pool = object.__new__(PagedKVPool)
    pool._idle_batches, pool._held_batches = [], [1, 2, 3]
    live = {1: 0, 2: 1, 3: 0, 9: 1}

    def graphs_of(h):
        if h == 1:
            pool._held_batches.append(9)  # dropped by another thread just now
        return live[h]

    monkeypatch.setattr(PagedKVPool, "_graphs_of", staticmethod(graphs_of))
    got = [pool._acquire_batch(), pool._acquire_batch()]
    assert sorted(got) == [1, 3]
    assert sorted(pool._held_batches) == [2, 9] and not pool._idle_batches

    class Emptied(list):  # another thread takes the last one after this one has seen it
        def pop(self, *a):
            self.clear()
            raise IndexError

    pool._held_batches, pool._idle_batches = [], Emptied([5])

    class Lib:
        def pk_batch_create(self, pool, out):
            out._obj.value = 77
            return 0

    monkeypatch.setattr(_lib, "load", Lib)
    pool._h = type("H", (), {"ptr": 1})()
    assert pool._acquire_batch() == 77
    pool._idle_batches = []  # nothing for the pool's end to destroy


# ------------------------------------------------------------------ C entries
def test_allocations_that_fail_are_errors():
    """No exception leaves a C entry (which would end the process): a child asks for impossible sizes."""
    import subprocess
    import sys
    from pathlib import Path

    code = '''
import ctypes as C
from pagellm_b200 import _lib
lib = _lib.load()
one, n, big = (C.c_int64 * 2)(0, 0), C.c_int(), C.c_int64()
codes = [lib.pk_plan_partition(one, 1 << 61, 148, 1, None, C.byref(n)),
         lib.pk_plan_evict(1 << 60, 16, 1, one, None, one, one, None, 4, 0, 0, C.byref(big))]
print(codes, _lib.last_error())
'''
    root = Path(__file__).resolve().parents[1]
    got = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert got.returncode == 0, got.stderr
    assert got.stdout.startswith(str([_lib.PK_ERR_CUDA] * 2)) and "host allocation" in got.stdout


# ------------------------------------------------------------------ the sources
def test_shared_memory_of_wide_words_is_declared_aligned():
    """Dynamic shared memory lies behind a kernel's static arrays: where it is read and written in 16-byte
    words as `sm`, its declaration has to ask for that alignment."""
    import re
    from pathlib import Path

    csrc = Path(__file__).resolve().parents[1] / "pagellm_b200" / "csrc"
    found = 0
    for path in sorted(csrc.glob("*.cu")):
        for line in re.findall(r"extern __shared__[^;]*\bsm\[\]", path.read_text()):
            found += 1
            assert "__align__(16)" in line, f"{path.name}: {line}"
    assert found >= 3

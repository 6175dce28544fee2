"""Bounded caches on the GPU: windowed attention with sinks, accumulated attention weights and
eviction, against the 64-bit oracle on exactly the values the device holds.

Tolerances. eps = 2^-24 (fp32), a score s = q.k * scale of D products has an absolute error of at
most ds = 2 (D + 8) eps |q||k| scale (products and sums in fp32, in any order; the factor 2 covers
a tensor core that truncates, 2^-23), plus what rounding q costs. A probability's relative error is
then at most dp = 2 ds + (n + 16) eps: the exponent, the maximum, the sum over n keys. An output
sums p v with |v| <= V: dp V, plus half a step of bf16 (2^-8) on each p where P is rounded, plus
n eps V for the sum, plus half a step of the output's type. A weight sums R probabilities: relative
error dp + R eps, plus eps of the old weight it is added to."""

from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import Shape, torch_cuda
from oracle import bounded_oracle as bo

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
HALF_BF16 = 2.0 ** -8


class Case:
    """A pool, a step over scattered tables, and the values the oracle sees. Every slot that no row
    of the step sees holds NaN, and so do the weights behind a sequence's last token."""

    def __init__(self, dtype, H, KVH, D, bs, starts, new, window=None, sinks=0, weights=None, seed=0, io=None,
                 layers=1, layer=0, poison=True, q_scale=1.0, stale=False):
        torch = torch_cuda()
        from pagellm_b200.cache import PagedKVPool

        rng = np.random.default_rng(seed)
        self.starts, self.new = np.asarray(starts, np.int64), np.asarray(new, np.int64)
        self.window, self.sinks, self.mode, self.layer = window, sinks, weights, layer
        self.H, self.KVH, self.D, self.bs, self.dtype = H, KVH, D, bs, dtype
        nblk = -(-(self.starts + self.new) // bs)
        num = int(nblk.sum()) + 3
        perm = rng.permutation(num).astype(np.int32)
        self.tables = np.split(perm[:int(nblk.sum())], np.cumsum(nblk)[:-1])
        self.pool = PagedKVPool(Shape(layers, KVH, D), num, bs, "bfloat16" if dtype == "bf16" else np.float32,
                                track_weights=weights is not None)
        if stale:  # entries that no row reads name some other sequence's block
            for i in range(len(self.tables)):
                seen = self.seen_blocks(i)
                for j in range(len(self.tables[i])):
                    if j not in seen:
                        self.tables[i] = self.tables[i].copy()
                        self.tables[i][j] = self.tables[(i + 1) % len(self.tables)][-1]
        self.io = io or dtype
        tdt = torch.bfloat16 if self.io == "bf16" else torch.float32
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        self.pool.k.normal_(generator=g)
        self.pool.v.normal_(generator=g)
        rows = int(self.new.sum())
        self.q = (torch.randn((rows, H, D), generator=g, device="cuda") * q_scale).to(tdt)
        self.k = torch.randn((rows, KVH, D), generator=g, device="cuda").to(tdt)
        self.v = torch.randn((rows, KVH, D), generator=g, device="cuda").to(tdt)
        if weights is not None:
            self.pool.weights.copy_(torch.rand(self.pool.weights.shape, generator=g, device="cuda") * 3)
        if poison:
            keep = torch.zeros((num, bs), dtype=torch.bool, device="cuda")
            for i in range(len(self.new)):
                if self.new[i] == 0:
                    continue
                pos = np.flatnonzero(self.seen(i))
                pos = pos[pos < self.starts[i]]
                keep[torch.as_tensor(self.tables[i][pos // bs].astype(np.int64)).cuda(),
                     torch.as_tensor(pos % bs).cuda()] = True
            self.pool.k[:, ~keep] = math.nan
            self.pool.v[:, ~keep] = math.nan
        self.before = None if weights is None else self.pool.weights.clone()

    def seen(self, i):
        out = np.zeros(int(self.starts[i] + self.new[i]), bool)
        for p in range(int(self.starts[i]), int(self.starts[i] + self.new[i])):
            out[bo.visible(p, self.window, self.sinks)] = True
        return out

    def seen_blocks(self, i):
        return set((np.flatnonzero(self.seen(i)) // self.bs).tolist()) if self.new[i] else set()

    def batch(self):
        from pagellm_b200.cache import PagedBatch

        return PagedBatch(self.pool, self.tables, self.starts, self.new, window=self.window, sinks=self.sinks,
                          weights=self.mode)

    def run(self, batch=None):
        batch = batch or self.batch()
        out = batch.write_and_attend(self.layer, self.q, self.k, self.v)
        batch.check()
        return out

    def rows(self, i):
        a = int(self.new[:i].sum())
        return slice(a, a + int(self.new[i]))

    def cached(self, i):
        """K and V of sequence i as the pool must hold them after the step (unseen ones zero)."""
        torch = torch_cuda()
        n = int(self.starts[i] + self.new[i])
        pos = np.arange(n)
        slots = torch.as_tensor(self.tables[i][pos // self.bs].astype(np.int64) * self.bs + pos % self.bs).cuda()
        seen = torch.as_tensor(self.seen(i)).cuda()
        res = []
        for flat in (self.pool.k_flat, self.pool.v_flat):
            x = flat[self.layer][slots].double()
            x[~seen] = 0.0
            res.append(x.cpu().numpy())
        return res

    def check(self, out, q_step=0.0, append=True):
        """Against the oracle; q_step: the relative half step that q may lose."""
        o = out.double().cpu().numpy()
        q = self.q.double().cpu().numpy()
        assert np.isfinite(o).all()
        bf_pool, scale = self.dtype == "bf16", 1.0 / math.sqrt(self.D)
        w_after = None if self.mode is None else self.pool.weights[self.layer].double().cpu().numpy()
        touched = None if self.mode is None else np.zeros(w_after.shape, bool)
        for i in range(len(self.new)):
            if self.new[i] == 0:
                continue
            r, st = self.rows(i), int(self.starts[i])
            k, v = self.cached(i)
            if append:
                tdt = np.float64
                want = self.k[r].to(self.pool.k.dtype).double().cpu().numpy()
                assert np.array_equal(k[st:], want.astype(tdt)), f"appended K of sequence {i}"
                assert np.array_equal(v[st:], self.v[r].to(self.pool.v.dtype).double().cpu().numpy())
            ref, w, seen = bo.attend_sequence(q[r], k, v, st, self.window, self.sinks)
            n = int(seen.sum())
            qk = np.linalg.norm(q[r], axis=-1).max() * np.linalg.norm(k, axis=-1).max() * scale
            ds = (2 * (self.D + 8) * EPS + q_step) * qk
            dp = 2 * ds + (n + 16) * EPS
            V = np.abs(v[seen]).max()
            tol = (dp + (HALF_BF16 if bf_pool else 0.0) + n * EPS) * V * 1.01
            tol = tol + np.abs(ref) * (HALF_BF16 if self.io == "bf16" else EPS)
            err = np.abs(o[r] - ref)
            assert (err <= tol).all(), f"sequence {i}: {err.max():.3g} > {tol[err > tol].min():.3g}"
            if self.mode is None:
                continue
            pos = np.flatnonzero(seen)
            blk, off = self.tables[i][pos // self.bs], pos % self.bs
            got = w_after[blk, :, off]
            old = self.before[self.layer].double().cpu().numpy()[blk, :, off] * (pos < st)[:, None]
            if self.mode == "replace":
                old = old * 0.0
            R = int(self.new[i]) * (self.H // self.KVH)
            wtol = w[pos] * (dp + (R + 4) * EPS) * 1.01 + (old + w[pos]) * 2 * EPS + 1e-35
            werr = np.abs(got - old - w[pos])
            assert (werr <= wtol).all(), f"weights of {i}: {(werr / np.maximum(wtol, 1e-300)).max():.3g} x tolerance"
            touched[blk[:, None], np.arange(self.KVH)[None], off[:, None]] = True
        if self.mode is not None:  # everything else as it was, on every layer
            now, was = self.pool.weights, self.before
            t = torch_cuda().as_tensor(touched).cuda()
            same = now == was
            same[self.layer] |= t
            assert bool(same.all()), "weights of unseen slots changed"


BF = [("bf16", 8, 2, 128, 16), ("bf16", 8, 8, 128, 16), ("bf16", 3, 1, 64, 32), ("bf16", 10, 2, 64, 16),
      ("bf16", 16, 1, 128, 64), ("bf16", 8, 1, 256, 16), ("bf16", 16, 8, 256, 16), ("bf16", 64, 8, 128, 16),
      ("bf16", 17, 1, 128, 16), ("bf16", 6, 2, 96, 8), ("bf16", 24, 12, 64, 16), ("bf16", 12, 4, 128, 48)]
FP = [("fp32", 4, 2, 32, 16), ("fp32", 8, 2, 128, 16), ("fp32", 5, 1, 96, 8), ("fp32", 6, 3, 17, 5),
      ("fp32", 4, 4, 64, 16), ("fp32", 9, 1, 256, 32), ("fp32", 2, 1, 512, 16)]
BOUNDS = [(1, 0), (1, 3), (16, 0), (37, 5), (64, 16), (50, 70), (1000, 4)]
DECODE = ([0, 1, 15, 16, 63, 64, 100, 250, 333], [1] * 9)
MIXED = ([0, 5, 130, 60, 0, 200], [9, 0, 5, 1, 1, 33])


@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("bounds", BOUNDS)
@pytest.mark.parametrize("shape", BF + FP, ids=lambda s: "-".join(map(str, s)))
def test_windowed_decode(shape, bounds, weights):
    c = Case(*shape, *DECODE, window=bounds[0], sinks=bounds[1], weights=weights, seed=sum(bounds))
    c.check(c.run())


@pytest.mark.parametrize("weights", [None, "add"])
@pytest.mark.parametrize("bounds", [(1, 0), (7, 3), (40, 0), (40, 20), (500, 1)])
@pytest.mark.parametrize("shape", BF + FP, ids=lambda s: "-".join(map(str, s)))
def test_windowed_windows_of_rows(shape, bounds, weights):
    c = Case(*shape, *MIXED, window=bounds[0], sinks=bounds[1], weights=weights, seed=sum(bounds))
    c.check(c.run())


@pytest.mark.parametrize("mode", ["add", "replace"])
@pytest.mark.parametrize("step", [DECODE, MIXED])
@pytest.mark.parametrize("shape", BF + FP, ids=lambda s: "-".join(map(str, s)))
def test_weights_without_a_window(shape, step, mode):
    c = Case(*shape, *step, weights=mode, seed=7)
    c.check(c.run())


@pytest.mark.parametrize("weights", [None, "replace"])
@pytest.mark.parametrize("bounds", [(None, 0), (100, 4), (256, 0), (129, 130), (64, 1)])
@pytest.mark.parametrize("shape", [("bf16", 8, 2, 128, 16), ("bf16", 4, 4, 128, 64), ("bf16", 16, 1, 128, 32),
                                   ("bf16", 6, 2, 128, 16), ("bf16", 4, 2, 64, 16), ("fp32", 4, 2, 64, 16)],
                         ids=lambda s: "-".join(map(str, s)))
def test_chunks(shape, bounds, weights):
    if bounds[0] is None and weights is None:
        pytest.skip("not a bounded step")
    c = Case(*shape, [0, 300, 131, 40], [200, 150, 1, 4], window=bounds[0], sinks=bounds[1], weights=weights, seed=3)
    c.check(c.run())


@pytest.mark.parametrize("bounds", [(33, 2), (200, 0)])
@pytest.mark.parametrize("weights", [None, "add"])
def test_fp32_rows_on_a_bf16_pool(bounds, weights):
    """q may be used at bf16: half a step of it, 2^-8 relative, on every score."""
    for shape in (("bf16", 8, 2, 128, 16), ("bf16", 8, 1, 64, 16), ("bf16", 6, 2, 96, 8)):
        c = Case(*shape, [0, 70, 300, 10], [1, 5, 1, 90], window=bounds[0], sinks=bounds[1], weights=weights, io="fp32")
        c.check(c.run(), q_step=HALF_BF16)


def test_numpy_rows_match_device_rows():
    torch = torch_cuda()
    c = Case("fp32", 4, 2, 32, 16, [30, 7], [1, 3], window=9, sinks=2, weights="replace")
    out = c.run()
    w = c.pool.weights.clone()
    host = c.batch().write_and_attend(0, c.q.cpu().numpy(), c.k.cpu().numpy(), c.v.cpu().numpy())
    assert isinstance(host, np.ndarray) and np.array_equal(host, out.cpu().numpy())
    assert torch.equal(w, c.pool.weights)
    again = c.batch().attend(0, c.q.cpu().numpy())
    np.testing.assert_allclose(again, host, rtol=1e-5, atol=1e-6)


def test_attend_reads_the_cache_alone():
    for dtype in ("bf16", "fp32"):
        c = Case(dtype, 8, 2, 128, 16, [40, 90], [1, 6], window=33, sinks=4, weights="add")
        c.run()
        c.before = c.pool.weights.clone()
        out = c.batch().attend(0, c.q)
        c.check(out, append=False)


def test_add_twice_and_layers():
    c = Case("bf16", 8, 2, 128, 16, [100, 20], [1, 1], window=50, sinks=2, weights="add", layers=3, layer=2)
    b = c.batch()
    c.check(c.run(b))
    c.before = c.pool.weights.clone()
    c.check(c.run(b))


def test_stale_table_entries_outside_the_window():
    for dtype, new in (("bf16", [1, 1, 5]), ("fp32", [1, 2, 1]), ("bf16", [1, 1, 100])):
        c = Case(dtype, 8, 2, 128, 16, [300, 250, 400], new, window=40, sinks=3, weights="add", stale=True)
        c.check(c.run())


def test_peaked_and_infinite_values():
    """Scores of a few hundred, and an infinite V and K in a masked place beside seen keys."""
    c = Case("bf16", 8, 2, 128, 16, [100, 35], [1, 1], window=20, sinks=1, weights="add", q_scale=30.0)
    c.pool.k.masked_fill_(c.pool.k.isnan(), math.inf)
    c.pool.v.masked_fill_(c.pool.v.isnan(), -math.inf)
    c.check(c.run())


def test_repeated_slots_and_shared_blocks():
    """Two sequences that write one block: the last writer's rows stay, as without a window; with
    weights such a step is refused."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    pool = PagedKVPool(Shape(1, 2, 64), 4, 16, "bfloat16", track_weights=True)
    tables, starts, new = [[0, 1], [2, 1]], [20, 20], [1, 1]
    q = torch.randn((2, 4, 64), device="cuda", dtype=torch.bfloat16)
    k = torch.randn((2, 2, 64), device="cuda", dtype=torch.bfloat16)
    b = PagedBatch(pool, tables, starts, new, window=8)
    out = b.write_and_attend(0, q, k, k)
    b.check()
    assert torch.equal(pool.k[0, 1, 4], k[1]) and bool(out.isfinite().all())
    with pytest.raises(ValueError, match="read twice"):
        PagedBatch(pool, tables, starts, new, weights="add")
    with pytest.raises(ValueError, match="read twice"):
        PagedBatch(pool, [[0, 0]], [20], [1], weights="add")
    # blocks outside every window may be shared
    b = PagedBatch(pool, [[0, 1, 2], [0, 1, 3]], [40, 40], [1, 1], window=9, weights="add")
    b.write_and_attend(0, q, k, k)
    b.check()
    # and the refusals leave the handle fit for the next step
    b = PagedBatch(pool, [[0, 1]], [20], [1])
    b.write_and_attend(0, q[:1].float(), k[:1].float(), k[:1].float())
    b.check()


def test_refusals():
    torch = torch_cuda()
    from pagellm_b200 import _lib
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    lib = _lib.load()
    plain = PagedKVPool(Shape(1, 2, 64), 4, 16, "bfloat16")
    assert plain.weights is None
    with pytest.raises(ValueError):
        PagedBatch(plain, [[0]], [3], [1], weights="add")
    with pytest.raises(ValueError, match="track"):
        plain.evict([[0]], [3], 2)
    b = PagedBatch(plain, [[0]], [3], [1])
    x = torch.zeros((1, 2, 64), device="cuda", dtype=torch.bfloat16)
    args = (x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), None)
    assert lib.pk_batch_write_and_attend_bf16(b._b, 0, 2, *args) == _lib.PK_ERR_UNSUPPORTED
    assert lib.pk_batch_set_bounds(b._b, 0, 3, 0) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_batch_set_bounds(b._b, -1, 0, 0) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_batch_set_bounds(b._b, 0, 0, 1) == _lib.PK_ERR_INVALID_ARG  # no weights tracked
    assert lib.pk_batch_set_bounds(b._b, 0, 0, 3) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_batch_set_bounds(b._b, 5, 1, 0) == _lib.PK_OK
    assert lib.pk_batch_write_and_attend_bf16(b._b, 0, 2, *args) == _lib.PK_ERR_INVALID_ARG  # plan again
    assert lib.pk_batch_set_bounds(b._b, 0, 0, 0) == _lib.PK_OK
    w = PagedBatch(plain, [[0]], [3], [1], window=2)
    assert lib.pk_batch_write_and_attend_bf16(w._b, 1, 2, *args) == _lib.PK_ERR_OUT_OF_RANGE
    assert lib.pk_batch_write_and_attend_bf16(w._b, 0, 3, *args) == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_batch_write_and_attend_bf16(w._b, 0, 2, x.data_ptr(), None, x.data_ptr(), x.data_ptr(), None) \
        == _lib.PK_ERR_INVALID_ARG
    assert lib.pk_batch_write_and_attend_bf16(w._b, 0, 2, x.data_ptr() + 2, *args[1:]) == _lib.PK_ERR_INVALID_ARG
    f32 = PagedKVPool(Shape(1, 2, 64), 4, 16)
    f = PagedBatch(f32, [[0]], [3], [1], window=2)
    assert lib.pk_batch_write_and_attend_bf16(f._b, 0, 2, *args) == _lib.PK_ERR_UNSUPPORTED
    out = f.write_and_attend(0, x, x, x)  # bf16 rows on an fp32 pool: converted, as without a window
    assert out.dtype == torch.bfloat16
    empty = PagedBatch(plain, [], [], [], window=4)
    assert empty.write_and_attend(0, x[:0], x[:0], x[:0]).shape == (0, 2, 64)


def test_handles_forget_their_bounds():
    """A recycled batch handle plans a plain step again, with the results it had before."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch

    c = Case("bf16", 8, 2, 128, 16, [100, 60], [1, 1], window=8, poison=False)
    q, k, v = c.q.float(), c.k.float(), c.v.float()
    want = PagedBatch(c.pool, c.tables, c.starts, c.new).write_and_attend(0, q, k, v)
    b = c.batch()
    c.check(c.run(b))
    del b
    assert torch.equal(PagedBatch(c.pool, c.tables, c.starts, c.new).write_and_attend(0, q, k, v), want)


def test_other_streams_and_capture():
    torch = torch_cuda()
    c = Case("bf16", 8, 2, 128, 16, [100, 333, 40], [1, 1, 80], window=60, sinks=4, weights="replace")
    side = torch.cuda.Stream()
    b = c.batch()  # planned on the current stream, run on another
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = b.write_and_attend(0, c.q, c.k, c.v)
    torch.cuda.synchronize()
    c.check(out)
    # a graph replays with new rows
    graph = torch.cuda.CUDAGraph()
    q = c.q.clone()
    with torch.cuda.graph(graph):
        got = b.write_and_attend(0, q, c.k, c.v)
    c.q = torch.randn_like(c.q)
    q.copy_(c.q)
    graph.replay()
    torch.cuda.synchronize()
    c.check(got)
    b.check()
    # the first call with some n_heads cannot be captured
    fresh = c.batch()
    with pytest.raises(Exception, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.write_and_attend(0, q, c.k, c.v)
    torch.cuda.synchronize()
    c.check(fresh.write_and_attend(0, c.q, c.k, c.v))


def test_results_repeat_bit_for_bit():
    torch = torch_cuda()
    c = Case("bf16", 32, 8, 128, 16, [3000, 800, 40, 500], [1, 5, 1, 200], window=700, sinks=4, weights="replace")
    b = c.batch()
    out, w = c.run(b).clone(), c.pool.weights.clone()
    for _ in range(5):
        assert torch.equal(c.run(b), out) and torch.equal(c.pool.weights, w)


def test_copied_blocks_take_their_weights_along():
    torch = torch_cuda()
    from pagellm_b200.cache import PagedKVPool

    pool = PagedKVPool(Shape(2, 3, 32), 6, 4, track_weights=True)
    assert pool.weights.shape == (2, 6, 3, 4) and not bool(pool.weights.any())
    pool.weights.normal_()
    want = pool.weights.clone()
    want[:, 1], want[:, 4] = want[:, 3].clone(), want[:, 3].clone()
    want[:, 5] = want[:, 1]
    pool.copy_blocks([(3, 1), (3, 4), (1, 5)])
    assert torch.equal(pool.weights, want)


# ------------------------------------------------------------------ eviction
def _evict_case(dtype, KVH, D, bs, lengths, layers=2, seed=0, values="heavy", in_place=()):
    torch = torch_cuda()
    from pagellm_b200.cache import PagedKVPool

    rng = np.random.default_rng(seed)
    lens = np.asarray(lengths, np.int64)
    nblk = -(-lens // bs)
    num = 2 * int(nblk.sum()) + 2
    perm = rng.permutation(num).astype(np.int32)
    parts = np.split(perm[:2 * int(nblk.sum())], np.cumsum(np.concatenate([nblk, nblk]))[:-1])
    old, new = parts[:len(lens)], list(parts[len(lens):])
    for i in in_place:
        new[i] = old[i]
    pool = PagedKVPool(Shape(layers, KVH, D), num, bs, "bfloat16" if dtype == "bf16" else np.float32, track_weights=True)
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool.k.normal_(generator=g)
    pool.v.normal_(generator=g)
    w = pool.weights
    if values == "heavy":
        w.normal_(generator=g).exp_()
        w.masked_fill_(torch.rand(w.shape, generator=g, device="cuda") < 0.1, 0.0)
    elif values == "ties":
        w.copy_(torch.randint(-2, 3, w.shape, generator=g, device="cuda").float())
        w.masked_fill_(torch.rand(w.shape, generator=g, device="cuda") < 0.2, -0.0)
    elif values == "equal":
        w.fill_(0.25)
    else:  # every kind of float
        w.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, w.shape, generator=g, device="cuda", dtype=torch.int64)
                .to(torch.int32).view(torch.float32))
    return pool, old, new, lens


def _check_evict(pool, old, new, lens, budget, sinks, recent, **kw):
    torch = torch_cuda()
    bs = pool.block_size
    bits = (lambda t: t.view(torch.int16) if t.dtype == torch.bfloat16 else t.view(torch.int32))
    k0, v0, w0 = bits(pool.k).cpu().numpy().copy(), bits(pool.v).cpu().numpy().copy(), pool.weights.cpu().numpy().copy()
    new_lens, kept = pool.evict(old, lens, budget, sinks=sinks, recent=recent, new_tables=new, return_kept=True, **kw)
    assert np.array_equal(new_lens, np.minimum(lens, budget))
    want_k, want_v, want_w = k0.copy(), v0.copy(), w0.copy()
    want_kept = np.full((pool.n_layers, len(lens), pool.n_kv_heads, budget), -1, np.int32)
    for i, n in enumerate(lens.tolist()):
        pos = np.arange(n)
        for li in range(pool.n_layers):
            for h in range(pool.n_kv_heads):
                keep = bo.evict_keep(w0[li, old[i][pos // bs], h, pos % bs], budget, sinks, recent)
                want_kept[li, i, h, :len(keep)] = keep
                y = np.arange(len(keep))
                sb, so, db, do = old[i][keep // bs], keep % bs, new[i][y // bs], y % bs
                want_k[li, db, do, h], want_v[li, db, do, h] = k0[li, sb, so, h], v0[li, sb, so, h]
                want_w[li, db, h, do] = w0[li, sb, h, so]
    assert np.array_equal(kept.cpu().numpy(), want_kept)
    assert np.array_equal(bits(pool.k).cpu().numpy(), want_k)
    assert np.array_equal(bits(pool.v).cpu().numpy(), want_v)
    assert np.array_equal(pool.weights.cpu().numpy().view(np.int32), want_w.view(np.int32))


@pytest.mark.parametrize("values", ["heavy", "ties", "equal", "any"])
@pytest.mark.parametrize("budget, sinks, recent", [(1, 0, 0), (1, 1, 0), (17, 0, 0), (64, 4, 16), (64, 40, 24),
                                                   (100, 0, 99), (299, 1, 1), (1000, 4, 4)])
def test_evict_chooses_and_moves(budget, sinks, recent, values):
    _check_evict(*_evict_case("fp32", 2, 32, 16, [300, 64, 0, 1, 65, 257, 100], seed=budget, values=values),
                 budget, sinks, recent)


@pytest.mark.parametrize("in_place", [(), (0, 1, 2, 3), (1, 3)])
@pytest.mark.parametrize("shape", [("bf16", 8, 128, 16), ("bf16", 1, 256, 64), ("bf16", 3, 96, 8), ("bf16", 2, 17, 5),
                                   ("fp32", 4, 64, 16), ("fp32", 3, 17, 5), ("bf16", 2, 6, 16)],
                         ids=lambda s: "-".join(map(str, s)))
def test_evict_shapes_and_places(shape, in_place):
    _check_evict(*_evict_case(*shape, [777, 300, 513, 40], seed=5, in_place=in_place), 290, 3, 20)


def test_evict_long_sequences():
    """Longer than shared memory holds weights for, and one that it holds."""
    for in_place in ((), (0, 1)):
        _check_evict(*_evict_case("bf16", 1, 16, 64, [45000, 40000], layers=1, in_place=in_place), 30000, 5, 1111)


def test_evict_some_fresh_some_own_blocks():
    pool, old, new, lens = _evict_case("bf16", 2, 64, 16, [200, 333], seed=9)
    mixed = [np.concatenate([new[i][:4], old[i][4:]]) for i in range(2)]
    _check_evict(pool, old, mixed, lens, 150, 2, 30)


def test_evict_on_two_streams_and_without_kept():
    torch = torch_cuda()
    pool, old, new, lens = _evict_case("bf16", 2, 64, 16, [200, 333], layers=1, seed=2)
    other, old2, new2, lens2 = _evict_case("bf16", 2, 64, 16, [200, 333], layers=1, seed=2)
    pool.evict(old, lens, 90, new_tables=new)
    side = torch.cuda.Stream()
    other.evict([old2[0]], [200], 90, new_tables=[new2[0]])
    with torch.cuda.stream(side):
        other.evict([old2[1]], [333], 90, new_tables=[new2[1]])
    torch.cuda.synchronize()
    assert torch.equal(pool.k, other.k) and torch.equal(pool.v, other.v) and torch.equal(pool.weights, other.weights)
    assert len(pool.evict([], [], 3)) == 0


def test_evict_refusals_leave_the_pool_alone():
    torch = torch_cuda()
    pool, old, new, lens = _evict_case("fp32", 2, 32, 16, [100, 90])
    k, w = pool.k.clone(), pool.weights.clone()
    for bad in (dict(budget=0), dict(budget=8, sinks=5, recent=4), dict(budget=200000000000)):
        with pytest.raises(Exception):
            pool.evict(old, lens, **bad)
    with pytest.raises(ValueError):
        pool.evict(old, lens, 50, new_tables=[old[1], old[0]])
    with pytest.raises(ValueError):
        pool.evict([old[0], old[0]], [100, 100], 50)
    with pytest.raises(IndexError):
        pool.evict(old, [100, 9999], 50)
    with pytest.raises(ValueError):
        pool.evict(old, [100], 50)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(Exception, match="capture"):
        with torch.cuda.graph(graph):
            pool.evict(old, lens, 50)
    torch.cuda.synchronize()
    assert torch.equal(pool.k, k) and torch.equal(pool.weights, w)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype, bs", [("fp32", 16), ("bf16", 16)])
def test_a_stream_through_a_bounded_cache(dtype, bs):
    """Prompt, decode with weights, eviction through the block manager with a forked sequence, and
    decoding on: each step against the oracle on a host copy of what every head should hold."""
    torch = torch_cuda()
    from pagellm_b200.cache import BlockManager, PagedBatch, PagedKVPool, evict_sequences

    H, KVH, D, layers, budget, sinks, recent = 4, 2, 64, 2, 48, 2, 8
    pool = PagedKVPool(Shape(layers, KVH, D), 40, bs, "bfloat16" if dtype == "bf16" else np.float32, track_weights=True)
    bm = BlockManager(40, bs, enable_prefix_caching=False)
    tdt = torch.bfloat16 if dtype == "bf16" else torch.float32
    g = torch.Generator(device="cuda").manual_seed(0)
    host = {}  # (seq, layer) -> [K, V, W] float64, (n, KVH, D) / (n, KVH)

    def step(seqs, new, window=None, mode="add"):
        starts = [host[s, 0][0].shape[0] if (s, 0) in host else 0 for s in seqs]
        copies = []
        for s, a, n in zip(seqs, starts, new):
            copies += bm.ensure_capacity(s, a + n, a)
        pool.copy_blocks(copies)
        batch = PagedBatch(pool, bm.tables_csr(seqs), starts, new, window=window, sinks=sinks if window else 0, weights=mode)
        for li in range(layers):
            rows = int(sum(new))
            q, k, v = (torch.randn((rows, h, D), generator=g, device="cuda").to(tdt) for h in (H, KVH, KVH))
            out = batch.write_and_attend(li, q, k, v).double().cpu().numpy()
            r0 = 0
            for s, a, n in zip(seqs, starts, new):
                K, V, W = host.get((s, li), [np.zeros((0, KVH, D)), np.zeros((0, KVH, D)), np.zeros((0, KVH))])
                r = slice(r0, r0 + n)
                K = np.concatenate([K, k[r].double().cpu().numpy()])
                V = np.concatenate([V, v[r].double().cpu().numpy()])
                ref, w, seen = bo.attend_sequence(q[r].double().cpu().numpy(), K, V, a, window, sinks if window else 0)
                tol = 2 * HALF_BF16 * np.abs(V).max() if dtype == "bf16" else 1e-5
                assert np.abs(out[r] - ref).max() <= tol
                W = np.concatenate([W, np.zeros((n, KVH))]) + w
                host[s, li] = [K, V, W]
                r0 += n
        batch.check()

    bm.allocate(1, list(range(70)))
    step([1], [70])
    bm.allocate(2, list(range(30)))
    step([1, 2], [1, 30])
    bm.fork(1, 3)
    for (s, li) in [(1, 0), (1, 1)]:
        host[3, li] = [x.copy() for x in host[s, li]]
    # forks share blocks: a step with weights has to be preceded by their copies
    with pytest.raises(ValueError):
        PagedBatch(pool, bm.tables_csr([1, 3]), [71, 71], [1, 1], weights="add")
    step([1, 2], [1, 1])
    # a weight lives in its token's block: sequences that share one share its weights
    t1, t3 = bm.block_table(1), bm.block_table(3)
    shared = sum(a == b for a, b in zip(t1, t3)) * bs
    assert shared == 64
    for li in range(layers):
        host[3, li][2][:shared] = host[1, li][2][:shared]
    lens = [host[s, 0][0].shape[0] for s in (1, 2, 3)]
    new_lens = evict_sequences(pool, bm, [1, 2, 3], lens, budget, sinks=sinks, recent=recent)
    assert new_lens.tolist() == [48, 31, 48]
    for i, s in enumerate((1, 2, 3)):
        for li in range(layers):
            K, V, W = host[s, li]
            if len(K) <= budget:
                continue
            table = np.asarray(bm.block_table(s))
            y = np.arange(budget)
            slots = torch.as_tensor(table[y // bs] * bs + y % bs).cuda()
            gk = pool.k_flat[li][slots].double().cpu().numpy()
            gv = pool.v_flat[li][slots].double().cpu().numpy()
            gw = pool.weights[li].double().cpu().numpy()[table[y // bs], :, y % bs]
            for h in range(KVH):
                # which tokens stayed: their K rows identify them; the choice must be right up to
                # weights that the two computations may order differently
                idx = [int(np.flatnonzero((K[:, h] == gk[t, h]).all(1))[0]) for t in range(budget)]
                assert idx == sorted(idx) and idx[:sinks] == list(range(sinks))
                assert idx[-recent:] == list(range(len(K) - recent, len(K)))
                assert np.array_equal(gv[:, h], V[idx, h])
                assert np.allclose(gw[:, h], W[idx, h], rtol=1e-4, atol=1e-6)
                out_idx = sorted(set(range(len(K))) - set(idx))
                assert W[out_idx, h].max() <= W[idx[sinks:-recent], h].min() * (1 + 1e-4) + 1e-6
            host[s, li] = [gk, gv, gw]
    for _ in range(3):
        step([1, 2, 3], [1, 1, 1], window=20)
    step([1, 3], [5, 1])
    for s in (1, 2, 3):
        bm.free(s)
    assert bm.alloc.num_free == 40

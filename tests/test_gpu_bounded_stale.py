"""What lies in a pool from earlier owners of its blocks reaches no later sequence."""

from __future__ import annotations

import numpy as np
import pytest

from gpu_util import Shape, torch_cuda
from oracle import bounded_oracle as bo
from pagellm_b200 import _lib

pytestmark = pytest.mark.gpu

POOLS = [("bf16", 2, 128, 16), ("fp32", 2, 32, 16), ("bf16", 3, 96, 8), ("fp32", 1, 17, 5), ("bf16", 8, 128, 32)]
STEPS = [([30, 5, 0, 64], [1, 1, 0, 1]), ([30, 0, 7], [1, 90, 9])]


@pytest.mark.parametrize("call", ["device", "host", "bf16", "windowed", "append"])
@pytest.mark.parametrize("starts, new", STEPS)
@pytest.mark.parametrize("shape", POOLS, ids=lambda s: "-".join(map(str, s)))
def test_tokens_stored_without_weights_start_at_zero(shape, starts, new, call):
    """A block's last owner leaves its weights there; a step that keeps none stores tokens of weight zero,
    on its layer, and touches no other weight."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    dtype, KVH, D, bs = shape
    H = 2 * KVH
    nblk = [-(-(s + n) // bs) for s, n in zip(starts, new)]
    ids = np.random.default_rng(0).permutation(sum(nblk) + 2).astype(np.int32)
    tables = np.split(ids[:sum(nblk)], np.cumsum(nblk)[:-1])
    pool = PagedKVPool(Shape(2, KVH, D), sum(nblk) + 2, bs, "bfloat16" if dtype == "bf16" else np.float32,
                       track_weights=True)
    pool.weights.uniform_(1, 2)
    want = pool.weights.clone()
    for t, s, n in zip(tables, starts, new):
        for p in range(s, s + n):
            want[1, int(t[p // bs]), :, p % bs] = 0
    rows = sum(new)
    q, k = (torch.randn((rows, h, D), device="cuda") for h in (H, KVH))
    b = PagedBatch(pool, tables, starts, new, window=20 if call in ("windowed", "bf16") else None)
    if call == "append":
        slots = b.slots_device()
        assert _lib.load().pk_pool_append(pool.handle, 1, k.data_ptr(), k.data_ptr(), slots.data_ptr(), rows,
                                          torch.cuda.current_stream().cuda_stream) == 0
    elif call == "host":
        b.write_and_attend(1, *(x.cpu().numpy() for x in (q, k, k)))
    elif call == "bf16":
        b.write_and_attend(1, *(x.bfloat16() for x in (q, k, k)))
    else:
        b.write_and_attend(1, q, k, k)
    b.check()
    assert torch.equal(pool.weights, want)
    b.attend(1, q)  # stores nothing
    b.check()
    assert torch.equal(pool.weights, want)


def test_repeated_slots_and_graphs_clear_too():
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    pool = PagedKVPool(Shape(1, 2, 64), 4, 16, "bfloat16", track_weights=True)
    pool.weights.fill_(1.0)
    want = pool.weights.clone()
    want[0, 1, :, 4] = 0
    q, k = (torch.randn((2, h, 64), device="cuda") for h in (4, 2))
    b = PagedBatch(pool, [[0, 1], [2, 1]], [20, 20], [1, 1])  # both write slot 4 of block 1
    b.write_and_attend(0, q, k, k)
    assert torch.equal(pool.weights, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.write_and_attend(0, q, k, k)
    pool.weights.fill_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(pool.weights, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_prompt_without_weights_before_steps_that_add_them(dtype):
    """A second sequence in the first one's blocks: prompt without weights, decodes that add, against the
    formula from weights of zero. Tolerance: the probabilities' of test_gpu_bounded.py, far below 1e-3 of a
    sum of probabilities at these sizes; what an earlier owner leaves is 1 and more."""
    torch = torch_cuda()
    from pagellm_b200.cache import PagedBatch, PagedKVPool

    H, KVH, D, bs, n = 4, 2, 64, 16, 40
    pool = PagedKVPool(Shape(1, KVH, D), 4, bs, "bfloat16" if dtype == "bf16" else np.float32, track_weights=True)
    g = torch.Generator(device="cuda").manual_seed(3)
    tdt = torch.bfloat16 if dtype == "bf16" else torch.float32

    def step(start, new, weights):
        q, k, v = (torch.randn((new, h, D), generator=g, device="cuda").to(tdt) for h in (H, KVH, KVH))
        PagedBatch(pool, [[2, 0, 3, 1]], [start], [new], weights=weights).write_and_attend(0, q, k, v)
        return [x.double().cpu().numpy() for x in (q, k, v)]

    step(0, n, "add")
    step(n, 1, "add")
    q, K, V = step(0, n, None)  # the blocks' next owner
    W = np.zeros((n, KVH))
    for t in range(n, n + 5):
        q, k, v = step(t, 1, "add")
        K, V, W = np.concatenate([K, k]), np.concatenate([V, v]), np.concatenate([W, np.zeros((1, KVH))])
        W = W + bo.attend_sequence(q, K, V, t, None, 0)[1]
    pos = np.arange(n + 5)
    got = pool.weights[0].double().cpu().numpy()[np.array([2, 0, 3, 1])[pos // bs], :, pos % bs]
    assert np.allclose(got, W, rtol=1e-3, atol=1e-6)

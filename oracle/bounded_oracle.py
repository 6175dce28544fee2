"""64-bit oracle of the bounded-cache operators (TEST INFRASTRUCTURE ONLY): windowed attention
with sinks, the attention weight of every cached token, and eviction by that weight. pagellm has
none of them; the formulas are stated at each function and written out one row at a time."""

from __future__ import annotations

import math

import numpy as np

__all__ = ["visible", "attend_sequence", "evict_keep"]


def visible(pos: int, window: int | None, sinks: int) -> np.ndarray:
    """Keys that the row at position ``pos`` sees: j <= pos with j < sinks or j > pos - window."""
    j = np.arange(pos + 1)
    return j if window is None else j[(j < sinks) | (j > pos - window)]


def attend_sequence(q, k, v, start: int, window: int | None, sinks: int):
    """(out, weights, seen) of one sequence's rows in float64.

    q (n, H, d) at positions start.., k and v (start + n, KVH, d). out[r, h] = softmax(q.k /
    sqrt(d)) v over the visible keys; weights[j, kh] = sum of those probabilities over the rows
    and kh's query heads; seen[j]: some row sees key j."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, H, d = q.shape
    kvh = k.shape[1]
    g = H // kvh
    out = np.zeros((n, H, d))
    weights = np.zeros((start + n, kvh))
    seen = np.zeros(start + n, bool)
    for r in range(n):
        j = visible(start + r, window, sinks)
        seen[j] = True
        for h in range(kvh):
            s = q[r, h * g:(h + 1) * g] @ k[j, h].T / math.sqrt(d)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[r, h * g:(h + 1) * g] = p @ v[j, h]
            weights[j, h] += p.sum(0)
    return out, weights, seen


def evict_keep(w, budget: int, sinks: int, recent: int) -> np.ndarray:
    """Positions that one head keeps, ascending, given its tokens' weights: all of them up to
    ``budget``, else the first ``sinks``, the last ``recent`` and the largest of the rest (ties
    to the lowest position, NaN the largest)."""
    n = len(w)
    if n <= budget:
        return np.arange(n)
    with np.errstate(invalid="ignore"):  # signalling NaNs widen too
        mid = np.asarray(w[sinks:n - recent], np.float64)
    rank = np.where(np.isnan(mid), np.inf, mid)
    order = sorted(range(len(mid)), key=lambda i: (not np.isnan(mid[i]), -rank[i], i))
    take = [sinks + i for i in order[:budget - sinks - recent]]
    return np.array(sorted(list(range(sinks)) + take + list(range(n - recent, n))), np.int64)

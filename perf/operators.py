"""Timed cases of the bounded-cache operators: what a program that serves streams longer than
its cache runs on every layer of every step.

* ``window``  - attention over the paged cache with a sliding window and a few first tokens
  that stay visible: ``PagedBatch(..., window=, sinks=).write_and_attend(layer, q, k, v)``.
* ``weights`` - the same step, windowed or not, that also adds up per cached token and KV head
  the attention weight it got: ``PagedBatch(..., weights="add" | "replace")`` on a pool made
  with ``track_weights=True``.
* ``evict``   - per layer, sequence and KV head, the ``budget`` tokens worth keeping (first
  tokens, recent tokens, then the largest accumulated weights, ties to the lowest position)
  moved in order into the sequence's new blocks: ``pool.evict(...)``.

``own = False`` computes them with elementary torch operations in 32 bits on plain tensors;
``own = True`` through the framework. One pass is one layer of a step (all layers for
``evict``): a program plans a step once and runs every layer on that plan, so the plan is
made in ``prepare``. A step's own rows are written to the same slots on every pass.
"""

import math
import random

import numpy as np
import torch

own = False

_GOLDEN = 0.6180339887498949


# ------------------------------------------------------------------ cases
def _attend(name, op, dtype, heads, kv_heads, head_dim, block, seqs, new, ctx, window, sinks, chunk=0, chunk_start=0,
            mode="none"):
    return {"name": name, "op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "block": block, "seqs": seqs, "new": new, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "window": window,
            "sinks": sinks, "chunk": chunk, "chunk_start": chunk_start, "mode": mode}


def _evict(name, dtype, kv_heads, head_dim, block, layers, seqs, ctx, budget, sinks, recent):
    return {"name": name, "op": "evict", "dtype": dtype, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
            "layers": layers, "seqs": seqs, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "budget": budget, "sinks": sinks,
            "recent": recent}


def listed():
    return [
        # the small fp32 model's decode step: a few kilobytes, latency alone
        _attend("window decode small fp32", "window", "fp32", 4, 2, 32, 16, 8, 1, (1, 256), 64, 4),
        # one layer of an 8B-shaped decode batch whose contexts have outgrown the window
        _attend("window decode", "window", "bf16", 32, 8, 128, 16, 64, 1, (512, 4096), 1024, 4),
        # a long-context decode batch of a 70B shape: most of each cache lies outside the window
        _attend("window decode long", "window", "bf16", 64, 8, 128, 16, 128, 1, (1024, 32768), 4096, 16),
        # speculative verification, window and sinks that end inside blocks
        _attend("window verify odd", "window", "bf16", 32, 8, 128, 16, 64, 5, (512, 4096), 509, 3),
        # a mixed step: decodes beside one prompt chunk
        _attend("window mixed step", "window", "bf16", 32, 8, 128, 16, 16, 1, (256, 2048), 640, 4, 512, 1024),
        # a long prompt's chunk against a full window
        _attend("window prompt chunk", "window", "bf16", 32, 8, 128, 16, 0, 1, (1, 1), 4096, 4, 2048, 6144),
        # the small model's decode step with weights kept up
        _attend("weights decode small fp32", "weights", "fp32", 4, 2, 32, 16, 8, 1, (1, 256), 0, 0, mode="add"),
        # the 8B-shaped decode batch, weights added up for a later eviction
        _attend("weights decode", "weights", "bf16", 32, 8, 128, 16, 64, 1, (512, 4096), 0, 0, mode="add"),
        # a prompt's last chunk, whose own weights decide what of the prompt is kept
        _attend("weights prompt chunk", "weights", "bf16", 32, 8, 128, 16, 0, 1, (1, 1), 0, 0, 2048, 2048, "replace"),
        # the small model's caches cut to a quarter
        _evict("evict small fp32", "fp32", 2, 32, 16, 4, 8, (60, 256), 64, 4, 16),
        # an 8B-shaped batch cut to a fixed budget (two of its layers)
        _evict("evict batch", "bf16", 8, 128, 16, 2, 64, (512, 4096), 1024, 4, 256),
        # few very long contexts (four layers): the choice among many tokens counts
        _evict("evict long", "bf16", 8, 128, 16, 4, 4, (32000, 32768), 8191, 16, 1000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    caps = [_cost(c) for c in listed()]
    cap = {k: max(c[k] for c in caps) for k in caps[0]}
    while True:
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        kvh = rng.choice([1, 2, 4, 8])
        D = rng.choice([64, 128, 128, 256]) if dtype == "bf16" else rng.choice([32, 64, 96, 128])
        bs = rng.choice([16, 16, 32, 64]) if dtype == "bf16" else rng.choice([8, 16, 32])
        op = rng.choice(["window", "weights", "evict"])
        if op == "evict":
            hi = _log(rng, 40, 32768)
            lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
            budget = max(1, int(hi * rng.uniform(0.05, 0.9)))
            sinks = min(rng.choice([0, 1, 4, 7, 16]), budget)
            recent = int((budget - sinks) * rng.uniform(0.0, 0.6))
            c = _evict("drawn", dtype, kvh, D, bs, rng.choice([1, 2, 3, 4]), _log(rng, 1, 64), (lo, hi), budget, sinks,
                       recent)
        else:
            g = rng.choice([1, 2, 3, 4, 5, 8])
            kind = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
            seqs = 0 if kind == "chunk" else _log(rng, 1, 128)
            new = rng.randint(2, 9) if kind == "verify" else 1
            hi = max(_log(rng, 16, 32768 if op == "window" else 8192), new)
            lo = max(new, int(hi * rng.uniform(0.05, 1.0)))
            chunk = _log(rng, 17, 2048) if kind in ("chunk", "mixed") else 0
            start = rng.choice([0, _log(rng, 1, 4096)]) if chunk else 0
            windowed = op == "window" or rng.random() < 0.3
            window = _log(rng, 1, 4096) if windowed else 0
            sinks = rng.choice([0, 1, 3, 4, 16, 37]) if windowed else 0
            mode = rng.choice(["add", "replace"]) if op == "weights" else "none"
            c = _attend("drawn", op, dtype, kvh * g, kvh, D, bs, seqs, new, (lo, hi), window, sinks, chunk, start, mode)
        del c["name"]
        cost = _cost(c)
        if all(cost[k] <= cap[k] for k in cap):
            return c


def _lens(case):
    """(starts, new tokens) of every sequence, spread over the case's range (over its logarithm
    where it spans more than a factor of ten); the same for every seed."""
    lo, hi, n = case["ctx_lo"], case["ctx_hi"], case["seqs"]
    f = (np.arange(n) * _GOLDEN + 0.5) % 1.0
    ctx = lo * (hi / lo) ** f if hi > 10 * lo else lo + (hi - lo) * f
    ctx = np.clip(np.rint(ctx).astype(np.int64), lo, hi)
    new = np.full(n, case.get("new", 0), np.int64)
    starts = ctx - new
    if case.get("chunk"):
        starts = np.append(starts, case["chunk_start"])
        new = np.append(new, case["chunk"])
    return starts, new


def _visible(case):
    """(tokens whose K/V the step has to read, sum over its rows of the keys a row sees)."""
    starts, new = _lens(case)
    p = np.repeat(starts - np.cumsum(new) + new, new) + np.arange(int(new.sum()))  # every row's position
    if case["window"] == 0:
        return int((starts + new).sum()), int((p + 1).sum())
    W, S = case["window"], case["sinks"]
    first = np.maximum(0, starts - W + 1)
    tokens = starts + new - first + np.minimum(S, first)
    lo = np.maximum(0, p - W + 1)
    return int(tokens.sum()), int((p - lo + 1 + np.minimum(S, lo)).sum())


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    kvh, D = case["kv_heads"], case["head_dim"]
    starts, new = _lens(case)
    if case["op"] == "evict":
        # every weight read once; kept rows of K, V and the weight read and written once
        kept = np.minimum(starts, case["budget"]).sum()
        moved = int(kept) * (2 * D * e + 4) * 2
        return {"bytes": case["layers"] * kvh * (4 * int((starts - np.minimum(starts, case["budget"])).sum()) + moved
                                                 + 4 * int(kept)), "flops": 0}
    tokens, pairs = _visible(case)
    rows = int(new.sum())
    b = (tokens - rows) * kvh * 2 * D * e  # cached K and V
    b += rows * kvh * 2 * D * e * 2        # the step's own, read and stored
    b += rows * case["heads"] * D * e * 2  # q and out
    flops = 4 * pairs * case["heads"] * D
    if case["mode"] != "none":
        b += tokens * kvh * 4 * (2 if case["mode"] == "add" else 1)
    return {"bytes": b, "flops": flops}


def _cost(case):
    """What bounds a drawn case: its work, its pool and the plain form's largest arrays."""
    w = work(case)
    starts, new = _lens(case)
    e = 2 if case["dtype"] == "bf16" else 4
    tok = -(-(starts + new) // case["block"]) * case["block"]
    pool = int(tok.sum()) * case["kv_heads"] * case["head_dim"] * 2 * e * case.get("layers", 1)
    if case["op"] == "evict":
        plain = case["layers"] * case["seqs"] * case["budget"] * case["kv_heads"] * case["head_dim"] * 4
    else:
        n, L = int(new.max()), _span(case)
        plain = max(len(new) * case["heads"] * n * L * 4, len(new) * L * case["kv_heads"] * case["head_dim"] * 4)
    return {"bytes": w["bytes"], "flops": w["flops"], "pool": pool, "plain": plain}


def _span(case):
    """Most positions that a sequence's rows see together: the padded key axis of the plain form."""
    starts, new = _lens(case)
    L = int((starts + new).max())
    return L if case["window"] == 0 else min(L, case["sinks"] + case["window"] - 1 + int(new.max()))


# ------------------------------------------------------------------ inputs
class _Shape:
    def __init__(self, n_layers, n_kv_heads, head_dim):
        self.n_layers, self.n_kv_heads, self.head_dim = n_layers, n_kv_heads, head_dim


def _gen(seed, k):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 16 + k)


def _fill(t, seed, k):
    return t.normal_(generator=_gen(seed, k))


def _fill_weights(t, seed):
    """Accumulated weights as decoding leaves them: heavy-tailed, some tokens never attended."""
    g = _gen(seed, 7)
    t.normal_(generator=g).mul_(1.5).exp_()
    never = torch.rand(t.shape, generator=g, device=t.device) < 0.05
    return t.masked_fill_(never, 0.0)


def _tables(case, seed):
    """Blocks of every sequence (and, for evict, of its shortened form), scattered over the pool."""
    starts, new = _lens(case)
    bs = case["block"]
    nblk = -(-(starts + new) // bs)
    nnew = -(-np.minimum(starts, case["budget"]) // bs) if case["op"] == "evict" else np.zeros_like(nblk)
    need = int(nblk.sum() + nnew.sum())
    num = max(1, math.ceil(1.25 * need))
    perm = np.random.default_rng(seed).permutation(num).astype(np.int32)
    cut = np.cumsum(np.concatenate([nblk, nnew]))
    parts = np.split(perm[:need], cut[:-1])
    return num, parts[:len(nblk)], parts[len(nblk):], starts, new


def _padded(tables):
    n = np.array(list(map(len, tables)))
    out = np.zeros((len(n), max(1, int(n.max()))), np.int64)
    out[np.arange(out.shape[1])[None] < n[:, None]] = np.concatenate(tables)
    return torch.from_numpy(out).cuda()


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case = case
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    kvh, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    num, tables, new_tables, starts, new = _tables(case, seed)
    layers = case.get("layers", 1)
    tracked = case["op"] != "window"
    shape = (layers, num, bs, kvh, D)
    if own:  # the user's pool; the same values in the same layout as the plain tensors
        from pagellm_b200.cache import PagedBatch, PagedKVPool

        more = {"track_weights": True} if tracked else {}
        s.pool = PagedKVPool(_Shape(layers, kvh, D), num, bs, case["dtype"], **more)
        s.k, s.v = s.pool.k, s.pool.v
        s.w = s.pool.weights if tracked else None
    else:
        s.k, s.v = torch.empty(shape, dtype=dt, device="cuda"), torch.empty(shape, dtype=dt, device="cuda")
        s.w = torch.empty((layers, num, kvh, bs), device="cuda") if tracked else None
    _fill(s.k, seed, 1)
    _fill(s.v, seed, 2)
    if tracked:
        _fill_weights(s.w, seed)
    if case["op"] == "evict":
        s.tables, s.new_tables, s.lens = tables, new_tables, starts
        if not own:
            _plan_evict(s)
        return s
    rows = int(new.sum())
    s.q = _fill(torch.empty((rows, case["heads"], D), dtype=dt, device="cuda"), seed, 3)
    s.kn = _fill(torch.empty((rows, kvh, D), dtype=dt, device="cuda"), seed, 4)
    s.vn = _fill(torch.empty((rows, kvh, D), dtype=dt, device="cuda"), seed, 5)
    s.w0 = s.w.clone() if case["mode"] == "add" else None
    if own:
        mode = None if case["mode"] == "none" else case["mode"]
        s.batch = PagedBatch(s.pool, tables, starts, new, window=case["window"] or None, sinks=case["sinks"],
                             weights=mode)
    else:
        _plan_attend(s, tables, starts, new)
    return s


# ------------------------------------------------------------------ plain form
def _plan_attend(s, tables, starts, new):
    """Index arrays of the step, which a program keeps for all its layers: where rows are stored
    and, padded to the longest, which positions each sequence's rows read and which rows see them."""
    c = s.case
    bs, W, S = c["block"], c["window"], c["sinks"]
    tab = _padded(tables)
    st = torch.from_numpy(starts).cuda()[:, None]
    n = torch.from_numpy(new).cuda()[:, None]
    B, nmax, L = len(new), int(new.max()), _span(c)
    r = torch.arange(nmax, device="cuda")[None]
    s.row_of = torch.from_numpy(np.concatenate([[0], np.cumsum(new)[:-1]])).cuda()[:, None] + r  # padded row -> row
    s.row_live = r < n
    s.row_of = torch.where(s.row_live, s.row_of, 0)
    s.rows_flat = s.row_live.flatten().nonzero()[:, 0]  # live rows, in order
    qpos = st + r
    p = torch.where(s.row_live, qpos, st).flatten()[s.rows_flat]
    b = torch.arange(B, device="cuda")[:, None].expand(B, nmax).flatten()[s.rows_flat]
    s.slot_new = tab[b, p // bs] * bs + p % bs
    first = (st - W + 1).clamp(min=0) if W else torch.zeros_like(st)  # first windowed key of the first row
    ns = first.clamp(max=S)                                           # sinks in front of it
    x = torch.arange(L, device="cuda")[None]
    pos = torch.where(x < ns, x, x - ns + first)
    live = pos < st + n
    pos = torch.where(live, pos, 0)
    s.slot_key = torch.gather(tab, 1, pos // bs) * bs + pos % bs
    seen = live[:, None, :] & (pos[:, None, :] <= qpos[:, :, None])
    if W:
        seen &= (pos[:, None, :] < S) | (pos[:, None, :] > qpos[:, :, None] - W)
    s.mask = seen & s.row_live[:, :, None]
    if c["mode"] != "none":
        s.key_flat = live.flatten().nonzero()[:, 0]
        slot = s.slot_key.flatten()[s.key_flat]
        s.key_blk, s.key_off = slot // bs, slot % bs
        s.key_old = (pos < st).flatten()[s.key_flat] if c["mode"] == "add" else None


def _attend_plain(s):
    c = s.case
    H, kvh, D = c["heads"], c["kv_heads"], c["head_dim"]
    g = H // kvh
    kf, vf = s.k[0].view(-1, kvh, D), s.v[0].view(-1, kvh, D)
    kf[s.slot_new] = s.kn
    vf[s.slot_new] = s.vn
    if s.w0 is not None:
        s.w.copy_(s.w0)
    B, n = s.row_of.shape
    L = s.slot_key.shape[1]
    K = kf[s.slot_key].float().permute(0, 2, 1, 3)                      # B kvh L D
    q = s.q[s.row_of].float().view(B, n, kvh, g, D).permute(0, 2, 3, 1, 4).reshape(B, kvh, g * n, D)
    p = (q @ K.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(B, kvh, g, n, L)
    del K
    hidden = ~s.mask[:, None, None]
    p.masked_fill_(hidden, -math.inf)
    top = p.amax(4, keepdim=True).clamp_(min=-3e38)  # padded rows see nothing
    p.sub_(top).exp_()
    p.div_(p.sum(4, keepdim=True).clamp_(min=1e-38))
    V = vf[s.slot_key].float().permute(0, 2, 1, 3)
    o = p.view(B, kvh, g * n, L) @ V
    o = o.view(B, kvh, g, n, D).permute(0, 3, 1, 2, 4).reshape(B * n, H, D)[s.rows_flat].to(s.q.dtype)
    if c["mode"] == "none":
        return {"out": o, "k": s.k, "v": s.v}
    add = p.sum((2, 3)).transpose(1, 2).reshape(B * L, kvh)[s.key_flat]
    w = s.w[0]
    if c["mode"] == "add":  # rows of this step start anew: their slots' old values are another token's
        add = add + torch.where(s.key_old[:, None], w[s.key_blk, :, s.key_off], 0.0)
    w[s.key_blk, :, s.key_off] = add
    return {"out": o, "k": s.k, "v": s.v, "weights": s.w}


def _plan_evict(s):
    c = s.case
    bs = c["block"]
    tab, ntab = _padded(s.tables), _padded(s.new_tables)
    n = torch.from_numpy(s.lens).cuda()[:, None]
    x = torch.arange(int(s.lens.max()), device="cuda")[None]
    s.live = x < n
    pos = torch.where(s.live, x, 0)
    s.blk, s.off = torch.gather(tab, 1, pos // bs), pos % bs
    s.pinned = s.live & ((x < c["sinks"]) | (x >= n - c["recent"]))
    y = torch.arange(c["budget"], device="cuda")[None]
    s.to_live = (y < n.clamp(max=c["budget"])).flatten().nonzero()[:, 0]  # live (sequence, new position) pairs
    slot = (torch.gather(ntab, 1, torch.where(y < n, y, 0) // bs) * bs + y % bs).flatten()[s.to_live]
    s.to_blk, s.to_off = slot // bs, slot % bs
    s.seq = torch.arange(len(s.lens), device="cuda")[:, None]
    s.of_seq = (s.seq.expand(-1, c["budget"])).flatten()[s.to_live]


def _evict_plain(s):
    c = s.case
    B, L, T = len(s.lens), s.live.shape[1], c["budget"]
    kvh = c["kv_heads"]
    w = s.w[:, s.blk, :, s.off]                                 # B L layers kvh
    key = torch.where(s.pinned[:, :, None, None], math.inf, w)
    key = torch.where(s.live[:, :, None, None], key, -math.inf)
    order = key.sort(dim=1, descending=True, stable=True).indices[:, :T]
    short = T - order.shape[1]
    kept = torch.where(torch.gather(s.live, 1, order.flatten(1)).view(order.shape), order, L).sort(1).values
    kept = torch.nn.functional.pad(kept, (0, 0, 0, 0, 0, short), value=L) if short > 0 else kept  # B T layers kvh
    out = torch.where(kept < L, kept, -1).permute(2, 0, 3, 1).to(torch.int32).contiguous()
    src = kept.flatten(0, 1)[s.to_live]                         # live pairs, layers, kvh
    li = torch.arange(c["layers"], device="cuda")[None, :, None]
    h = torch.arange(kvh, device="cuda")[None, None]
    b = s.of_seq[:, None, None]
    blk, off = s.blk[b, src], s.off[b, src]
    tb, to = s.to_blk[:, None, None], s.to_off[:, None, None]
    s.k[li, tb, to, h] = s.k[li, blk, off, h]
    s.v[li, tb, to, h] = s.v[li, blk, off, h]
    s.w[li, tb, h, to] = s.w[li, blk, h, off]
    return {"k": s.k, "v": s.v, "weights": s.w, "kept": out}


# ------------------------------------------------------------------ one pass
def run(s):
    c = s.case
    if c["op"] == "evict":
        if not own:
            return _evict_plain(s)
        kept = s.pool.evict(s.tables, s.lens, c["budget"], sinks=c["sinks"], recent=c["recent"],
                            new_tables=s.new_tables, return_kept=True)[1]
        return {"k": s.k, "v": s.v, "weights": s.w, "kept": kept}
    if not own:
        return _attend_plain(s)
    if s.w0 is not None:  # every pass starts from the same sums
        s.w.copy_(s.w0)
    res = {"out": s.batch.write_and_attend(0, s.q, s.kn, s.vn), "k": s.k, "v": s.v}
    if s.w is not None:
        res["weights"] = s.w
    return res


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    """Sequence by sequence from the formulas: softmax over the visible keys; a cached token's
    weight is its probability summed over the step's rows and the KV head's query heads."""
    if _cost(case)["plain"] > 3 << 30:
        return None
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    kvh, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    num, tables, new_tables, starts, new = _tables(case, seed)
    layers = case.get("layers", 1)
    k = _fill(torch.empty((layers, num, bs, kvh, D), dtype=dt, device="cuda"), seed, 1)
    v = _fill(torch.empty((layers, num, bs, kvh, D), dtype=dt, device="cuda"), seed, 2)
    w = None
    if case["op"] != "window":
        w = _fill_weights(torch.empty((layers, num, kvh, bs), device="cuda"), seed)
    if case["op"] == "evict":
        kept = torch.full((layers, len(starts), kvh, case["budget"]), -1, dtype=torch.int32, device="cuda")
        k2, v2, w2 = k.clone(), v.clone(), w.clone()
        head = torch.arange(kvh, device="cuda")
        for i, n in enumerate(starts.tolist()):
            t = torch.from_numpy(tables[i].astype(np.int64)).cuda()
            d = torch.from_numpy(new_tables[i].astype(np.int64)).cuda()
            m = min(n, case["budget"])
            for li in range(layers):
                wi = w[li, t].permute(1, 0, 2).reshape(kvh, -1)[:, :n].double()
                mid = wi[:, case["sinks"]:n - case["recent"]]
                if n <= case["budget"]:
                    keep = torch.arange(n, device="cuda").expand(kvh, n)
                else:
                    take = case["budget"] - case["sinks"] - case["recent"]
                    best = torch.argsort(-mid, dim=1, stable=True)[:, :take] + case["sinks"]
                    ends = torch.cat([torch.arange(case["sinks"], device="cuda"),
                                      torch.arange(n - case["recent"], n, device="cuda")]).expand(kvh, -1)
                    keep = torch.cat([ends, best], 1).sort(1).values
                kept[li, i, :, :m] = keep.to(torch.int32)
                y = torch.arange(m, device="cuda")
                sb, so = t[keep // bs], keep % bs
                db, do = d[y // bs][None], (y % bs)[None]
                k2[li][db, do, head[:, None]] = k[li][sb, so, head[:, None]]
                v2[li][db, do, head[:, None]] = v[li][sb, so, head[:, None]]
                w2[li][db, head[:, None], do] = w[li][sb, head[:, None], so]
        return {"k": k2, "v": v2, "weights": w2, "kept": kept}
    H = case["heads"]
    g = H // kvh
    rows = int(new.sum())
    q = _fill(torch.empty((rows, H, D), dtype=dt, device="cuda"), seed, 3)
    kn = _fill(torch.empty((rows, kvh, D), dtype=dt, device="cuda"), seed, 4)
    vn = _fill(torch.empty((rows, kvh, D), dtype=dt, device="cuda"), seed, 5)
    out = torch.empty((rows, H, D), dtype=torch.float64, device="cuda")
    r0 = 0
    plans = []
    for i, (s0, n) in enumerate(zip(starts.tolist(), new.tolist())):
        t = torch.from_numpy(tables[i].astype(np.int64)).cuda()
        p = torch.arange(s0, s0 + n, device="cuda")
        k[0][t[p // bs], p % bs] = kn[r0:r0 + n]
        v[0][t[p // bs], p % bs] = vn[r0:r0 + n]
        plans.append((t, p, r0))
        r0 += n
    w2 = w.double() if w is not None else None
    W = case["window"]
    for t, p, r0 in plans:
        n, ctx = len(p), int(p[-1]) + 1
        j = torch.arange(ctx, device="cuda")
        first = max(0, int(p[0]) - W + 1) if W else 0
        j = j[(j < case["sinks"]) | (j >= first)]
        see = j[None] <= p[:, None]
        if W:
            see &= (j[None] > p[:, None] - W) | (j[None] < case["sinks"])
        blk, off = t[j // bs], j % bs
        for h in range(kvh):
            kk, vv = k[0][blk, off, h].double(), v[0][blk, off, h].double()
            total = torch.zeros(len(j), dtype=torch.float64, device="cuda")
            for e in range(g):
                a = q[r0:r0 + n, h * g + e].double() @ kk.T / math.sqrt(D)
                a = torch.softmax(a.masked_fill(~see, -math.inf), 1)
                out[r0:r0 + n, h * g + e] = a @ vv
                total += a.sum(0)
            if w is not None:
                if case["mode"] == "add":
                    total += torch.where(j < int(p[0]), w[0][blk, h, off].double(), 0.0)
                w2[0][blk, h, off] = total
    res = {"out": out, "k": k, "v": v}
    if w is not None:
        res["weights"] = w2
    return res

// Bounded caches on the CUDA cores: windowed attention with sinks for any pool, the
// attention weight each cached token got, and the eviction of tokens by that weight.
//
//   attention   row at position p sees the keys j <= p with j < sinks or j > p - window
//   weights     a[j, h] = sum over the step's rows r and the query heads of KV head h that see
//               key j of softmax(q.k)[r, j]; stored per pool slot as [block][kv head][offset]
//   eviction    per (layer, sequence, KV head): the first `sinks` tokens, the last `recent`, and
//               of the rest the largest weights (ties to the lowest position), moved in order
//
// pagellm has none of the three (its caches only grow until a sequence ends); they extend
// cache/paged.py:383-464 (PagedBatch) and cache/paged.py:282-300 (PagedKVPool).

#include <cuda_bf16.h>

#include <algorithm>

#include "pk_device.cuh"
#include "pk_internal.h"

namespace pk {

namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// ------------------------------------------------------------------ attention
// One CTA (4 warps) per (row, query head): keys dealt to warps one at a time, lanes over
// dimensions, online softmax in the exp2 domain, the four warps merged at the end. The row's
// visible keys are numbered 0..nvis-1: the sinks in front of the window, then the window.
template <typename T, typename IO, int DPL>
__global__ void __launch_bounds__(128) bounded_rows_kernel(const BoundedParams p) {
    constexpr int NW = 4;
    __shared__ float sm_m[NW], sm_l[NW];
    extern __shared__ float sm_acc[];  // [NW][D]
    const int r = p.rows[blockIdx.x];
    const int head = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seq = p.row_seq[r];
    const int pos = p.starts[seq] + (r - p.offsets[seq]);
    const int lo = max(0, pos - p.window + 1);  // first key of the row's window
    const int ns = min(p.sinks, lo);            // sinks in front of it
    const int nvis = ns + pos - lo + 1;
    const int kh = head / (p.H / p.kvh);
    const T* kpool = static_cast<const T*>(p.pool_k);
    const T* vpool = static_cast<const T*>(p.pool_v);
    const int32_t* tbl = p.ids + p.indptr[seq];

    float qv[DPL], acc[DPL];
    const IO* qp = static_cast<const IO*>(p.q) + (static_cast<size_t>(r) * p.H + head) * p.D;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
        const int d = lane + 32 * i;
        qv[i] = d < p.D ? to_f(qp[d]) : 0.f;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int x = warp; x < nvis; x += NW) {
        const int j = x < ns ? x : x - ns + lo;
        const int64_t slot = static_cast<int64_t>(tbl[j / p.bs]) * p.bs + (j % p.bs);
        const size_t off = (static_cast<size_t>(slot) * p.kvh + kh) * p.D;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
            const int d = lane + 32 * i;
            if (d < p.D) dot = fmaf(qv[i], to_f(kpool[off + d]), dot);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const float s = dot * p.qscale;
        const float mnew = fmaxf(m, s);
        const float base = mnew == -INFINITY ? 0.f : mnew;
        const float corr = exp2f(m - base);
        const float w = exp2f(s - base);
        l = l * corr + w;
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
            const int d = lane + 32 * i;
            acc[i] = fmaf(w, d < p.D ? to_f(vpool[off + d]) : 0.f, acc[i] * corr);
        }
        m = mnew;
    }
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
        const int d = lane + 32 * i;
        if (d < p.D) sm_acc[warp * p.D + d] = acc[i];
    }
    __syncthreads();
    float mx = -INFINITY;
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sm_m[w]);
    float den = 0.f;
    float wt[NW];
    for (int w = 0; w < NW; ++w) {
        wt[w] = sm_m[w] == -INFINITY ? 0.f : exp2f(sm_m[w] - mx);
        den += wt[w] * sm_l[w];
    }
    const size_t orow = static_cast<size_t>(r) * p.H + head;
    if (p.ml != nullptr && threadIdx.x == 0) p.ml[orow] = make_float2(mx, 1.f / den);
    IO* op = static_cast<IO*>(p.out) + orow * p.D;
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
        float num = 0.f;
        for (int w = 0; w < NW; ++w) num += wt[w] * sm_acc[w * p.D + d];
        put(op + d, num / den);
    }
}

template <typename T, typename IO>
cudaError_t launch_rows_t(const BoundedParams& p, cudaStream_t st) {
    const dim3 grid(p.nrows, p.H);
    const size_t smem = 4 * p.D * sizeof(float);
    const int dpl = (p.D + 31) / 32;
    if (dpl <= 1) bounded_rows_kernel<T, IO, 1><<<grid, 128, smem, st>>>(p);
    else if (dpl <= 2) bounded_rows_kernel<T, IO, 2><<<grid, 128, smem, st>>>(p);
    else if (dpl <= 4) bounded_rows_kernel<T, IO, 4><<<grid, 128, smem, st>>>(p);
    else if (dpl <= 8) bounded_rows_kernel<T, IO, 8><<<grid, 128, smem, st>>>(p);
    else if (dpl <= 16) bounded_rows_kernel<T, IO, 16><<<grid, 128, smem, st>>>(p);
    else return cudaErrorInvalidValue;
    return cudaGetLastError();
}

// ------------------------------------------------------------------ weights
// One CTA per (touched block, KV head), warp = key: the key's row in registers, its score with
// every row of the sequence that sees it recomputed, probability 2^(s - m) / l from the row's
// statistics, summed in row order (one owner per key: no atomics, a fixed order).
template <typename T, typename IO, int DPL>
__global__ void __launch_bounds__(128) weight_rows_kernel(const BoundedParams p, const WeightParams w) {
    const int e = blockIdx.x, kh = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seq = w.t_seq[e], lb = w.t_blk[e];
    const int start = p.starts[seq], row0 = p.offsets[seq], n = p.offsets[seq + 1] - row0;
    const int ctx = start + n;
    const int lo = max(0, start - p.window + 1);
    const int phys = p.ids[p.indptr[seq] + lb];
    const int g = p.H / p.kvh;
    const T* kpool = static_cast<const T*>(p.pool_k);
    for (int t = warp; t < p.bs; t += 4) {
        const int j = lb * p.bs + t;
        if (j >= ctx || (j >= p.sinks && j < lo)) continue;
        const size_t off = ((static_cast<size_t>(phys) * p.bs + t) * p.kvh + kh) * p.D;
        float kv[DPL];
#pragma unroll
        for (int i = 0; i < DPL; ++i) kv[i] = lane + 32 * i < p.D ? to_f(kpool[off + lane + 32 * i]) : 0.f;
        float sum = 0.f;
        for (int r = max(0, j - start); r < n; ++r) {
            if (j >= p.sinks && j <= start + r - p.window) break;  // this and every later row is past it
            for (int c = 0; c < g; ++c) {
                const size_t row = static_cast<size_t>(row0 + r) * p.H + kh * g + c;
                const IO* qp = static_cast<const IO*>(p.q) + row * p.D;
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < DPL; ++i)
                    if (lane + 32 * i < p.D) dot = fmaf(to_f(qp[lane + 32 * i]), kv[i], dot);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                const float2 ml = p.ml[row];
                sum += exp2f(dot * p.qscale - ml.x) * ml.y;
            }
        }
        if (lane == 0) {
            float* dst = w.weights + (static_cast<size_t>(phys) * p.kvh + kh) * p.bs + t;
            *dst = w.add && j < start ? *dst + sum : sum;
        }
    }
}

template <typename T, typename IO>
cudaError_t launch_weight_rows_t(const BoundedParams& p, const WeightParams& w, cudaStream_t st) {
    const dim3 grid(w.ntouched, p.kvh);
    const int dpl = (p.D + 31) / 32;
    if (dpl <= 1) weight_rows_kernel<T, IO, 1><<<grid, 128, 0, st>>>(p, w);
    else if (dpl <= 2) weight_rows_kernel<T, IO, 2><<<grid, 128, 0, st>>>(p, w);
    else if (dpl <= 4) weight_rows_kernel<T, IO, 4><<<grid, 128, 0, st>>>(p, w);
    else if (dpl <= 8) weight_rows_kernel<T, IO, 8><<<grid, 128, 0, st>>>(p, w);
    else if (dpl <= 16) weight_rows_kernel<T, IO, 16><<<grid, 128, 0, st>>>(p, w);
    else return cudaErrorInvalidValue;
    return cudaGetLastError();
}

// The scores of the touched blocks are still in L2 (8 to 64 bytes per key and KV head beside the
// 512 of its K and V), so summing them costs a fraction of reading K again. Units of a sequence in
// order, columns in order: the sum does not depend on the schedule.
__global__ void __launch_bounds__(256) weight_scores_kernel(const ScoreWeightParams p) {
    const int64_t x = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
    const int64_t e64 = x / (p.kvh * p.bs);
    if (e64 >= p.w.ntouched) return;
    const int e = static_cast<int>(e64);
    const int hx = static_cast<int>(x - e64 * (p.kvh * p.bs));
    const int h = hx / p.bs, t = hx - h * p.bs;
    const int seq = p.w.t_seq[e], lb = p.w.t_blk[e];
    const int start = p.starts[seq], ctx = start + p.offsets[seq + 1] - p.offsets[seq];
    const int j = lb * p.bs + t;
    if (j >= ctx || (j >= p.sinks && j <= start - p.window)) return;
    float sum = 0.f;
    for (int u = p.seq_u[seq]; u < p.seq_u[seq + 1]; ++u) {
        const int4 b = __ldg(p.u_bound + u);
        const int4 m0 = __ldg(p.u_meta + 2 * u), m1 = __ldg(p.u_meta + 2 * u + 1);
        const int nblk = m1.z - m1.y;
        const int i = lb < b.x ? lb : lb - b.y;
        if (i >= nblk || (lb >= b.x && i < b.x)) continue;  // not a block of this unit
        const int ncol = m0.y * p.g, colp = (ncol + 1) & ~1;
        const float* sp = p.score + (static_cast<int64_t>(static_cast<uint32_t>(b.z)) | (static_cast<int64_t>(b.w) << 32)) +
                          ((static_cast<int64_t>(h) * nblk + i) * p.bs + t) * colp;
        const float2* ml = p.ml + static_cast<size_t>(m0.w) * p.H + h * p.g;
        for (int c = 0; c < ncol; c += 2) {
            const float2 s = __ldcg(reinterpret_cast<const float2*>(sp + c));
            const float2 a = __ldg(ml + (c / p.g) * p.H + c % p.g);
            sum += exp2f(s.x - a.x) * a.y;
            if (c + 1 < ncol) {
                const float2 b2 = __ldg(ml + ((c + 1) / p.g) * p.H + (c + 1) % p.g);
                sum += exp2f(s.y - b2.x) * b2.y;
            }
        }
    }
    const int phys = p.ids[p.indptr[seq] + lb];
    float* dst = p.w.weights + (static_cast<size_t>(phys) * p.kvh + h) * p.bs + t;
    *dst = p.w.add && j < start ? *dst + sum : sum;
}

// ------------------------------------------------------------------ append of bf16 rows
// Step rows given as bf16 are stored as they are; the slot comes from the block table (row ->
// sequence -> position -> block id). W: the widest word that divides a row.
template <typename W>
__global__ void append_rows16_kernel(__nv_bfloat16* __restrict__ pk_, __nv_bfloat16* __restrict__ pv_,
                                     const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v,
                                     const int32_t* __restrict__ row_seq, const int32_t* __restrict__ offsets,
                                     const int32_t* __restrict__ starts, const int32_t* __restrict__ indptr,
                                     const int32_t* __restrict__ ids, int bs, const int32_t* __restrict__ rows,
                                     int64_t n, int rowlen) {
    constexpr int kPer = sizeof(W) / 2;
    const int per_row = rowlen / kPer;
    const int64_t total = n * per_row;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t ri = i / per_row;
        const int c = static_cast<int>(i - ri * per_row);
        const int64_t r = rows ? rows[ri] : ri;
        const int s = row_seq[r];
        const int64_t pos = static_cast<int64_t>(starts[s]) + (r - offsets[s]);
        const int64_t blk = pos / bs;
        const int64_t slot = static_cast<int64_t>(ids[indptr[s] + blk]) * bs + (pos - blk * bs);
        reinterpret_cast<W*>(pk_ + slot * rowlen)[c] = reinterpret_cast<const W*>(k + r * rowlen)[c];
        reinterpret_cast<W*>(pv_ + slot * rowlen)[c] = reinterpret_cast<const W*>(v + r * rowlen)[c];
    }
}

// Copied blocks' weights (grid = pairs x layers).
__global__ void copy_weights_kernel(float* __restrict__ w, const int64_t* __restrict__ pairs, int64_t layer_floats,
                                    int block) {
    float* base = w + blockIdx.y * layer_floats;
    const float* s = base + pairs[2 * blockIdx.x] * block;
    float* d = base + pairs[2 * blockIdx.x + 1] * block;
    for (int i = threadIdx.x; i < block; i += blockDim.x) d[i] = s[i];
}

// ------------------------------------------------------------------ eviction
// Order-preserving integer of a weight: larger weights have larger keys, -0 equals 0, and NaN
// (either sign) is the largest.
__device__ __forceinline__ uint32_t weight_key(float x) {
    if (isnan(x)) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 256;

// Which tokens of (layer, sequence, KV head) stay: one CTA each. The threshold weight - the
// T-th largest of the middle [sinks, n - recent) - is found digit by digit from the top (radix
// select, 8 bits per pass over the keys); then one ordered pass writes the kept positions
// (larger than the threshold, or equal to it while ties remain to be taken, lowest first).
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
    extern __shared__ float vals[];  // the sequence's weights, when they fit
    __shared__ int hist[256];
    __shared__ int warp_gt[kSelThreads / 32], warp_eq[kSelThreads / 32];
    __shared__ int sh_digit, sh_rank;
    const int i = blockIdx.x, h = blockIdx.y, layer = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = p.lengths[i];
    const int m = min(n, p.budget);
    const int32_t* tbl = p.ids + p.indptr[i];
    const int32_t* ntbl = p.new_ids + p.new_indptr[i];
    float* wl = p.weights + static_cast<size_t>(layer) * p.num_blocks * p.kvh * p.bs;
    int32_t* kept = p.kept + ((static_cast<size_t>(layer) * p.nseq + i) * p.kvh + h) * p.budget;
    const bool cached = n <= p.cache_cap;
    auto at = [&](int j) {
        return wl + (static_cast<size_t>(tbl[j / p.bs]) * p.kvh + h) * p.bs + j % p.bs;
    };
    if (cached)
        for (int j = tid; j < n; j += kSelThreads) vals[j] = *at(j);
    __syncthreads();
    auto value = [&](int j) { return cached ? vals[j] : *at(j); };

    const int lo = p.sinks, hi = n - p.recent;  // the middle (used only when n > budget)
    uint32_t thr = 0;
    int ties = 0;  // keys equal to the threshold to take
    if (n > p.budget) {
        int rank = p.budget - p.sinks - p.recent;  // still to find among keys with the prefix
        if (rank > 0) {
            uint32_t mask = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int b = tid; b < 256; b += kSelThreads) hist[b] = 0;
                __syncthreads();
                for (int j = lo + tid; j < hi; j += kSelThreads) {
                    const uint32_t k = weight_key(value(j));
                    if ((k & mask) == thr) atomicAdd(&hist[(k >> shift) & 255], 1);
                }
                __syncthreads();
                if (tid == 0) {
                    int left = rank, b = 255;
                    while (hist[b] < left) left -= hist[b--];  // rank <= keys counted: ends at b >= 0
                    sh_digit = b;
                    sh_rank = left;
                }
                __syncthreads();
                thr |= static_cast<uint32_t>(sh_digit) << shift;
                mask |= 255u << shift;
                rank = sh_rank;
                __syncthreads();
            }
            ties = rank;
        } else {
            thr = 0xFFFFFFFFu;  // nothing of the middle is kept: no key is larger, no tie is taken
        }
    }
    // ordered pass: kept positions before this tile, ties before this tile
    int base = 0, eq_base = 0;
    for (int j0 = 0; j0 < n; j0 += kSelThreads) {
        const int j = j0 + tid;
        bool gt = false, eq = false;
        if (j < n) {
            if (n <= p.budget || j < lo || j >= hi) {
                gt = true;
            } else {
                const uint32_t k = weight_key(value(j));
                gt = k > thr;
                eq = k == thr;
            }
        }
        const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) {
            warp_gt[warp] = __popc(bg);
            warp_eq[warp] = __popc(be);
        }
        __syncthreads();
        int g0 = base, e0 = eq_base, gall = 0, eall = 0;
        for (int w = 0; w < kSelThreads / 32; ++w) {
            if (w < warp) {
                g0 += warp_gt[w];
                e0 += warp_eq[w];
            }
            gall += warp_gt[w];
            eall += warp_eq[w];
        }
        const unsigned below = (1u << lane) - 1;
        const int eq_before = e0 + __popc(be & below);  // ties at lower positions
        // kept before j: larger ones (counted in g0) and the ties taken so far
        const int y = g0 + __popc(bg & below) + min(eq_before, ties);
        if (gt || (eq && eq_before < ties)) kept[y] = j;
        base += gall;
        eq_base += eall;
        __syncthreads();
    }
    for (int y = m + tid; y < p.budget; y += kSelThreads) kept[y] = -1;
    __syncthreads();
    // The weights move with their tokens. New position y <= old position, so a tile's values are
    // read before any of them is overwritten, and later tiles' sources lie behind this one's
    // destinations (new_tables may name the old blocks, position by position).
    for (int y0 = 0; y0 < m; y0 += kSelThreads) {
        const int y = y0 + tid;
        float x = 0.f;
        if (y < m) x = value(kept[y]);
        __syncthreads();
        if (y < m) wl[(static_cast<size_t>(ntbl[y / p.bs]) * p.kvh + h) * p.bs + y % p.bs] = x;
    }
}

// Kept K (blockIdx.z even) or V rows into the new blocks: one CTA per work item (rows
// [y0, y1) of a sequence's new positions), (layer, KV head), tensor. Within an item rows move
// in tiles, all of a tile read before any is written; a sequence whose new table names some of
// its old blocks is one item, so that its tiles run in order (see evict_select_kernel).
template <typename W>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
    const int item = blockIdx.x;
    const int i = p.items[3 * item], y0 = p.items[3 * item + 1], y1 = p.items[3 * item + 2];
    const int h = blockIdx.y % p.kvh, layer = blockIdx.y / p.kvh;
    uint8_t* base = static_cast<uint8_t*>(blockIdx.z == 0 ? p.pool_k : p.pool_v) +
                    static_cast<size_t>(layer) * p.num_blocks * p.bs * p.kvh * p.row_bytes;
    const int32_t* tbl = p.ids + p.indptr[i];
    const int32_t* ntbl = p.new_ids + p.new_indptr[i];
    const int32_t* kept = p.kept + ((static_cast<size_t>(layer) * p.nseq + i) * p.kvh + h) * p.budget;
    const int words = p.row_bytes / static_cast<int>(sizeof(W));
    const int64_t total = static_cast<int64_t>(y1 - y0) * words;
    constexpr int kPer = 4;
    auto row_at = [&](const int32_t* t, int j) {
        return reinterpret_cast<W*>(base + ((static_cast<size_t>(t[j / p.bs]) * p.bs + j % p.bs) * p.kvh + h) * p.row_bytes);
    };
    for (int64_t x0 = 0; x0 < total; x0 += 256 * kPer) {
        W val[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int64_t x = x0 + e * 256 + threadIdx.x;
            if (x < total) val[e] = row_at(tbl, kept[y0 + x / words])[x % words];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int64_t x = x0 + e * 256 + threadIdx.x;
            if (x < total) row_at(ntbl, y0 + static_cast<int>(x / words))[x % words] = val[e];
        }
    }
}

}  // namespace

cudaError_t launch_bounded_rows(int dtype, bool io16, const BoundedParams& p, cudaStream_t st) {
    if (p.nrows <= 0) return cudaSuccess;
    if (dtype == 0) return io16 ? cudaErrorInvalidValue : launch_rows_t<float, float>(p, st);
    return io16 ? launch_rows_t<__nv_bfloat16, __nv_bfloat16>(p, st) : launch_rows_t<__nv_bfloat16, float>(p, st);
}

cudaError_t launch_weight_rows(int dtype, bool io16, const BoundedParams& p, const WeightParams& w, cudaStream_t st) {
    if (w.ntouched <= 0) return cudaSuccess;
    if (dtype == 0) return io16 ? cudaErrorInvalidValue : launch_weight_rows_t<float, float>(p, w, st);
    return io16 ? launch_weight_rows_t<__nv_bfloat16, __nv_bfloat16>(p, w, st)
                : launch_weight_rows_t<__nv_bfloat16, float>(p, w, st);
}

cudaError_t launch_weight_scores(const ScoreWeightParams& p, cudaStream_t st) {
    if (p.w.ntouched <= 0) return cudaSuccess;
    const int64_t threads = static_cast<int64_t>(p.w.ntouched) * p.kvh * p.bs;
    const int64_t blocks = (threads + 255) / 256;
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    weight_scores_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_append_rows16(void* pool_k_layer, void* pool_v_layer, const void* k, const void* v,
                                 const int32_t* row_seq, const int32_t* offsets, const int32_t* starts,
                                 const int32_t* indptr, const int32_t* ids, int bs, const int32_t* rows, int64_t n,
                                 int rowlen, cudaStream_t st) {
    if (n <= 0) return cudaSuccess;
    auto* a = static_cast<__nv_bfloat16*>(pool_k_layer);
    auto* b = static_cast<__nv_bfloat16*>(pool_v_layer);
    const auto* x = static_cast<const __nv_bfloat16*>(k);
    const auto* y = static_cast<const __nv_bfloat16*>(v);
    const auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    const bool vec = rowlen % 8 == 0 && a16(a) && a16(b) && a16(x) && a16(y);
    const int64_t work = n * (vec ? rowlen / 8 : rowlen);
    const int grid = static_cast<int>(std::min<int64_t>((work + 255) / 256, 148 * 16));
    if (vec)
        append_rows16_kernel<uint4><<<grid, 256, 0, st>>>(a, b, x, y, row_seq, offsets, starts, indptr, ids, bs, rows, n, rowlen);
    else
        append_rows16_kernel<uint16_t><<<grid, 256, 0, st>>>(a, b, x, y, row_seq, offsets, starts, indptr, ids, bs, rows, n, rowlen);
    return cudaGetLastError();
}

cudaError_t launch_copy_weights(float* weights, const int64_t* pairs, int64_t npairs, int layers, int64_t layer_floats,
                                int block, cudaStream_t st) {
    if (npairs <= 0) return cudaSuccess;
    copy_weights_kernel<<<dim3(static_cast<unsigned>(npairs), layers), 128, 0, st>>>(weights, pairs, layer_floats, block);
    return cudaGetLastError();
}

cudaError_t launch_evict(const EvictParams& p, int max_len, cudaStream_t st) {
    if (p.nseq <= 0) return cudaSuccess;
    EvictParams q = p;
    // the weights of a sequence are kept in shared memory while they fit
    constexpr int kMaxCached = 40960;  // floats: 160 KB
    q.cache_cap = std::min(max_len, kMaxCached);
    const size_t smem = static_cast<size_t>(q.cache_cap) * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kMaxCached * static_cast<int>(sizeof(float)));
    if (e != cudaSuccess) return e;
    evict_select_kernel<<<dim3(p.nseq, p.kvh, p.layers), kSelThreads, smem, st>>>(q);
    e = cudaGetLastError();
    if (e != cudaSuccess || p.nitems <= 0) return e;
    const dim3 grid(p.nitems, p.kvh * p.layers, 2);
    if (p.row_bytes % 16 == 0) evict_move_kernel<uint4><<<grid, 256, 0, st>>>(q);
    else if (p.row_bytes % 4 == 0) evict_move_kernel<uint32_t><<<grid, 256, 0, st>>>(q);
    else evict_move_kernel<uint16_t><<<grid, 256, 0, st>>>(q);
    return cudaGetLastError();
}

}  // namespace pk

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
// Weights from K once more: a key's row in registers, its score with every row of the sequence that
// sees it recomputed, probability 2^(s - m) / l from the row's statistics. One owner per key and a
// fixed order of addition: no atomics. For what neither cc_attn_kernel nor tile_weight_kernel sums: few
// columns in several rows or groups, head sizes above 256 or no multiples of 4. BY_ROW = false: one CTA
// per (touched block, KV head), a warp takes every eighth key and all rows. BY_ROW = true (16 rows and
// more): one CTA per (touched block, KV head, key), the rows dealt to its eight warps, whose sums are
// added in order; with a warp per key a 191-row chunk of 48 (block, head)s kept 192 warps busy and took
// 0.9 ms.
template <typename T, typename IO, int DPL, bool BY_ROW>
__global__ void __launch_bounds__(256) weight_rows_kernel(const BoundedParams p, const WeightParams w) {
    constexpr int NW = 8;
    __shared__ float part[NW];
    const int e = blockIdx.x, kh = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seq = w.t_seq[e], lb = w.t_blk[e];
    const int start = p.starts[seq], row0 = p.offsets[seq], n = p.offsets[seq + 1] - row0;
    const int ctx = start + n;
    const int lo = max(0, start - p.window + 1);
    const int phys = p.ids[p.indptr[seq] + lb];
    const int g = p.H / p.kvh;
    const T* kpool = static_cast<const T*>(p.pool_k);
    for (int t = BY_ROW ? static_cast<int>(blockIdx.z) : warp; t < p.bs; t += BY_ROW ? p.bs : NW) {
        const int j = lb * p.bs + t;
        if (j >= ctx || (j >= p.sinks && j < lo)) continue;  // (the same for all warps when BY_ROW)
        const size_t off = ((static_cast<size_t>(phys) * p.bs + t) * p.kvh + kh) * p.D;
        float kv[DPL];
#pragma unroll
        for (int i = 0; i < DPL; ++i) kv[i] = lane + 32 * i < p.D ? to_f(kpool[off + lane + 32 * i]) : 0.f;
        float sum = 0.f;
        // rows from the key's own on, until its window has passed it
        const int r_end = j < p.sinks || j - start > INT32_MAX - p.window ? n : min(n, j - start + p.window);
        for (int r = max(0, j - start) + (BY_ROW ? warp : 0); r < r_end; r += BY_ROW ? NW : 1) {
            const size_t row = static_cast<size_t>(row0 + r) * p.H + kh * g;
            const IO* qp = static_cast<const IO*>(p.q) + row * p.D;
#pragma unroll 2
            for (int c = 0; c < g; ++c) {
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < DPL; ++i)
                    if (lane + 32 * i < p.D) dot = fmaf(to_f(qp[static_cast<size_t>(c) * p.D + lane + 32 * i]), kv[i], dot);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                const float2 ml = p.ml[row + c];
                sum += exp2f(dot * p.qscale - ml.x) * ml.y;
            }
        }
        if (BY_ROW) {
            if (lane == 0) part[warp] = sum;
            __syncthreads();
            sum = 0.f;
            for (int x = 0; x < NW; ++x) sum += part[x];
        }
        if (lane == 0 && (!BY_ROW || warp == 0)) {
            float* dst = w.weights + (static_cast<size_t>(phys) * p.kvh + kh) * p.bs + t;
            *dst = w.add && j < start ? *dst + sum : sum;
        }
    }
}

template <typename T, typename IO, int DPL>
cudaError_t launch_weight_rows_d(const BoundedParams& p, const WeightParams& w, cudaStream_t st) {
    const dim3 grid(w.ntouched, p.kvh, w.max_rows >= 16 ? p.bs : 1);
    if (grid.z > 1) weight_rows_kernel<T, IO, DPL, true><<<grid, 256, 0, st>>>(p, w);
    else weight_rows_kernel<T, IO, DPL, false><<<grid, 256, 0, st>>>(p, w);
    return cudaGetLastError();
}

template <typename T, typename IO>
cudaError_t launch_weight_rows_t(const BoundedParams& p, const WeightParams& w, cudaStream_t st) {
    if (p.kvh > 65535 || p.bs > 65535) return cudaErrorInvalidValue;
    const int dpl = (p.D + 31) / 32;
    if (dpl <= 1) return launch_weight_rows_d<T, IO, 1>(p, w, st);
    if (dpl <= 2) return launch_weight_rows_d<T, IO, 2>(p, w, st);
    if (dpl <= 4) return launch_weight_rows_d<T, IO, 4>(p, w, st);
    if (dpl <= 8) return launch_weight_rows_d<T, IO, 8>(p, w, st);
    if (dpl <= 16) return launch_weight_rows_d<T, IO, 16>(p, w, st);
    return cudaErrorInvalidValue;
}

// The scores of the touched blocks are still in L2 (8 to 64 bytes per key and KV head beside the
// 512 of its K and V), so summing them costs a fraction of reading K again. One warp per touched
// block, its (KV head, token) pairs over the lanes, four of them in flight; records from the plan, so
// that the chain is record -> unit -> scores. MANY (a sequence of 16 units and more): one CTA per
// (touched block, 32 pairs), the units dealt to its eight warps. Sums are added in a fixed order.
// Bound by its chain of loads: 64 decodes over 148k tokens 20 us of the step's 124 (128 where the
// compiler is not told that one CTA per SM will do, 140 held to 40 registers).
template <bool MANY>
__global__ void __launch_bounds__(256, 1) weight_scores_kernel(const ScoreWeightParams p) {
    constexpr int NW = 8, kPer = MANY ? 1 : 4;
    __shared__ float part[MANY ? NW : 1][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int e = MANY ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) * NW + warp;
    if (e >= p.w.ntouched) return;
    const int4 r0 = __ldg(p.t_meta + 2 * e), r1 = __ldg(p.t_meta + 2 * e + 1);
    const int phys = r0.x, lb = r0.y, u0 = r0.z, u1 = r0.w, start = r1.x, ctx = r1.y;
    const int pairs = p.kvh * p.bs;
    float* wb = p.w.weights + static_cast<size_t>(phys) * p.kvh * p.block + r1.z;
    auto place = [&](int h, int t) { return wb + h * p.block + t; };
    for (int x0 = lane + (MANY ? 32 * static_cast<int>(blockIdx.y) : 0); MANY || x0 < pairs; x0 += 32 * kPer) {
        float sum[kPer], old[kPer];
        int h[kPer], t[kPer];
        bool live[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int x = x0 + 32 * k;
            h[k] = p.bs_shift >= 0 ? x >> p.bs_shift : x / p.bs;
            t[k] = x - h[k] * p.bs;
            const int j = lb * p.bs + t[k];
            live[k] = x < pairs && j < ctx && (j < p.sinks || j > start - p.window);
            sum[k] = 0.f;
            old[k] = live[k] && p.w.add && j < start ? *place(h[k], t[k]) : 0.f;
        }
        for (int u = u0 + (MANY ? warp : 0); u < u1; u += MANY ? NW : 1) {
            const int4 b = __ldg(p.u_bound + u);
            const int4 m0 = __ldg(p.u_meta + 2 * u), m1 = __ldg(p.u_meta + 2 * u + 1);
            const int nblk = m1.z - m1.y;
            const int i = lb < b.x ? lb : lb - b.y;
            if (i >= nblk || (lb >= b.x && i < b.x)) continue;  // not a block of this unit
            const int ncol = m0.y * p.g, colp = (ncol + 1) & ~1;
            const float* sp = p.score + (static_cast<int64_t>(static_cast<uint32_t>(b.z)) | (static_cast<int64_t>(b.w) << 32));
            for (int c = 0; c < ncol; c += 2) {
                // columns c and c + 1: query token c / g, head c % g of the KV head's
                const int ta = c / p.g, tb = (c + 1) / p.g;
                const size_t ra = static_cast<size_t>(m0.w + ta) * p.H + (c - ta * p.g);
                const size_t rb = static_cast<size_t>(m0.w + tb) * p.H + (c + 1 - tb * p.g);
                float2 s[kPer], ma[kPer], mb[kPer];
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    if (!live[k]) continue;
                    s[k] = __ldcg(reinterpret_cast<const float2*>(
                        sp + ((static_cast<int64_t>(h[k]) * nblk + i) * p.bs + t[k]) * colp + c));
                    ma[k] = __ldg(p.ml + ra + h[k] * p.g);
                    if (c + 1 < ncol) mb[k] = __ldg(p.ml + rb + h[k] * p.g);
                }
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    if (!live[k]) continue;
                    sum[k] += exp2f(s[k].x - ma[k].x) * ma[k].y;
                    if (c + 1 < ncol) sum[k] += exp2f(s[k].y - mb[k].x) * mb[k].y;
                }
            }
        }
        if (MANY) {
            part[warp][lane] = sum[0];
            __syncthreads();
            if (warp == 0 && live[0]) {
                float total = old[0];
                for (int x = 0; x < NW; ++x) total += part[x][lane];
                *place(h[0], t[0]) = total;
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (live[k]) *place(h[k], t[k]) = old[k] + sum[k];
    }
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

// Tokens stored by a step that keeps no weights: theirs start at zero, whatever the block's last owner
// left there. One thread per (row, KV head); slots given, or from the block table. A few KB of stores, so
// a launch and a chain of loads: 64 decodes of 8 KV heads over 100 / 2000 tokens take 36.9 / 92.0 us with it,
// 32.8 / 90.8 without. Launched only on pools that track weights.
__global__ void clear_weights_kernel(float* __restrict__ w, const int64_t* __restrict__ slots,
                                     const int32_t* __restrict__ row_seq, const int32_t* __restrict__ offsets,
                                     const int32_t* __restrict__ starts, const int32_t* __restrict__ indptr,
                                     const int32_t* __restrict__ ids, int bs, int kvh, int64_t n) {
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < n * kvh;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t r = i / kvh;
        const int h = static_cast<int>(i - r * kvh);
        int64_t blk, off;
        if (slots != nullptr) {
            blk = slots[r] / bs;
            off = slots[r] - blk * bs;
        } else {
            const int s = row_seq[r];
            const int64_t pos = static_cast<int64_t>(starts[s]) + (r - offsets[s]);
            off = pos % bs;
            blk = ids[indptr[s] + pos / bs];
        }
        w[(blk * kvh + h) * bs + off] = 0.f;
    }
}

// ------------------------------------------------------------------ eviction
// Order-preserving integer of a weight: larger weights have larger keys, -0 equals 0, and NaN
// (either sign) is the largest.
__device__ __forceinline__ uint32_t weight_key(float x) {
    if (isnan(x)) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Division by a size that is usually a power of two: shift >= 0 is its logarithm.
__device__ __forceinline__ int div_by(int x, int d, int shift) { return shift >= 0 ? x >> shift : x / d; }

constexpr int kSelBins = 2048;  // 11-bit digits: sign, exponent and 2 bits first, so heavy tails spread
// Place of a bin in shared memory: every eighth word is skipped, so that threads which own 8
// consecutive bins each touch different banks.
__device__ __forceinline__ int bin_at(int b) { return b + (b >> 3); }

// Which tokens of (layer, sequence, KV head) stay: one CTA each, its weights in shared memory when
// they fit. The threshold weight - the T-th largest of the middle [sinks, n - recent) - is found
// digit by digit from the top (radix select in three passes); then one ordered pass writes the
// kept positions (larger than the threshold, or equal to it while ties remain to be taken, lowest
// first) and their weights. Latency bound - n loads, then barriers and passes over shared memory -
// so everything goes four positions at a time, and few long sequences get 1024 threads each.
template <int NT>
__global__ void __launch_bounds__(NT, NT == 256 ? 8 : 1) evict_select_kernel(const EvictParams p) {
    extern __shared__ float4 vals4[];  // the sequence's weights, when they fit
    constexpr int NW = NT / 32, PER = kSelBins / NT;
    __shared__ int hist[kSelBins + kSelBins / 8];
    __shared__ int warp_a[32], warp_b[32];
    __shared__ int sh_digit, sh_rank;
    const int i = blockIdx.x, h = blockIdx.y, layer = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = p.lengths[i];
    const int m = min(n, p.budget);
    const int32_t* tbl = p.ids + p.indptr[i];
    const int32_t* ntbl = p.new_ids + p.new_indptr[i];
    float* wl = p.weights + static_cast<size_t>(p.layer0 + layer) * p.num_blocks * p.kvh * p.bs;
    int32_t* kept = p.kept + ((static_cast<size_t>(layer) * p.nseq + i) * p.kvh + h) * p.budget;
    const bool cached = n <= p.cache_cap;
    auto at = [&](const int32_t* t, int j) {
        const int b = div_by(j, p.bs, p.bs_shift);
        return wl + (static_cast<size_t>(t[b]) * p.kvh + h) * p.bs + (j - b * p.bs);
    };
    // weights of positions j .. j + 3 (j a multiple of 4; what lies behind the last token is unused)
    auto fetch4 = [&](int j) {
        if ((p.bs & 3) == 0) return *reinterpret_cast<const float4*>(at(tbl, j));
        float4 x = make_float4(*at(tbl, j), 0.f, 0.f, 0.f);
        if (j + 1 < n) x.y = *at(tbl, j + 1);
        if (j + 2 < n) x.z = *at(tbl, j + 2);
        if (j + 3 < n) x.w = *at(tbl, j + 3);
        return x;
    };
    if (cached) {
#pragma unroll 4
        for (int j = 4 * tid; j < n; j += 4 * NT) vals4[j >> 2] = fetch4(j);
    }
    for (int b = tid; b < kSelBins + kSelBins / 8; b += NT) hist[b] = 0;
    __syncthreads();
    auto value4 = [&](int j) { return cached ? vals4[j >> 2] : fetch4(j); };

    const int lo = p.sinks, hi = n - p.recent;  // the middle (used only when n > budget)
    uint32_t thr = 0;
    int ties = 0;  // keys equal to the threshold to take
    if (n > p.budget) {
        int rank = p.budget - p.sinks - p.recent;  // still to find among keys with the prefix
        if (rank > 0) {
            uint32_t mask = 0;
            // digits of 11, 11 and 10 bits
            for (int pass = 0; pass < 3; ++pass) {
                const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
                const int bins = pass == 2 ? 1024 : kSelBins;
#pragma unroll 2
                for (int j = (lo & ~3) + 4 * tid; j < hi; j += 4 * NT) {
                    const float4 x = value4(j);
                    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t k = weight_key(v[r]);
                        if (j + r >= lo && j + r < hi && (k & mask) == thr) atomicAdd(&hist[bin_at((k >> shift) & (bins - 1))], 1);
                    }
                }
                __syncthreads();
                // suffix sums from the largest bin: thread t owns bins kSelBins - 1 - (t * PER ..)
                int cnt[PER], own = 0;
#pragma unroll
                for (int b = 0; b < PER; ++b) {
                    cnt[b] = hist[bin_at(kSelBins - 1 - (tid * PER + b))];
                    own += cnt[b];
                }
                int scan = own;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, scan, o);
                    if (lane >= o) scan += y;
                }
                if (lane == 31) warp_a[warp] = scan;
                __syncthreads();
                int front = lane < warp ? warp_a[lane] : 0;  // NW <= 32
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) front += __shfl_xor_sync(0xffffffffu, front, o);
                int above = front + scan - own;  // keys in larger bins than this thread's
                if (above < rank && rank <= above + own) {  // one thread
#pragma unroll
                    for (int b = 0; b < PER; ++b) {
                        if (above < rank && rank <= above + cnt[b]) {
                            sh_digit = kSelBins - 1 - (tid * PER + b);
                            sh_rank = rank - above;
                        }
                        above += cnt[b];
                    }
                }
#pragma unroll
                for (int b = 0; b < PER; ++b) hist[bin_at(kSelBins - 1 - (tid * PER + b))] = 0;
                __syncthreads();
                thr |= static_cast<uint32_t>(sh_digit) << shift;
                mask |= static_cast<uint32_t>(bins - 1) << shift;
                rank = sh_rank;
            }
            ties = rank;
        } else {
            thr = 0xFFFFFFFFu;  // nothing of the middle is kept: no key is larger, no tie is taken
        }
    }
    // Ordered pass: a thread judges 4 consecutive positions of a tile; kept positions and ties are
    // counted by a scan over the threads.
    int base = 0, eq_base = 0;  // larger ones and ties in earlier tiles
    for (int j0 = 0; j0 < n; j0 += 4 * NT) {
        unsigned gt = 0, eq = 0;
        const int jb = j0 + 4 * tid;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (jb < n) {
            const float4 x = value4(jb);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = jb + r;
                if (j >= n) continue;
                if (n <= p.budget || j < lo || j >= hi) {
                    gt |= 1u << r;
                } else {
                    const uint32_t k = weight_key(v[r]);
                    gt |= (k > thr ? 1u : 0u) << r;
                    eq |= (k == thr ? 1u : 0u) << r;
                }
            }
        }
        // both counts in one scan: a tile has at most 4096 of each
        const int own = __popc(gt) | __popc(eq) << 16;
        int scan = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += y;
        }
        if (lane == 31) warp_b[warp] = scan;
        __syncthreads();
        const int mine = lane < NW ? warp_b[lane] : 0;
        int front = lane < warp ? mine : 0, all = mine;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            front += __shfl_xor_sync(0xffffffffu, front, o);
            all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        front += scan - own;
        int g0 = base + (front & 0xFFFF), e0 = eq_base + (front >> 16);
        base += all & 0xFFFF;
        eq_base += all >> 16;
        // uncached: every source of this tile has been read (the barrier above) before a weight
        // moves; destinations never pass their sources, so later tiles' sources stay whole
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool g = gt >> r & 1, q = eq >> r & 1;
            if (g || (q && e0 < ties)) {
                const int y = g0 + min(e0, ties);  // larger ones before it, and the ties taken so far
                kept[y] = jb + r;
                *at(ntbl, y) = v[r];
            }
            g0 += g;
            e0 += q;
        }
        __syncthreads();
    }
    for (int y = m + tid; y < p.budget; y += NT) kept[y] = -1;
}

// Kept K (blockIdx.z even) or V rows into the new blocks: one CTA per work item (rows
// [y0, y1) of a sequence's new positions), (layer, KV head), tensor. Rows move in tiles of up to
// kMoveWords words: the tile's row addresses first (one chain of loads, kept position -> block ->
// slot, per row and not per word), then every word of it is read before any is written. A sequence
// whose new table names some of its old blocks is one item, so that its tiles run in order (see
// evict_select_kernel). HBM bound: every kept row is read and written once.
constexpr int kMoveThreads = 256, kMovePer = 8, kMoveWords = kMoveThreads * kMovePer;
static_assert(kMoveWords >= kMaxBoundedDim, "a tile holds a row of any word size");
template <typename W>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
    __shared__ int64_t src[kMoveThreads], dst[kMoveThreads];  // first word of each row of the tile
    const int item = blockIdx.x;
    const int i = p.items[3 * item], y0 = p.items[3 * item + 1], y1 = p.items[3 * item + 2];
    const int h = blockIdx.y % p.kvh, layer = blockIdx.y / p.kvh;
    const int words = p.row_words;
    W* base = static_cast<W*>(blockIdx.z == 0 ? p.pool_k : p.pool_v) +
              (static_cast<size_t>(p.layer0 + layer) * p.num_blocks * p.bs * p.kvh + h) * words;
    const int32_t* tbl = p.ids + p.indptr[i];
    const int32_t* ntbl = p.new_ids + p.new_indptr[i];
    const int32_t* kept = p.kept + ((static_cast<size_t>(layer) * p.nseq + i) * p.kvh + h) * p.budget;
    const int64_t stride = static_cast<int64_t>(p.kvh) * words;  // words from one slot to the next
    const int rows = min(kMoveThreads, kMoveWords / words);
    auto word_of = [&](const int32_t* t, int j) {
        const int b = div_by(j, p.bs, p.bs_shift);
        return (static_cast<int64_t>(t[b]) * p.bs + (j - b * p.bs)) * stride;
    };
    for (int y = y0; y < y1; y += rows) {
        const int nr = min(rows, y1 - y), total = nr * words;
        if (threadIdx.x < nr) {
            src[threadIdx.x] = word_of(tbl, kept[y + threadIdx.x]);
            dst[threadIdx.x] = word_of(ntbl, y + threadIdx.x);
        }
        __syncthreads();
        W val[kMovePer];
#pragma unroll
        for (int e = 0; e < kMovePer; ++e) {
            const int x = e * kMoveThreads + threadIdx.x;
            if (x < total) {
                const int r = div_by(x, words, p.words_shift);
                val[e] = base[src[r] + (x - r * words)];
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kMovePer; ++e) {
            const int x = e * kMoveThreads + threadIdx.x;
            if (x < total) {
                const int r = div_by(x, words, p.words_shift);
                base[dst[r] + (x - r * words)] = val[e];
            }
        }
        __syncthreads();
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
    if (p.max_units >= 16)
        weight_scores_kernel<true><<<dim3(p.w.ntouched, (p.kvh * p.bs + 31) / 32), 256, 0, st>>>(p);
    else
        weight_scores_kernel<false><<<(p.w.ntouched + 7) / 8, 256, 0, st>>>(p);
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

cudaError_t launch_clear_weights(float* weights, const int64_t* slots, const int32_t* row_seq, const int32_t* offsets,
                                 const int32_t* starts, const int32_t* indptr, const int32_t* ids, int bs, int kvh,
                                 int64_t n, cudaStream_t st) {
    if (n <= 0) return cudaSuccess;
    const int grid = static_cast<int>(std::min<int64_t>((n * kvh + 255) / 256, 148 * 8));
    clear_weights_kernel<<<grid, 256, 0, st>>>(weights, slots, row_seq, offsets, starts, indptr, ids, bs, kvh, n);
    return cudaGetLastError();
}

cudaError_t launch_evict(const EvictParams& p, int max_len, cudaStream_t st) {
    if (p.nseq <= 0) return cudaSuccess;
    EvictParams q = p;
    const auto log2_of = [](int x) {
        int s = 0;
        while ((1 << s) < x) ++s;
        return (1 << s) == x ? s : -1;
    };
    // the weights of a sequence are kept in shared memory while they fit
    constexpr int kMaxCached = 40960;  // floats: 160 KB
    q.cache_cap = std::min(max_len, kMaxCached);
    q.bs_shift = log2_of(p.bs);
    const size_t smem = (static_cast<size_t>(q.cache_cap) * sizeof(float) + 15) & ~size_t(15);
    // 1024 threads a CTA where one CTA per SM is all there is to run, or fits beside its weights
    const int64_t ctas = static_cast<int64_t>(p.nseq) * p.kvh * p.layers;
    const bool wide = max_len > 2048 && (ctas <= 2 * 148 || max_len > 16384);
    auto sel = wide ? evict_select_kernel<1024> : evict_select_kernel<256>;
    cudaError_t e = cudaFuncSetAttribute(sel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kMaxCached * static_cast<int>(sizeof(float)));
    if (e != cudaSuccess) return e;
    sel<<<dim3(p.nseq, p.kvh, p.layers), wide ? 1024 : 256, smem, st>>>(q);
    e = cudaGetLastError();
    if (e != cudaSuccess || p.nitems <= 0) return e;
    const dim3 grid(p.nitems, p.kvh * p.layers, 2);
    // the widest word that divides a row
    const int w = p.row_bytes % 16 == 0 ? 16 : p.row_bytes % 4 == 0 ? 4 : 2;
    q.row_words = p.row_bytes / w;
    q.words_shift = log2_of(q.row_words);
    if (w == 16) evict_move_kernel<uint4><<<grid, kMoveThreads, 0, st>>>(q);
    else if (w == 4) evict_move_kernel<uint32_t><<<grid, kMoveThreads, 0, st>>>(q);
    else evict_move_kernel<uint16_t><<<grid, kMoveThreads, 0, st>>>(q);
    return cudaGetLastError();
}

}  // namespace pk

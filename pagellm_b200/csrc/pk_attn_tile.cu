// Windowed attention with sinks, and its accumulated weights, for chunks of rows on the CUDA cores:
// the pools that the tensor-core kernels do not take (float32 ones above all, whose scores and sums
// stay in float32 throughout), where a sequence brings kTileMinCols (row, head) pairs of a KV head or
// more. With fewer, or with head_dim above 256, cc_attn_kernel and weight_rows_kernel take them.
//
// A row at position p sees the keys j <= p with j < sinks or j > p - window.
//
// tile_attn_kernel: one CTA per (up to 64 consecutive columns of a sequence and KV head, a column being
// a (token, head) pair; split of their visible keys). 64 keys at a time go through shared memory; each
// of 256 threads holds 4 x 4 scores and 4 rows x D / 16 outputs in registers. The 16 threads of a row
// lie in one half-warp, so that the running maximum takes four shuffles and probabilities pass from
// scores to outputs inside a warp, through the shared memory of the keys already used. Products are
// packed pairs of float32 multiply-adds. With few columns and a long context the keys are split over
// CTAs, whose partials the last one to finish joins, in order.
// Bound by the multiply-adds: 4 D of them per (row, head, key), of which 53 % of the SMs' 128 a clock are
// reached (scores read 8 words of shared memory per 64 multiply-adds). cc_attn_kernel, a key per group
// of lanes along its row, spends as much again on shuffles and reads every key once per row: a
// 1024-token chunk of 16 heads of 128 behind 1024 cached tokens, window 1000, float32: 925 us there, 298
// here (113 at the full rate). A tile costs its 64 columns even where fewer are live: with 16 of them
// (4 rows of 4 heads, 16 contexts up to 4096, window 1000) 168 us here, 142 there; hence kTileMinCols.
//
// tile_weight_kernel: the same scores, summed the other way - a CTA keeps 64 keys of a KV head and goes
// over all columns that see any of them, adding 2^(s - m) / l into 4 sums per thread, which are joined
// at the end in a fixed order; where keys are few the columns are dealt to several CTAs. 240 us for that
// chunk without a window; a warp per key (weight_rows_kernel) took 1950.

#include <cuda_bf16.h>

#include <algorithm>

#include "pk_device.cuh"
#include "pk_internal.h"
#include "pk_tcgen05.cuh"

namespace pk {

namespace {

constexpr int kThreads = 256, kCols = kTileCols, kKeys = kTileKeys;
constexpr int kPStride = kKeys + 4;  // floats of a row of probabilities (an odd number of 16-byte words)
static_assert(kCols == 64 && kKeys == 64, "4 x 4 scores per thread of 256");

__device__ __forceinline__ float4 vec4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ float4 vec4(const __nv_bfloat16* p) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    return make_float4(bf16_lo_f(w.x), bf16_hi_f(w.x), bf16_lo_f(w.y), bf16_hi_f(w.y));
}
__device__ __forceinline__ void put4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void put4(__nv_bfloat16* p, float4 x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
}

// Rows of shared memory: an odd number of 16-byte words, so that equal words of consecutive rows
// lie in different banks; fixed at compile time (NC: 64 values each), so that loads need one base.
template <int NC>
constexpr int kStride = 4 * (16 * NC + 1);

// A row of D values to shared memory by eight lanes, CH of its 16-byte words each (zeros where !live).
template <int CH, typename T>
__device__ __forceinline__ void stage_row(float* dst, const T* src, bool live, int l8, int nvec) {
    float4 x[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = l8 + 8 * i;
        x[i] = live && c < nvec ? vec4(src + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (l8 + 8 * i < nvec) put4(dst + 4 * (l8 + 8 * i), x[i]);
}

// s[i][j] = q row (r0 + i) . key (tc + 16 j)
template <int NC>
__device__ __forceinline__ void scores_4x4(const float* qs, const float* ks, int r0, int tc, int nvec, float (&s)[4][4]) {
    constexpr int st = kStride<NC>;
    qs += r0 * st;
    ks += tc * st;
    uint64_t a2[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) a2[i][j] = 0;
#pragma unroll 4
    for (int c = 0; c < nvec; ++c) {
        ulonglong2 a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const ulonglong2*>(qs + i * st + 4 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const ulonglong2*>(ks + 16 * j * st + 4 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a2[i][j] = fma_f32x2(a[i].x, b[j].x, a2[i][j]);
                a2[i][j] = fma_f32x2(a[i].y, b[j].y, a2[i][j]);
            }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float lo, hi;
            unpack_f32x2(a2[i][j], lo, hi);
            s[i][j] = lo + hi;
        }
}

template <typename T, typename IO, int NC>
__global__ void __launch_bounds__(kThreads, NC <= 2 ? 2 : 1) tile_attn_kernel(const TileParams p) {
    extern __shared__ __align__(16) float sm[];
    __shared__ int sh_last;
    constexpr int st = kStride<NC>;
    const int nvec = p.D / 4;
    float* qs = sm;                                   // [64][st]
    float* vs = qs + kCols * st;                      // [64][st]
    float* ks = vs + kKeys * st;                      // [64][st], then probabilities [64][kPStride]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tc = lane & 15, r0 = warp * 8 + (lane >> 4) * 4;  // this thread's columns r0 .. r0 + 3
    const int4 u = __ldg(p.meta + blockIdx.x);        // first row, first table entry, its position, tokens
    const int kh = blockIdx.y, split = blockIdx.z, nsplit = gridDim.z;
    const int g = p.H / p.kvh, ncol = u.w * g;
    const int pos = u.z, last = pos + u.w - 1;
    const int lo = max(0, pos - p.window + 1), ns = min(p.sinks, lo);
    const int nvis = ns + last - lo + 1, ntiles = (nvis + kKeys - 1) / kKeys;
    const int x_begin = static_cast<int>(static_cast<int64_t>(ntiles) * split / nsplit) * kKeys;
    const int x_end = min(nvis, static_cast<int>(static_cast<int64_t>(ntiles) * (split + 1) / nsplit) * kKeys);
    const int32_t* tbl = p.ids + u.y;
    const T* kpool = static_cast<const T*>(p.pool_k);
    const T* vpool = static_cast<const T*>(p.pool_v);
    const int l8 = tid & 7;
    // column c: place of its row in [rows][H]
    auto column = [&](int c) { return static_cast<size_t>(u.x + c / g) * p.H + kh * g + c % g; };

    for (int c = tid >> 3; c < kCols; c += kThreads / 8)
        stage_row<2 * NC>(qs + c * st, static_cast<const IO*>(p.q) + column(c < ncol ? c : 0) * p.D, c < ncol, l8, nvec);
    int cpos[4];
    float m[4], l[4];
    uint64_t acc[4][NC][2];
    int cv[NC];
#pragma unroll
    for (int v = 0; v < NC; ++v) cv[v] = 4 * min(tc + 16 * v, nvec - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cpos[i] = pos + min(r0 + i, ncol - 1) / g;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int v = 0; v < NC; ++v) acc[i][v][0] = acc[i][v][1] = 0;
    }
    for (int x0 = x_begin; x0 < x_end; x0 += kKeys) {
        __syncthreads();  // the last tile's probabilities and values are used
#pragma unroll
        for (int k = tid >> 3; k < kKeys; k += kThreads / 8) {
            const int x = x0 + k;
            const bool live = x < x_end;
            const int j = live ? (x < ns ? x : x - ns + lo) : pos;
            const int b = p.bs_shift >= 0 ? j >> p.bs_shift : j / p.bs;
            const size_t off = ((static_cast<size_t>(__ldg(tbl + b)) * p.bs + (j - b * p.bs)) * p.kvh + kh) * p.D;
            stage_row<2 * NC>(ks + k * st, kpool + off, live, l8, nvec);
            stage_row<2 * NC>(vs + k * st, vpool + off, live, l8, nvec);
        }
        __syncthreads();
        float s[4][4];
        scores_4x4<NC>(qs, ks, r0, tc, nvec, s);
        __syncthreads();  // all have read the keys
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int x = x0 + tc + 16 * j;
                const int kp = x < ns ? x : x - ns + lo;
                const bool see = x < x_end && kp <= cpos[i] && (kp < p.sinks || kp > cpos[i] - p.window);
                s[i][j] = see ? s[i][j] * p.qscale : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mnew = fmaxf(m[i], mx), base = mnew == -INFINITY ? 0.f : mnew;
            const float corr = exp2f(m[i] - base);
            m[i] = mnew;
            l[i] *= corr;
            const uint64_t c2 = pack_f32x2(corr, corr);
#pragma unroll
            for (int v = 0; v < NC; ++v) {
                acc[i][v][0] = fma_f32x2(acc[i][v][0], c2, 0);
                acc[i][v][1] = fma_f32x2(acc[i][v][1], c2, 0);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w = exp2f(s[i][j] - base);
                l[i] += w;
                ks[(r0 + i) * kPStride + tc + 16 * j] = w;
            }
        }
        __syncwarp();
        const int n4 = (min(kKeys, x_end - x0) + 3) / 4;
        for (int k4 = 0; k4 < n4; ++k4) {
            float w[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(w[i]) = *reinterpret_cast<const float4*>(ks + (r0 + i) * kPStride + 4 * k4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                ulonglong2 y[NC];
#pragma unroll
                for (int v = 0; v < NC; ++v) y[v] = *reinterpret_cast<const ulonglong2*>(vs + (4 * k4 + kk) * st + cv[v]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint64_t w2 = pack_f32x2(w[i][kk], w[i][kk]);
#pragma unroll
                    for (int v = 0; v < NC; ++v) {
                        acc[i][v][0] = fma_f32x2(w2, y[v].x, acc[i][v][0]);
                        acc[i][v][1] = fma_f32x2(w2, y[v].y, acc[i][v][1]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    IO* out = static_cast<IO*>(p.out);
    const size_t unit = static_cast<size_t>(blockIdx.x) * p.kvh + kh;
    const int pst = p.D + 4;  // floats of a partial row: D sums, maximum, sum (rows stay on 16 bytes)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = r0 + i;
        if (c >= ncol) continue;
        const float inv = nsplit == 1 ? 1.f / l[i] : 1.f;
        float* part = nsplit == 1 ? nullptr : p.part + ((unit * nsplit + split) * kCols + c) * pst;
#pragma unroll
        for (int v = 0; v < NC; ++v) {
            if (tc + 16 * v >= nvec) continue;
            float4 a;
            unpack_f32x2(acc[i][v][0], a.x, a.y);
            unpack_f32x2(acc[i][v][1], a.z, a.w);
            a.x *= inv, a.y *= inv, a.z *= inv, a.w *= inv;
            if (nsplit == 1) put4(out + column(c) * p.D + cv[v], a);
            else put4(part + cv[v], a);
        }
        if (tc == 0) {
            if (nsplit > 1) part[p.D] = m[i], part[p.D + 1] = l[i];
            else if (p.ml != nullptr) p.ml[column(c)] = make_float2(m[i], inv);
        }
    }
    if (nsplit == 1) return;
    // ---- the last CTA of the unit joins the partials in order
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        sh_last = atomicAdd(p.counters + unit, 1) == nsplit - 1;
        if (sh_last) p.counters[unit] = 0;  // for the next launch
    }
    __syncthreads();
    if (!sh_last) return;
    __threadfence();
    const float* all = p.part + unit * nsplit * kCols * pst;
    for (int x = tid; x < ncol * nvec; x += kThreads) {
        const int c = x / nvec, d = 4 * (x - c * nvec);
        float mx = -INFINITY, den = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < nsplit; ++s) mx = fmaxf(mx, __ldcg(all + (s * kCols + c) * pst + p.D));
        for (int s = 0; s < nsplit; ++s) {
            const float* ph = all + (s * kCols + c) * pst;
            const float ms = __ldcg(ph + p.D);
            const float f = ms == -INFINITY ? 0.f : exp2f(ms - mx);
            const float4 y = __ldcg(reinterpret_cast<const float4*>(ph + d));
            den = fmaf(f, __ldcg(ph + p.D + 1), den);
            a.x = fmaf(f, y.x, a.x), a.y = fmaf(f, y.y, a.y), a.z = fmaf(f, y.z, a.z), a.w = fmaf(f, y.w, a.w);
        }
        const float inv = 1.f / den;
        put4(out + column(c) * p.D + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
        if (p.ml != nullptr && d == 0) p.ml[column(c)] = make_float2(mx, inv);
    }
}

template <typename T, typename IO, int NC>
__global__ void __launch_bounds__(kThreads, NC <= 2 ? 2 : 1) tile_weight_kernel(const TileParams p, const TileWeightParams w) {
    extern __shared__ __align__(16) float sm[];
    __shared__ float sums[kThreads / 32][kKeys];
    __shared__ int sh_last;
    constexpr int st = kStride<NC>;
    const int nvec = p.D / 4;
    float* ks = sm;              // [64][st]
    float* qs = sm + kKeys * st;  // [64][st]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tc = lane & 15, r0 = warp * 8 + (lane >> 4) * 4, l8 = tid & 7;
    // sequence: first row, first table entry, start, rows; keys: first touched block, their number, first slot
    const int4 a0 = __ldg(w.meta + 2 * blockIdx.x), a1 = __ldg(w.meta + 2 * blockIdx.x + 1);
    const int row0 = a0.x, start = a0.z, n = a0.w, slots = a1.y * p.bs, slot0 = a1.z;
    const int kh = blockIdx.y, g = p.H / p.kvh, ctx = start + n;
    const int lo = max(0, start - p.window + 1);
    const int32_t* tbl = p.ids + a0.y;
    // slot x of the sequence's touched blocks: its position (-1: no key that a row sees) and place
    auto slot = [&](int x, int& phys, int& t) {
        phys = t = 0;
        if (x >= slots) return -1;
        const int b = p.bs_shift >= 0 ? x >> p.bs_shift : x / p.bs;
        t = x - b * p.bs;
        const int lb = __ldg(w.t_blk + a1.x + b);
        phys = __ldg(tbl + lb);
        const int64_t j = static_cast<int64_t>(lb) * p.bs + t;
        return j < ctx && (j < p.sinks || j >= lo) ? static_cast<int>(j) : -1;
    };
    int phys, t;
    for (int k = tid >> 3; k < kKeys; k += kThreads / 8) {
        const int j = slot(slot0 + k, phys, t);
        stage_row<2 * NC>(ks + k * st,
                          static_cast<const T*>(p.pool_k) + ((static_cast<size_t>(phys) * p.bs + t) * p.kvh + kh) * p.D,
                          j >= 0, l8, nvec);
    }
    // this thread's keys, the tokens that see them, and the CTA's: those that see any
    int kp[4], ra = INT32_MAX, rb = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kp[j] = slot(slot0 + tc + 16 * j, phys, t);
        if (kp[j] < 0) continue;
        ra = min(ra, max(0, kp[j] - start));
        rb = max(rb, kp[j] < p.sinks || kp[j] - start > INT32_MAX - p.window ? n : min(n, kp[j] - start + p.window));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        ra = min(ra, __shfl_xor_sync(0xffffffffu, ra, o));
        rb = max(rb, __shfl_xor_sync(0xffffffffu, rb, o));
    }
    const int tpt = kCols / g;  // tokens of a column tile
    // columns that this thread stages and scores: places in a tile's [tokens][H] rows, and tokens
    constexpr int kStage = kCols * 8 / kThreads;
    int at_stage[kStage], at_row[4], tok_row[4];
#pragma unroll
    for (int x = 0; x < kStage; ++x) {
        const int c = min((tid >> 3) + x * (kThreads / 8), tpt * g - 1);
        at_stage[x] = c / g * p.H + c % g;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = min(r0 + i, tpt * g - 1);
        tok_row[i] = c / g;
        at_row[i] = tok_row[i] * p.H + c % g;
    }
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const int ntiles = rb > ra ? (rb - ra + tpt - 1) / tpt : 0;
    const int c_begin = static_cast<int>(static_cast<int64_t>(ntiles) * blockIdx.z / gridDim.z);
    const int c_end = static_cast<int>(static_cast<int64_t>(ntiles) * (blockIdx.z + 1) / gridDim.z);
    for (int ct = c_begin; ct < c_end; ++ct) {
        const int tok0 = ra + ct * tpt, ncol = min(tpt, rb - tok0) * g;
        const size_t first = static_cast<size_t>(row0 + tok0) * p.H + kh * g;
        const IO* qp = static_cast<const IO*>(p.q) + first * p.D;
        __syncthreads();  // the last tile's queries are used
#pragma unroll
        for (int x = 0; x < kStage; ++x) {
            const int c = (tid >> 3) + x * (kThreads / 8);
            stage_row<2 * NC>(qs + c * st, qp + static_cast<int64_t>(at_stage[x]) * p.D, c < ncol, l8, nvec);
        }
        float2 ml[4];
        int pos[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool live = r0 + i < ncol;
            ml[i] = live ? __ldg(p.ml + first + at_row[i]) : make_float2(0.f, 0.f);
            pos[i] = live ? start + tok0 + tok_row[i] : -1;  // (-1: sees nothing)
        }
        __syncthreads();
        float s[4][4];
        scores_4x4<NC>(qs, ks, r0, tc, nvec, s);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool see = kp[j] >= 0 && kp[j] <= pos[i] && (kp[j] < p.sinks || kp[j] > pos[i] - p.window);
                if (see) sum[j] += exp2f(s[i][j] * p.qscale - ml[i].x) * ml[i].y;
            }
    }
    // ---- join the rows: half-warps, then warps in order, then the CTAs of the keys in order
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 16);
        if (lane < 16) sums[warp][tc + 16 * j] = sum[j];
    }
    __syncthreads();
    const size_t unit = static_cast<size_t>(blockIdx.x) * p.kvh + kh;
    const int nparts = gridDim.z;
    float total = 0.f;
    if (tid < kKeys) {
        for (int x = 0; x < kThreads / 32; ++x) total += sums[x][tid];
        if (nparts > 1) w.part[(unit * nparts + blockIdx.z) * kKeys + tid] = total;
    }
    if (nparts > 1) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            sh_last = atomicAdd(w.counters + unit, 1) == nparts - 1;
            if (sh_last) w.counters[unit] = 0;  // for the next launch
        }
        __syncthreads();
        if (!sh_last) return;
        __threadfence();
        if (tid < kKeys) {
            total = 0.f;
            for (int z = 0; z < nparts; ++z) total += __ldcg(w.part + (unit * nparts + z) * kKeys + tid);
        }
    }
    if (tid >= kKeys) return;
    const int j = slot(slot0 + tid, phys, t);
    if (j < 0) return;
    float* dst = w.weights + (static_cast<size_t>(phys) * p.kvh + kh) * p.bs + t;
    *dst = w.add && j < start ? *dst + total : total;
}

template <typename K>
cudaError_t allow_smem(K kern, size_t smem) {
    return smem > 48 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem))
                            : cudaSuccess;
}

template <typename T, typename IO, int NC>
cudaError_t launch_attn_n(const TileParams& p, cudaStream_t st) {
    static_assert(kKeys * kStride<NC> >= kCols * kPStride, "the probabilities take the place of the keys");
    const size_t smem = (kCols + 2 * kKeys) * kStride<NC> * sizeof(float);
    cudaError_t e = allow_smem(tile_attn_kernel<T, IO, NC>, smem);
    if (e != cudaSuccess) return e;
    tile_attn_kernel<T, IO, NC><<<dim3(p.nunits, p.kvh, p.nsplit), kThreads, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T, typename IO, int NC>
cudaError_t launch_weight_n(const TileParams& p, const TileWeightParams& w, cudaStream_t st) {
    const size_t smem = (kCols + kKeys) * kStride<NC> * sizeof(float);
    cudaError_t e = allow_smem(tile_weight_kernel<T, IO, NC>, smem);
    if (e != cudaSuccess) return e;
    tile_weight_kernel<T, IO, NC><<<dim3(w.ntiles, p.kvh, w.nparts), kThreads, smem, st>>>(p, w);
    return cudaGetLastError();
}

template <typename T, typename IO>
cudaError_t launch_attn_t(const TileParams& p, cudaStream_t st) {
    return p.D <= 64 ? launch_attn_n<T, IO, 1>(p, st) : p.D <= 128 ? launch_attn_n<T, IO, 2>(p, st) : launch_attn_n<T, IO, 4>(p, st);
}

template <typename T, typename IO>
cudaError_t launch_weight_t(const TileParams& p, const TileWeightParams& w, cudaStream_t st) {
    return p.D <= 64    ? launch_weight_n<T, IO, 1>(p, w, st)
           : p.D <= 128 ? launch_weight_n<T, IO, 2>(p, w, st)
                        : launch_weight_n<T, IO, 4>(p, w, st);
}

}  // namespace

cudaError_t launch_tile_attention(int dtype, bool io16, const TileParams& p, cudaStream_t st) {
    if (p.D % 4 != 0 || p.D > kTileMaxDim || p.kvh > 65535 || (dtype == 0 && io16)) return cudaErrorInvalidValue;
    if (dtype == 0) return launch_attn_t<float, float>(p, st);
    return io16 ? launch_attn_t<__nv_bfloat16, __nv_bfloat16>(p, st) : launch_attn_t<__nv_bfloat16, float>(p, st);
}

cudaError_t launch_tile_weights(int dtype, bool io16, const TileParams& p, const TileWeightParams& w, cudaStream_t st) {
    if (p.D % 4 != 0 || p.D > kTileMaxDim || p.kvh > 65535 || (dtype == 0 && io16)) return cudaErrorInvalidValue;
    if (dtype == 0) return launch_weight_t<float, float>(p, w, st);
    return io16 ? launch_weight_t<__nv_bfloat16, __nv_bfloat16>(p, w, st) : launch_weight_t<__nv_bfloat16, float>(p, w, st);
}

}  // namespace pk

// Windowed attention with sinks on the CUDA cores, for the pools that the tensor-core kernels do not
// take: float32 pools, and bf16 pools of other head sizes, block sizes or many KV heads. Rows of
// 4-element multiples up to 512; others go to bounded_rows_kernel.
//
// A row at position p sees the keys j <= p with j < sinks or j > p - window, numbered 0..nvis-1: the
// sinks in front of the window, then the window.
//
// One CTA per (row, KV head, group of up to G of its query heads, split of the visible keys). A key's
// row lies across LPK lanes as 4-element vectors, so that a warp takes 32 / LPK keys side by side
// with 16-byte (float) loads, KB of them in flight; scores are summed over the LPK lanes by shuffles
// and serve all G heads from one read of K. Every lane group keeps its own running maximum, sum and
// output; groups and warps are joined once at the end, in a fixed order. With few rows and long
// contexts the keys are split over CTAs, whose partials the last one to finish joins, in order.
// Many rows are bound by the latency of the keys' loads: a group of 4 heads of 128 takes 244 registers, so two
// CTAs share an SM and 8 warps have too few loads in flight (32 decodes of 4 x 8 heads over 74k float32
// tokens with their weights, 604 MB: 270 us, 2.2 TB/s; issue slots 31 % busy, multiply-add pipe 17 %, the
// first stall is the load). Few rows are bound by the chain row record -> block id -> key -> join (8 decodes
// over a small pool: 9 us).
//
// Fused append: keys of the step itself are read from the inputs, rounded as the pool stores them,
// and the CTA of (row, KV head, first group, first split) stores the row. Fused weights (one row per
// sequence, one split, one group): the scores stay in shared memory until the row's maximum and sum
// are known, then every visible key's weight is stored.

#include <cuda_bf16.h>

#include <algorithm>

#include "pk_device.cuh"
#include "pk_internal.h"

namespace pk {

namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return make_float4(bf16_lo_f(w.x), bf16_hi_f(w.x), bf16_lo_f(w.y), bf16_hi_f(w.y));
}
__device__ __forceinline__ void store4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
}
// x as the pool would hold it
__device__ __forceinline__ float4 as_pool(float4 x, const float*) { return x; }
__device__ __forceinline__ float4 as_pool(float4 x, const __nv_bfloat16*) {
    const uint32_t a = pack_bf16(x.x, x.y), b = pack_bf16(x.z, x.w);
    return make_float4(bf16_lo_f(a), bf16_hi_f(a), bf16_lo_f(b), bf16_hi_f(b));
}

template <typename T, typename IO, int G, int NV, int LPK>
__global__ void __launch_bounds__(kWarps * 32) cc_attn_kernel(const CcParams p) {
    constexpr int KPW = 32 / LPK;                            // keys a warp takes side by side
    constexpr int KB = NV >= 4 ? 2 : 4;                      // keys of a lane group in flight
    extern __shared__ __align__(16) float sm[];              // [kWarps][G][D] outputs (16-byte words), then the scores (weights)
    __shared__ float sm_m[kWarps][G], sm_l[kWarps][G];
    __shared__ int sh_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane % LPK, grp = lane / LPK;
    const int4 r0 = __ldg(p.meta + 2 * blockIdx.x), r1 = __ldg(p.meta + 2 * blockIdx.x + 1);
    const int row = r0.x, pos = r0.z, start = r0.w, row_first = r1.x;
    const int32_t* tbl = p.ids + r0.y;
    const int kh = blockIdx.y % p.kvh, hg = blockIdx.y / p.kvh;
    const int split = blockIdx.z, nsplit = gridDim.z;
    const int g = p.H / p.kvh;
    const int ng = min(G, g - hg * G);                       // live heads of this group
    const int head0 = kh * g + hg * G;
    const int nvec = p.D / 4;
    const int lo = max(0, pos - p.window + 1);
    const int ns = min(p.sinks, lo);
    const int nvis = ns + pos - lo + 1;
    const int x_begin = static_cast<int>(static_cast<int64_t>(nvis) * split / nsplit);
    const int x_end = static_cast<int>(static_cast<int64_t>(nvis) * (split + 1) / nsplit);
    const T* kpool = static_cast<const T*>(p.pool_k);
    const T* vpool = static_cast<const T*>(p.pool_v);
    const IO* k_new = static_cast<const IO*>(p.k_new);
    const IO* v_new = static_cast<const IO*>(p.v_new);
    float* scores = sm + kWarps * G * p.D;                   // [nvis][G] when weights are fused
    const bool keep = p.weights != nullptr;

    float4 q[G][NV], acc[G][NV];
    float m[G], l[G];
    const IO* qp = static_cast<const IO*>(p.q) + (static_cast<size_t>(row) * p.H + head0) * p.D;
#pragma unroll
    for (int h = 0; h < G; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = sub + LPK * v;
            q[h][v] = h < ng && c < nvec ? load4(qp + h * p.D + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
            acc[h][v] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    // key x: its place in the pool, or among the step's rows
    auto key_at = [&](int x, bool& fresh) -> size_t {
        const int j = x < ns ? x : x - ns + lo;
        fresh = k_new != nullptr && j >= start;
        if (fresh) return (static_cast<size_t>(row_first + j - start) * p.kvh + kh) * p.D;
        const int b = p.bs_shift >= 0 ? j >> p.bs_shift : j / p.bs;
        return ((static_cast<size_t>(__ldg(tbl + b)) * p.bs + (j - b * p.bs)) * p.kvh + kh) * p.D;
    };
    constexpr int kStep = kWarps * KPW;  // keys between a lane group's consecutive ones
    for (int x0 = x_begin + warp * KPW + grp; __any_sync(0xffffffffu, x0 < x_end); x0 += kStep * KB) {
        float4 kv[KB][NV], vv[KB][NV];
        bool live[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int x = x0 + b * kStep;
            live[b] = x < x_end;
            bool fresh = false;
            const size_t off = live[b] ? key_at(x, fresh) : 0;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = sub + LPK * v;
                kv[b][v] = vv[b][v] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (!live[b] || c >= nvec) continue;
                if (fresh) {
                    kv[b][v] = as_pool(load4(k_new + off + 4 * c), kpool);
                    vv[b][v] = as_pool(load4(v_new + off + 4 * c), vpool);
                } else {
                    kv[b][v] = load4(kpool + off + 4 * c);
                    vv[b][v] = load4(vpool + off + 4 * c);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < G; ++h) {
            float s[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                float d = 0.f;
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    d = fmaf(q[h][v].x, kv[b][v].x, d);
                    d = fmaf(q[h][v].y, kv[b][v].y, d);
                    d = fmaf(q[h][v].z, kv[b][v].z, d);
                    d = fmaf(q[h][v].w, kv[b][v].w, d);
                }
#pragma unroll
                for (int o = LPK / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                s[b] = live[b] ? d * p.qscale : -INFINITY;
                if (keep && live[b] && sub == 0) scores[(x0 + b * kStep) * G + h] = s[b];
            }
            float mnew = m[h];
#pragma unroll
            for (int b = 0; b < KB; ++b) mnew = fmaxf(mnew, s[b]);
            const float base = mnew == -INFINITY ? 0.f : mnew;
            const float corr = exp2f(m[h] - base);
            float w[KB];
            l[h] *= corr;
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                w[b] = exp2f(s[b] - base);
                l[h] += w[b];
            }
            m[h] = mnew;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float4 a = acc[h][v];
                a.x *= corr, a.y *= corr, a.z *= corr, a.w *= corr;
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    a.x = fmaf(w[b], vv[b][v].x, a.x);
                    a.y = fmaf(w[b], vv[b][v].y, a.y);
                    a.z = fmaf(w[b], vv[b][v].z, a.z);
                    a.w = fmaf(w[b], vv[b][v].w, a.w);
                }
                acc[h][v] = a;
            }
        }
    }
    // the step's row into the pool
    if (k_new != nullptr && hg == 0 && split == 0) {
        const int b = pos / p.bs;
        const size_t dst = ((static_cast<size_t>(__ldg(tbl + b)) * p.bs + (pos - b * p.bs)) * p.kvh + kh) * p.D;
        const size_t src = (static_cast<size_t>(row) * p.kvh + kh) * p.D;
        for (int c = threadIdx.x; c < nvec; c += blockDim.x) {
            store4(const_cast<T*>(kpool) + dst + 4 * c, load4(k_new + src + 4 * c));
            store4(const_cast<T*>(vpool) + dst + 4 * c, load4(v_new + src + 4 * c));
        }
    }
    // ---- join the lane groups of a warp, then the warps
#pragma unroll
    for (int h = 0; h < G; ++h) {
        float mx = m[h];
#pragma unroll
        for (int o = LPK; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float f = m[h] == -INFINITY ? 0.f : exp2f(m[h] - mx);
        float sum = l[h] * f;
#pragma unroll
        for (int o = LPK; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            sm_m[warp][h] = mx;
            sm_l[warp][h] = sum;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float4 a = acc[h][v];
            a.x *= f, a.y *= f, a.z *= f, a.w *= f;
#pragma unroll
            for (int o = LPK; o < 32; o <<= 1) {
                a.x += __shfl_xor_sync(0xffffffffu, a.x, o);
                a.y += __shfl_xor_sync(0xffffffffu, a.y, o);
                a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
                a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
            }
            const int c = sub + LPK * v;
            if (grp == 0 && c < nvec) store4(sm + (warp * G + h) * p.D + 4 * c, a);
        }
    }
    __syncthreads();
    // maximum, sum and (un-normalised) output dimension d of head h over the warps
    auto joined_ml = [&](int h, float& mx, float& den, float (&f)[kWarps]) {
        mx = -INFINITY;
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm_m[w][h]);
        den = 0.f;
        for (int w = 0; w < kWarps; ++w) {
            f[w] = sm_m[w][h] == -INFINITY ? 0.f : exp2f(sm_m[w][h] - mx);
            den += f[w] * sm_l[w][h];
        }
    };
    IO* out = static_cast<IO*>(p.out) + (static_cast<size_t>(row) * p.H + head0) * p.D;
    if (nsplit == 1) {
        for (int c = threadIdx.x; c < ng * nvec; c += blockDim.x) {
            const int h = c / nvec, d = 4 * (c - h * nvec);
            float mx, den, f[kWarps];
            joined_ml(h, mx, den, f);
            const float inv = 1.f / den;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float4 x = load4(sm + (w * G + h) * p.D + d);
                a.x = fmaf(f[w], x.x, a.x);
                a.y = fmaf(f[w], x.y, a.y);
                a.z = fmaf(f[w], x.z, a.z);
                a.w = fmaf(f[w], x.w, a.w);
            }
            store4(out + h * p.D + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
            if (p.ml != nullptr && d == 0) p.ml[static_cast<size_t>(row) * p.H + head0 + h] = make_float2(mx, inv);
        }
        if (keep) {
            float mx[G], inv[G];
#pragma unroll
            for (int h = 0; h < G; ++h) {
                float den, f[kWarps];
                joined_ml(h, mx[h], den, f);
                inv[h] = h < ng ? 1.f / den : 0.f;
            }
            for (int x = threadIdx.x; x < nvis; x += blockDim.x) {
                float sum = 0.f;
#pragma unroll
                for (int h = 0; h < G; ++h)
                    if (h < ng) sum += exp2f(scores[x * G + h] - mx[h]) * inv[h];
                const int j = x < ns ? x : x - ns + lo;
                const int b = p.bs_shift >= 0 ? j >> p.bs_shift : j / p.bs;
                float* dst = p.weights + (static_cast<size_t>(__ldg(tbl + b)) * p.kvh + kh) * p.bs + (j - b * p.bs);
                *dst = p.add && j < start ? *dst + sum : sum;
            }
        }
        return;
    }
    // ---- split keys: this CTA's partial, then the last CTA of the row joins them in order
    const size_t pr = static_cast<size_t>(blockIdx.x) * gridDim.y + blockIdx.y;
    float* part = p.part + (pr * nsplit + split) * G * (p.D + 2);
    for (int c = threadIdx.x; c < ng * nvec; c += blockDim.x) {
        const int h = c / nvec, d = 4 * (c - h * nvec);
        float mx, den, f[kWarps];
        joined_ml(h, mx, den, f);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float4 x = load4(sm + (w * G + h) * p.D + d);
            a.x = fmaf(f[w], x.x, a.x);
            a.y = fmaf(f[w], x.y, a.y);
            a.z = fmaf(f[w], x.z, a.z);
            a.w = fmaf(f[w], x.w, a.w);
        }
        float* ph = part + h * (p.D + 2);
        ph[2 + d] = a.x, ph[3 + d] = a.y, ph[4 + d] = a.z, ph[5 + d] = a.w;
        if (d == 0) {
            ph[0] = mx;
            ph[1] = den;
        }
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        sh_last = atomicAdd(p.counters + pr, 1) == nsplit - 1;
        if (sh_last) p.counters[pr] = 0;  // for the next launch
    }
    __syncthreads();
    if (!sh_last) return;
    __threadfence();
    const float* all = p.part + pr * nsplit * G * (p.D + 2);
    for (int c = threadIdx.x; c < ng * p.D; c += blockDim.x) {
        const int h = c / p.D, d = c - h * p.D;
        float mx = -INFINITY, den = 0.f, a = 0.f;
        for (int s = 0; s < nsplit; ++s) mx = fmaxf(mx, __ldcg(all + (s * G + h) * (p.D + 2)));
        for (int s = 0; s < nsplit; ++s) {
            const float* ph = all + (s * G + h) * (p.D + 2);
            const float ms = __ldcg(ph);
            const float f = ms == -INFINITY ? 0.f : exp2f(ms - mx);
            den = fmaf(f, __ldcg(ph + 1), den);
            a = fmaf(f, __ldcg(ph + 2 + d), a);
        }
        const float inv = 1.f / den;
        if constexpr (sizeof(IO) == 2) out[h * p.D + d] = __float2bfloat16_rn(a * inv);
        else out[h * p.D + d] = a * inv;
        if (p.ml != nullptr && d == 0) p.ml[static_cast<size_t>(row) * p.H + head0 + h] = make_float2(mx, inv);
    }
}

template <typename T, typename IO, int G, int NV, int LPK>
cudaError_t launch_cc_i(const CcParams& p, cudaStream_t st) {
    const int g = p.H / p.kvh;
    const dim3 grid(p.nrows, p.kvh * ((g + G - 1) / G), p.nsplit);
    const size_t smem = (static_cast<size_t>(kWarps) * G * p.D + (p.weights ? static_cast<size_t>(p.max_vis) * G : 0)) * sizeof(float);
    auto kern = cc_attn_kernel<T, IO, G, NV, LPK>;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
    }
    kern<<<grid, kWarps * 32, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T, typename IO, int G>
cudaError_t launch_cc_g(const CcParams& p, cudaStream_t st) {
    const int nvec = p.D / 4;
    if (nvec <= 8) return launch_cc_i<T, IO, G, 1, 8>(p, st);
    if (nvec <= 16) return launch_cc_i<T, IO, G, 2, 8>(p, st);
    if (nvec <= 32) return launch_cc_i<T, IO, G, 4, 8>(p, st);
    if (nvec <= 64) return launch_cc_i<T, IO, G, 4, 16>(p, st);
    return launch_cc_i<T, IO, G, 4, 32>(p, st);
}

template <typename T, typename IO>
cudaError_t launch_cc_t(const CcParams& p, cudaStream_t st) {
    const int G = cc_group(p.H / p.kvh);
    if (G == 1) return launch_cc_g<T, IO, 1>(p, st);
    if (G == 2) return launch_cc_g<T, IO, 2>(p, st);
    return launch_cc_g<T, IO, 4>(p, st);
}

}  // namespace

cudaError_t launch_cc_attention(int dtype, bool io16, const CcParams& p, cudaStream_t st) {
    if (p.nrows <= 0) return cudaSuccess;
    if (dtype == 0) return io16 ? cudaErrorInvalidValue : launch_cc_t<float, float>(p, st);
    return io16 ? launch_cc_t<__nv_bfloat16, __nv_bfloat16>(p, st) : launch_cc_t<__nv_bfloat16, float>(p, st);
}

}  // namespace pk

// Prompt chunks of bounded steps (a sliding window with sinks and / or attention weights) on the
// 5th-generation tensor cores: bf16 pools, head_dim 128.
//
// A row at position p sees the keys j <= p with j < sinks or j > p - window; keys are read through
// the block table, as in pagellm's chunks (cache/paged.py:454-463), which see the whole cache.
//
// Work item = 128/g consecutive tokens x the g query heads of one KV head = 128 query rows; two
// neighbouring items of a sequence make a pair, so that a K/V tile of 128 keys serves 256 rows. A
// pair lists the key tiles of the sinks in front of its first row's window, then those from the
// window on (PairBound): tiles that nobody sees are neither read nor computed. One CTA per (pair,
// KV head), pairs with the most keys first.

#include "pk_device.cuh"
#include "pk_internal.h"
#include "pk_tcgen05.cuh"

namespace pk {

namespace {

constexpr int kRows = 128;          // query rows of a tile (UMMA M)
constexpr int kKeys = kWideKeys;    // keys of a tile (UMMA N of S, K of P.V)
constexpr int kDim = 128;           // head dim
constexpr int kTile = kRows * kDim * 2;  // 32 KB: a Q, K or V tile, [64-dim chunk][row][64] bf16, 128-byte swizzle
constexpr uint32_t kIdescS = idesc_bf16(kKeys, false);
constexpr uint32_t kIdescO = idesc_bf16(kDim, true);

// What a pair reads: entry jt of its tile list is key tile jt, and jt + skip from jt = head on;
// lo = first key of the window of its first row.
struct PairBound {
    int head, skip, lo, ntiles;
};
__device__ __forceinline__ PairBound load_pair(const int4* p, int pair) {
    const int4 b = __ldg(p + pair);
    return PairBound{b.x, b.y, b.z, b.w};
}

// One tile of 128 keys of KV head `head` (key tile kt of a table of nblk blocks): its block ids as
// independent loads, then a copy per (block, 64-dim chunk). Entries past the table's end repeat its
// last block (masked). No multicast.
__device__ __forceinline__ void load_key_tile(const CUtensorMap* map, uint8_t* dst, uint64_t* bar, const WideParams& p,
                                              const int32_t* tbl, int nblk, int kt, int head) {
    const int per_tile = kKeys / p.bs;
    int id[kKeys / 16];
#pragma unroll
    for (int b = 0; b < kKeys / 16; ++b)
        if (b < per_tile) id[b] = __ldg(tbl + min(kt * per_tile + b, nblk - 1));
    mbar_arrive_expect_tx(bar, kTile);
#pragma unroll
    for (int b = 0; b < kKeys / 16; ++b) {
        if (b >= per_tile) break;
        const int slot0 = static_cast<int>(p.layer_slot0 + static_cast<int64_t>(id[b]) * p.bs);
        for (int c = 0; c < 2; ++c) tma_load_4d(dst + c * (kKeys * 128) + b * p.bs * 128, map, 0, slot0, head, c, bar);
    }
}

// The query tile of (item, KV head). bf16 rows come straight from q, in one box of (64 dims, g
// heads, 128/g rows) per 64-dim chunk: rows behind the item's tokens are other rows of q, or zero
// past its end, and dead to the caller. Rows given as float have been packed (launch_wide_prep).
template <bool IO16>
__device__ __forceinline__ void load_query_tile(const CUtensorMap* tmq, uint8_t* dst, uint64_t* bar, const WideParams& p,
                                                int item, int head) {
    if constexpr (IO16) {
        const int row0 = __ldg(p.tok_row + __ldg(p.w_tok0 + item));
        for (int c = 0; c < 2; ++c) tma_load_4d(dst + c * (kRows * 128), tmq, 0, head * p.g, row0, c, bar);
    } else {
        bulk_load(dst, p.qpk + static_cast<size_t>(item * p.kvh + head) * kTile, kTile, bar);
    }
}

// Barrier over `count` threads that also tells whether `pred` held in all of them.
__device__ __forceinline__ bool bar_all(int id, int count, bool pred) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.cta.red.and.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"(id), "r"(count), "r"(pred ? 1u : 0u)
        : "memory");
    return r != 0;
}

// ---------------------------------------------------------------- attention
// Warps: 0 producer (K and V rings of 2 tiles, TMA), 1 TMEM owner and MMA issuer, then 8 softmax
// warps per query tile. Per key tile: S_t = Q_t.K^T into TMEM; two threads per row, 64 scores each,
// agree on the row's maximum through shared memory and write P_t (bf16) over S_t's first 64
// columns; O_t += P_t.V with A from TMEM. Issue order P_0V, S_0(next), P_1V, S_1(next), so that one
// tile's softmax runs beside the other's MMAs. The chain softmax -> P.V -> next S of a tile is what
// bounds the kernel (P lies on S, and 512 TMEM columns hold no second S), so the softmax is spread
// over 16 warps: with 8, one thread per row, a key-tile step of 256 rows took 2.9 us at 40 % of
// the tensor and of the exponential pipe; see the measurements at launch_chunk_attention. K rings
// of 2 tiles leave room for the exchange: a slot frees a whole step before it is needed again.
constexpr int kCStages = 2;
constexpr int kCThreads = 64 + 2 * 256;
constexpr uint32_t kColO = 2 * kKeys;  // TMEM: S_0, S_1, O_0, O_1, 128 columns each
constexpr int kCOffQ = 0;
constexpr int kCOffK = kCOffQ + 2 * kTile;
constexpr int kCOffV = kCOffK + kCStages * kTile;
constexpr int kCOffRed = kCOffV + kCStages * kTile;      // [2 steps][2 tiles][2 halves][128] floats
constexpr int kCOffBar = kCOffRed + 2 * 2 * 2 * kRows * 4;
constexpr int kCSmem = kCOffBar + 256 + 1024;

template <bool IO16>
__global__ void __launch_bounds__(kCThreads, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                      const __grid_constant__ CUtensorMap tmq, const __grid_constant__ WideParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* red = reinterpret_cast<float*>(smem + kCOffRed);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + kCOffBar);
    uint64_t* kempty = kfull + kCStages;
    uint64_t* vfull = kempty + kCStages;
    uint64_t* vempty = vfull + kCStages;
    uint64_t* qfull = vempty + kCStages;  // [tile]
    uint64_t* sfull = qfull + 2;          // [tile]
    uint64_t* pfull = sfull + 2;          // [tile], one arrival per softmax warp
    uint64_t* pvdone = pfull + 2;         // [tile]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pvdone + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pair = blockIdx.x / p.kvh, head = blockIdx.x % p.kvh;
    const PairBound pb = load_pair(p.pair_bound, pair);
    const int nt = pb.ntiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kCStages; ++s) {
            mbar_init(&kfull[s], 1);
            mbar_init(&kempty[s], 1);
            mbar_init(&vfull[s], 1);
            mbar_init(&vempty[s], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&qfull[t], 1);
            mbar_init(&sfull[t], 1);
            mbar_init(&pfull[t], 8);
            mbar_init(&pvdone[t], 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t smem_base = smem_u32(smem);

    if (warp == 0) {
        if (lane == 0) {
            prefetch_tensormap(&tmk);
            prefetch_tensormap(&tmv);
            for (int t = 0; t < 2; ++t) {
                const int item = p.w_pair[2 * pair + t];
                if (item >= 0) {
                    mbar_arrive_expect_tx(&qfull[t], kTile);
                    load_query_tile<IO16>(&tmq, smem + kCOffQ + t * kTile, &qfull[t], p, item, head);
                } else {
                    mbar_arrive(&qfull[t]);  // no second item: whatever is there, its rows are dead
                }
            }
            const int seq = p.w_seq[p.w_pair[2 * pair]];
            const int32_t* tbl = p.ids + p.indptr[seq];
            const int nblk = p.indptr[seq + 1] - p.indptr[seq];
            auto real = [&](int jt) { return jt >= pb.head ? jt + pb.skip : jt; };
            // K tile n as soon as its slot is free, V tile n after K tile n: polled, not waited for
            int nk = 0, nv = 0;
            unsigned long long idle_since = global_ns();
            while (nv < nt) {
                bool progressed = false;
                if (nk < nt && mbar_test_wait(&kempty[nk % kCStages], ((nk / kCStages) & 1u) ^ 1u)) {
                    load_key_tile(&tmk, smem + kCOffK + (nk % kCStages) * kTile, &kfull[nk % kCStages], p, tbl, nblk, real(nk), head);
                    ++nk;
                    progressed = true;
                }
                if (nv < nk && mbar_test_wait(&vempty[nv % kCStages], ((nv / kCStages) & 1u) ^ 1u)) {
                    load_key_tile(&tmv, smem + kCOffV + (nv % kCStages) * kTile, &vfull[nv % kCStages], p, tbl, nblk, real(nv), head);
                    ++nv;
                    progressed = true;
                }
                if (progressed) {
                    idle_since = global_ns();
                } else if (*abort_flag || global_ns() - idle_since > kWaitLimitNs) {
                    *abort_flag = 1;
                    atomicExch(p.err, kErrTimeout);
                    break;
                }
            }
            // never leave the CTA with copies still landing in its shared memory
            for (int t = 0; t < 2; ++t) mbar_wait_bounded(&qfull[t], 0u);
            for (int t = max(0, nk - kCStages); t < nk; ++t)
                mbar_wait_bounded(&kfull[t % kCStages], static_cast<uint32_t>(t / kCStages) & 1u);
            for (int t = max(0, nv - kCStages); t < nv; ++t)
                mbar_wait_bounded(&vfull[t % kCStages], static_cast<uint32_t>(t / kCStages) & 1u);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint64_t qd0 = smem_desc(smem_base + kCOffQ, 16, 1024);
            const uint64_t kd0 = smem_desc(smem_base + kCOffK, 16, 1024);
            const uint64_t vd0 = smem_desc(smem_base + kCOffV, kKeys * 128, 1024);
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                if (ok && (!mbar_wait_bounded(bar, parity) || *abort_flag)) ok = false;
                return ok;
            };
            auto issue_s = [&](int t, int n) {
                const uint32_t kb = static_cast<uint32_t>((n % kCStages) * kTile);
#pragma unroll
                for (int kk = 0; kk < kDim / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * (kRows * 128) + (kk & 3) * 32;
                    umma_bf16(tmem + t * kKeys, qd0 + ((t * kTile + off) >> 4), kd0 + ((kb + off) >> 4), kIdescS, kk > 0 ? 1u : 0u);
                }
                umma_commit(&sfull[t]);
            };
            auto issue_pv = [&](int t, int n) {
                const uint32_t vb = static_cast<uint32_t>((n % kCStages) * kTile);
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk)
                    umma_bf16_ts(tmem + kColO + t * kDim, tmem + t * kKeys + kk * 8, vd0 + ((vb + kk * 16 * 128) >> 4), kIdescO,
                                 (n > 0 || kk > 0) ? 1u : 0u);
                umma_commit(&pvdone[t]);
            };
            auto ph = [](int n) { return static_cast<uint32_t>(n / kCStages) & 1u; };
            if (wait(&kfull[0], 0u) && wait(&qfull[0], 0u)) {
                tc_fence_after();
                issue_s(0, 0);
                if (wait(&qfull[1], 0u)) {
                    tc_fence_after();
                    issue_s(1, 0);
                    umma_commit(&kempty[0]);
                }
            }
            for (int n = 0; n < nt && ok; ++n) {
                const bool more = n + 1 < nt;
                if (!wait(&vfull[n % kCStages], ph(n)) || !wait(&pfull[0], static_cast<uint32_t>(n & 1))) break;
                tc_fence_after();
                issue_pv(0, n);
                if (more) {
                    if (!wait(&kfull[(n + 1) % kCStages], ph(n + 1))) break;
                    tc_fence_after();
                    issue_s(0, n + 1);
                }
                if (!wait(&pfull[1], static_cast<uint32_t>(n & 1))) break;
                tc_fence_after();
                issue_pv(1, n);
                umma_commit(&vempty[n % kCStages]);
                if (more) {
                    issue_s(1, n + 1);
                    umma_commit(&kempty[(n + 1) % kCStages]);
                }
            }
            if (!ok) {
                *abort_flag = 1;
                atomicExch(p.err, kErrTimeout);
            }
        }
    } else {
        const int tile = (warp - 2) >> 3, half = ((warp - 2) >> 2) & 1;  // keys [64 * half, 64 * half + 64) of each tile
        const int q4 = warp & 3;                                         // TMEM lanes 32 * q4 .. + 31
        const int r = 32 * q4 + lane;
        const int bar = 1 + tile;
        const uint32_t trow = tmem + (static_cast<uint32_t>(32 * q4) << 16);
        const uint32_t tS = trow + tile * kKeys;
        const uint32_t tO = trow + kColO + tile * kDim;
        const int item = p.w_pair[2 * pair + tile];
        const int ntok = item >= 0 ? p.w_ntok[item] : 0;
        const int tok0 = item >= 0 ? p.w_tok0[item] : 0;
        const int t_row = r / p.g;
        const bool live = t_row < ntok;
        const int kv_end = p.pair_kend[pair];
        const int last_tile = (kv_end - 1) / kKeys;
        const int qlim = live ? p.tok_pos[tok0] + t_row : -1;  // last key of the row; consecutive tokens
        const int qlo = live ? qlim - p.window : -1;           // keys up to it and not among the sinks are past the window
        const size_t oidx = static_cast<size_t>(p.tok_row[tok0] + (live ? t_row : 0)) * p.H + head * p.g + r % p.g;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int n = 0; n < nt; ++n) {
            const int rt = n >= pb.head ? n + pb.skip : n;
            const int kb = rt * kKeys + 64 * half;  // this thread's first key
            // a timeout is agreed on at the barrier below, so that all of the tile's warps leave together
            bool got = ok && mbar_wait_bounded(&sfull[tile], static_cast<uint32_t>(n & 1)) && !*abort_flag;
            got = __all_sync(0xffffffffu, got);
            tc_fence_after();
            float sv[64];
            tmem_ld32(tS + half * 64, sv);
            tmem_ld32(tS + half * 64 + 32, sv + 32);
            tmem_wait_ld();
            if (kb + 63 > qlim || (kb <= qlo && kb + 63 >= p.sinks)) {
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (kb + i > qlim || (kb + i <= qlo && kb + i >= p.sinks)) sv[i] = -INFINITY;
            }
            float mx4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                mx4[k] = sv[k];
#pragma unroll
                for (int i = k + 4; i < 64; i += 4) mx4[k] = fmaxf(mx4[k], sv[i]);
            }
            float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            float* rx = red + ((n & 1) * 2 + tile) * 2 * kRows + r;
            rx[half * kRows] = mx;
            // both halves' scores are read and their maxima known (also: S may be overwritten by P)
            tc_fence_before();
            ok = bar_all(bar, 256, got);
            if (!ok) break;
            tc_fence_after();
            mx = fmaxf(mx, rx[(half ^ 1) * kRows]) * p.sscale;
            // Lazy rescale: the base of earlier tiles stays unless this tile's maximum exceeds it by
            // more than 8 (P stays <= 2^8 in bf16, l and O in fp32).
            const float mnew = (m == -INFINITY || mx > m + 8.f) ? mx : m;
            const float base = mnew == -INFINITY ? 0.f : mnew;
            const float corr = m == -INFINITY ? 0.f : ex2_approx(m - base);
            float sum4[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t pk[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float a = ex2_approx(fmaf(sv[2 * i], p.sscale, -base));
                const float b = ex2_approx(fmaf(sv[2 * i + 1], p.sscale, -base));
                sum4[i & 3] += a + b;
                pk[i] = pack_bf16(a, b);
            }
            tmem_st32u(tS + half * 32, pk);
            tmem_wait_st();
            l = l * corr + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
            m = mnew;
            // O to the new base before P.V of this tile may start; it holds the previous tile's P.V,
            // which was issued before this tile's S (the wait confirms it). Each half takes 64 dims.
            if (n > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pvdone[tile], static_cast<uint32_t>((n - 1) & 1)));
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    float o[32];
                    tmem_ld32(tO + half * 64 + c * 32, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= corr;
                    tmem_st32(tO + half * 64 + c * 32, o);
                }
                tmem_wait_st();
            }
            // V rows that no row of the pair sees - past the context in the last tile, or between the
            // sinks and the first row's window - are zeroed so that P = 0 meets 0 (tile 0's P.V is
            // issued first, so tile 1's sees the zeros too).
            const int k0 = rt * kKeys;
            const bool tail = rt == last_tile && kv_end < k0 + kKeys;
            const int za = max(0, p.sinks - k0), zb = min(kKeys, pb.lo - k0);
            if (tile == 0 && (tail || za < zb)) {
                const int s = n % kCStages;
                const bool landed = mbar_wait_bounded(&vfull[s], static_cast<uint32_t>(n / kCStages) & 1u);
                ok = __all_sync(0xffffffffu, landed) && ok;
                uint8_t* vd = smem + kCOffV + s * kTile;
                auto zero_rows = [&](int first, int end) {
                    for (int x = threadIdx.x - 64; x < (end - first) * 16; x += 256) {
                        const int key = first + x / 16;
                        *reinterpret_cast<uint4*>(vd + ((x / 8) & 1) * (kKeys * 128) + sw128(key, x & 7)) = make_uint4(0, 0, 0, 0);
                    }
                };
                if (tail) zero_rows(kv_end - k0, kKeys);
                if (za < zb) zero_rows(za, zb);
                fence_proxy_async_smem();  // the zeros (generic writes) before the MMA reads them
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pfull[tile]);
        }
        // ---- epilogue: O / l. Rows leave TMEM one per thread, 32 columns at a time, and go to global
        // memory through 4 KB of the tile's Q buffer (its S MMAs are done), so that a store covers
        // pieces of 4 rows; float4 slot i of staging row r sits at i ^ (r & 7): conflict-free.
        const bool done = ok && mbar_wait_bounded(&pvdone[tile], static_cast<uint32_t>((nt - 1) & 1)) && !*abort_flag;
        float* rx = red + ((nt & 1) * 2 + tile) * 2 * kRows + r;
        rx[half * kRows] = l;
        ok = bar_all(bar, 256, __all_sync(0xffffffffu, done));
        if (ok) {
            tc_fence_after();
            const float wo = live ? 1.f / (rx[0] + rx[kRows]) : 0.f;
            if (half == 0 && p.ml != nullptr && item >= 0)
                p.ml[(static_cast<size_t>(item) * p.kvh + head) * kRows + r] = live ? make_float2(m, wo) : make_float2(0.f, 0.f);
            float* stg = reinterpret_cast<float*>(smem + kCOffQ + tile * kTile + (half * 4 + q4) * 4096);
            auto stg4 = [&](int row, int i) { return reinterpret_cast<float4*>(stg + row * 32 + 4 * (i ^ (row & 7))); };
            const int sub = lane >> 3, cq = lane & 7;  // transposed: row 4 * k + sub, 4 columns at 4 * cq
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                float o[32];
                tmem_ld32(tO + half * 64 + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *stg4(lane, i) = make_float4(o[4 * i] * wo, o[4 * i + 1] * wo, o[4 * i + 2] * wo, o[4 * i + 3] * wo);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int row = 4 * k + sub;
                    const unsigned long long oi = __shfl_sync(0xffffffffu, static_cast<unsigned long long>(oidx), row);
                    const bool lv = __shfl_sync(0xffffffffu, live ? 1 : 0, row) != 0;
                    const float4 x = *stg4(row, cq);
                    const size_t off = static_cast<size_t>(oi) * kDim + half * 64 + c * 32 + 4 * cq;
                    if (!lv) continue;
                    if constexpr (IO16)
                        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + off) =
                            make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
                    else
                        *reinterpret_cast<float4*>(p.out + off) = x;
                }
                __syncwarp();
            }
        } else {
            *abort_flag = 1;
            if (lane == 0) atomicExch(p.err, kErrTimeout);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------- weights
// Attention weight of every key of a 128-key tile: a[j] = sum over query rows c of
// 2^(s[j, c] - m[c]) / l[c], with the row statistics of chunk_attn_kernel. The score tile is computed
// transposed, S^T = K . Q^T with keys as the MMA rows, so that a thread owns one key and sums its
// row alone: no reduction across threads, and a fixed order. A CTA takes one piece: a key tile of
// one KV head against consecutive query items [i0, i1); the pieces of a tile are added in order by
// weight_pieces_kernel. Q tiles stream through a 2-slot ring (their statistics through a 4-slot
// one: slot x + 4 is filled after the MMA of x + 2, which waited for the epilogue of x) and S^T
// through two TMEM buffers; at 102 KB of shared memory and 256 TMEM columns two CTAs share an SM,
// so that one's exponentials run beside the other's loads and MMAs. Bound: one exponential per
// score, 16 per clock and SM, twice the MMA's time.
constexpr int kGThreads = 192;  // producer, MMA issuer, 4 epilogue warps
constexpr int kGOffK = 0;
constexpr int kGOffQ = kGOffK + kTile;
constexpr int kGOffStat = kGOffQ + 2 * kTile;               // [4][128] {m, 1/l}
constexpr int kGOffBar = kGOffStat + 4 * kRows * 8;
constexpr int kGSmem = kGOffBar + 256 + 1024;

template <bool IO16>
__global__ void __launch_bounds__(kGThreads, 2)
    chunk_weight_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmq,
                        const __grid_constant__ WideParams p, const int4* __restrict__ pieces, float* __restrict__ part) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const float2* stat = reinterpret_cast<const float2*>(smem + kGOffStat);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + kGOffBar);
    uint64_t* qfull = kfull + 1;    // [2]
    uint64_t* qempty = qfull + 2;   // [2]
    uint64_t* sfull = qempty + 2;   // [2]
    uint64_t* sempty = sfull + 2;   // [2]
    uint64_t* stfull = sempty + 2;  // [4]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stfull + 4);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int4 pc = __ldg(pieces + blockIdx.x);
    const int seq = pc.x, kt = pc.y, i0 = pc.z, n = pc.w - pc.z;
    const int head = blockIdx.y;

    if (threadIdx.x == 0) {
        mbar_init(kfull, 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&qfull[b], 1);
            mbar_init(&qempty[b], 1);
            mbar_init(&sfull[b], 1);
            mbar_init(&sempty[b], 4);
        }
        for (int b = 0; b < 4; ++b) mbar_init(&stfull[b], 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 2 * kKeys);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t smem_base = smem_u32(smem);

    if (warp == 0) {
        if (lane == 0) {
            prefetch_tensormap(&tmk);
            load_key_tile(&tmk, smem + kGOffK, kfull, p, p.ids + p.indptr[seq], p.indptr[seq + 1] - p.indptr[seq], kt, head);
            int issued = 0;
            for (int x = 0; x < n; ++x) {
                if (!mbar_wait_bounded(&qempty[x & 1], ((x >> 1) & 1u) ^ 1u) || *abort_flag) {
                    *abort_flag = 1;
                    atomicExch(p.err, kErrTimeout);
                    break;
                }
                mbar_arrive_expect_tx(&stfull[x & 3], kRows * 8);
                bulk_load(smem + kGOffStat + (x & 3) * kRows * 8, p.ml + (static_cast<size_t>(i0 + x) * p.kvh + head) * kRows,
                          kRows * 8, &stfull[x & 3]);
                mbar_arrive_expect_tx(&qfull[x & 1], kTile);
                load_query_tile<IO16>(&tmq, smem + kGOffQ + (x & 1) * kTile, &qfull[x & 1], p, i0 + x, head);
                issued = x + 1;
            }
            // never leave the CTA with copies still landing in its shared memory
            mbar_wait_bounded(kfull, 0u);
            for (int x = max(0, issued - 2); x < issued; ++x) mbar_wait_bounded(&qfull[x & 1], (x >> 1) & 1u);
            for (int x = max(0, issued - 4); x < issued; ++x) mbar_wait_bounded(&stfull[x & 3], (x >> 2) & 1u);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint64_t kd0 = smem_desc(smem_base + kGOffK, 16, 1024);
            const uint64_t qd0 = smem_desc(smem_base + kGOffQ, 16, 1024);
            bool ok = mbar_wait_bounded(kfull, 0u);
            for (int x = 0; x < n && ok; ++x) {
                const int b = x & 1;
                ok = mbar_wait_bounded(&qfull[b], (x >> 1) & 1u) && mbar_wait_bounded(&sempty[b], ((x >> 1) & 1u) ^ 1u) &&
                     !*abort_flag;
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < kDim / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * (kRows * 128) + (kk & 3) * 32;
                    umma_bf16(tmem + b * kKeys, kd0 + (off >> 4), qd0 + ((b * kTile + off) >> 4), kIdescS, kk > 0 ? 1u : 0u);
                }
                umma_commit(&sfull[b]);
                umma_commit(&qempty[b]);
            }
            if (!ok) {
                *abort_flag = 1;
                atomicExch(p.err, kErrTimeout);
            }
        }
    } else {
        const int q4 = warp & 3;  // TMEM lanes 32 * q4 .. + 31
        const int key = 32 * q4 + lane;
        const int j = kt * kKeys + key;
        const uint32_t trow = tmem + (static_cast<uint32_t>(32 * q4) << 16);
        // items hold tpt = 128 / g consecutive tokens, all but a sequence's last one exactly
        const int tpt = kRows / p.g;
        const int pos_i0 = p.tok_pos[p.w_tok0[i0]];
        const int ntok_last = p.w_ntok[i0 + n - 1];
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        bool ok = true;
        for (int x = 0; x < n && ok; ++x) {
            const int b = x & 1;
            const bool got = mbar_wait_bounded(&stfull[x & 3], (x >> 2) & 1u) && mbar_wait_bounded(&sfull[b], (x >> 1) & 1u);
            ok = __all_sync(0xffffffffu, got && !*abort_flag);
            if (!ok) break;
            tc_fence_after();
            const float2* st = stat + (x & 3) * kRows;
            // token t of the item, at position pos0 + t, sees key j for t in [j - pos0, j - pos0 + window)
            // (without the upper limit when j is a sink); its columns are g * t .. g * t + g - 1
            const int pos0 = pos_i0 + x * tpt, ntok = x == n - 1 ? ntok_last : tpt;
            const int rel = j - pos0;
            const int t_lo = max(0, rel);
            const int t_hi = j < p.sinks || rel > INT32_MAX - p.window ? ntok : min(ntok, rel + p.window);
            const int c_lo = t_lo * p.g, c_hi = t_hi * p.g;
            const bool whole = __all_sync(0xffffffffu, c_lo == 0 && c_hi == kRows);
#pragma unroll 1
            for (int c0 = 0; c0 < kRows; c0 += 32) {
                float sv[32];
                tmem_ld32(trow + b * kKeys + c0, sv);
                tmem_wait_ld();
                const float4* mlp = reinterpret_cast<const float4*>(st + c0);
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float4 a = mlp[i];
                        sum[(2 * i) & 3] = fmaf(ex2_approx(fmaf(sv[2 * i], p.sscale, -a.x)), a.y, sum[(2 * i) & 3]);
                        sum[(2 * i + 1) & 3] = fmaf(ex2_approx(fmaf(sv[2 * i + 1], p.sscale, -a.z)), a.w, sum[(2 * i + 1) & 3]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 a = st[c0 + i];
                        const float e = c0 + i >= c_lo && c0 + i < c_hi ? ex2_approx(fmaf(sv[i], p.sscale, -a.x)) : 0.f;
                        sum[i & 3] = fmaf(e, a.y, sum[i & 3]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sempty[b]);
        }
        if (ok) {
            part[(static_cast<size_t>(blockIdx.x) * p.kvh + head) * kKeys + key] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        } else {
            *abort_flag = 1;
            if (lane == 0) atomicExch(p.err, kErrTimeout);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * kKeys);
    }
}

// Adds up a touched block's pieces, in order, into its weights: one thread per (block, KV head,
// token). t_piece: first piece of the block's key tile and how many.
__global__ void __launch_bounds__(256) weight_pieces_kernel(const WideParams p, const WeightParams w,
                                                            const int32_t* __restrict__ starts,
                                                            const int32_t* __restrict__ offsets,
                                                            const int2* __restrict__ t_piece, const float* __restrict__ part) {
    const int64_t x = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
    const int64_t e64 = x / (p.kvh * p.bs);
    if (e64 >= w.ntouched) return;
    const int e = static_cast<int>(e64);
    const int hx = static_cast<int>(x - e64 * (p.kvh * p.bs));
    const int h = hx / p.bs, t = hx - h * p.bs;
    const int seq = w.t_seq[e], lb = w.t_blk[e];
    const int start = starts[seq], ctx = start + offsets[seq + 1] - offsets[seq];
    const int j = lb * p.bs + t;
    if (j >= ctx || (j >= p.sinks && j <= start - p.window)) return;
    const int2 pr = t_piece[e];
    float sum = 0.f;
#pragma unroll 4
    for (int i = 0; i < pr.y; ++i) sum += __ldcg(part + (static_cast<size_t>(pr.x + i) * p.kvh + h) * kKeys + j % kKeys);
    float* dst = w.weights + (static_cast<size_t>(p.ids[p.indptr[seq] + lb]) * p.kvh + h) * p.bs + t;
    *dst = w.add && j < start ? *dst + sum : sum;
}

}  // namespace

size_t chunk_smem_bytes() { return kCSmem; }

cudaError_t launch_chunk_attention(const CUtensorMap* tmk1, const CUtensorMap* tmv1, const CUtensorMap* tmq,
                                   const WideParams& p, int npairs, cudaStream_t st) {
    if (npairs <= 0) return cudaSuccess;
    auto kern = p.io16 ? chunk_attn_kernel<true> : chunk_attn_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kCSmem);
    if (e != cudaSuccess) return e;
    kern<<<npairs * p.kvh, kCThreads, kCSmem, st>>>(*tmk1, *tmv1, *tmq, p);
    return cudaGetLastError();
}

cudaError_t launch_chunk_weights(const CUtensorMap* tmk1, const CUtensorMap* tmq, const WideParams& p, const int4* pieces,
                                 int npieces, float* part, const WeightParams& w, const int32_t* starts,
                                 const int32_t* offsets, const int2* t_piece, cudaStream_t st) {
    if (npieces <= 0 || w.ntouched <= 0) return cudaSuccess;
    auto kern = p.io16 ? chunk_weight_kernel<true> : chunk_weight_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGSmem);
    if (e != cudaSuccess) return e;
    kern<<<dim3(npieces, p.kvh), kGThreads, kGSmem, st>>>(*tmk1, *tmq, p, pieces, part);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    const int64_t blocks = (static_cast<int64_t>(w.ntouched) * p.kvh * p.bs + 255) / 256;
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    weight_pieces_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(p, w, starts, offsets, t_piece, part);
    return cudaGetLastError();
}

}  // namespace pk

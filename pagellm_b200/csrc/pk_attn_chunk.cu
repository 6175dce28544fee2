// Prompt chunks of bounded steps (a sliding window with sinks and / or attention weights) on the
// 5th-generation tensor cores: bf16 pools, head_dim 128.
//
// A row at position p sees the keys j <= p with j < sinks or j > p - window; keys are read through
// the block table, as in pagellm's chunks (cache/paged.py:454-463), which see the whole cache.
//
// Work item = 128/g consecutive tokens x the g query heads of one KV head = 128 query rows; two
// neighbouring items of a sequence make a pair, so that a K/V tile of 64 keys serves 256 rows. A
// pair lists the key tiles of the sinks in front of its first row's window, then those from the
// window on: tiles that nobody sees are neither read nor computed. The (pair, KV head)s are dealt to
// one CTA per SM, whole where that balances, else cut (build_wide_schedule).

#include "pk_device.cuh"
#include "pk_internal.h"
#include "pk_tcgen05.cuh"

namespace pk {

namespace {

constexpr int kRows = 128;          // query rows of a tile (UMMA M)
constexpr int kKeys = kWideKeys;    // keys of a tile of chunk_weight_kernel
constexpr int kDim = 128;           // head dim
constexpr int kTile = kRows * kDim * 2;  // 32 KB: 128 query rows or keys, [64-dim chunk][row][64] bf16, 128-byte swizzle
constexpr uint32_t kIdescS = idesc_bf16(kKeys, false);
constexpr uint32_t kIdescO = idesc_bf16(kDim, true);

// A CTA's work item: entries [t0, t1) of a pair's tile list for one KV head. Entry jt is key tile
// jt, and jt + skip from jt = head on; lo = first key of the window of the pair's first row. slot:
// where the partial goes when the list is cut between CTAs, or -1.
struct Segment {
    int pair, kvhead, t0, t1, slot;
    int head, skip, lo;
    __device__ __forceinline__ int tile(int jt) const { return jt >= head ? jt + skip : jt; }
};
__device__ __forceinline__ Segment load_segment(const WideParams& p, int i) {
    const int32_t* e = p.seg + 6 * i;
    Segment s{e[0], e[1], e[2], e[3], e[4], 0, 0, 0};
    const int4 b = __ldg(p.pair_bound + s.pair);
    s.head = b.x;
    s.skip = b.y;
    s.lo = b.z;
    return s;
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

// ---------------------------------------------------------------- attention
// One CTA per SM walks a list of segments. Warps: 0 and 1 producers (rings of 64-key K and V tiles and
// the next segment's queries, TMA), 2 and 3 MMA issuers of query tile 0 and 1 (2 owns the TMEM), then 4
// softmax warps per query tile, thread = row. Per tile of 64 keys: S_t = Q_t.K^T (M=128 N=64 K=128)
// into TMEM; a row's 64 scores are read and S_t is given back at once, so that the next S_t is
// computed while this one's exponentials run; P_t (bf16) goes to columns of its own and
// O_t += P_t.V (M=128 N=128 K=64, A from TMEM). At the end of a segment the next one's queries, keys
// and first S_t are under way while O_t is written out.
// Why 64 keys: with 128, S, P and O of two query tiles do not fit the 512 TMEM columns side by side,
// P has to lie on S, and each tile runs as one chain softmax -> P.V -> next S. Traced on the B200,
// clocks per 128 keys of 256 rows: 4400 in that form (2250 softmax, 340 hand-over, 690 + 750 the two
// products, 250 back), with the exponential unit (2048 at least) and the tensor cores (2140) each half
// idle; twice the softmax warps, faster copies or two issuers did not move it. Here 3800, bound by the
// products: an M=128 N=64 one costs 51 clocks against an N=128 one's 67, because its A operand fills
// the shared-memory port. 2048 rows of 32 heads over a window of 4096: 165 us (tensor cores 51 % active,
// exponential unit 52 %; 82 at the cuBLAS rate). A list of segments per CTA, because a CTA's start and end
// (TMEM, the first queries and keys, the output) take 14 us, which one per (pair, KV head) paid each time.
constexpr int kTurnAfter = 16;  // pairs of exponentials after which the other tile may start its own (4 to 24: within 1 %)
constexpr int kCKeys = kChunkKeys;  // 64
constexpr int kCKvTile = kCKeys * kDim * 2;  // 16 KB, [64-dim chunk][key][64]
constexpr int kCStages = 4;
constexpr int kCThreads = 32 * 4 + 2 * 128;
constexpr uint32_t kColP = 2 * kCKeys;  // TMEM: S_0, S_1 (64 columns each), P_0, P_1 (32 each), O_0, O_1
constexpr uint32_t kColO = 256;
constexpr uint32_t kIdescS64 = idesc_bf16(kCKeys, false);
constexpr int kCOffQ = 0;
constexpr int kCOffK = kCOffQ + 2 * kTile;
constexpr int kCOffV = kCOffK + kCStages * kCKvTile;
constexpr int kCOffStage = kCOffV + kCStages * kCKvTile;  // 4 KB per softmax warp for O on its way out
constexpr int kCOffBar = kCOffStage + 8 * 4096;
constexpr int kCSmem = kCOffBar + 384 + 1024;

template <bool IO16>
__global__ void __launch_bounds__(kCThreads, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                      const __grid_constant__ CUtensorMap tmq, const __grid_constant__ WideParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + kCOffBar);
    uint64_t* kempty = kfull + kCStages;  // two arrivals: S of both query tiles
    uint64_t* vfull = kempty + kCStages;
    uint64_t* vempty = vfull + kCStages;  // two arrivals: P.V of both
    uint64_t* qfull = vempty + kCStages;  // [tile], per segment
    uint64_t* qempty = qfull + 2;         // [tile], per segment: its S are done with Q
    uint64_t* sfull = qempty + 2;         // [tile], per key tile, as the next three
    uint64_t* sfree = sfull + 2;          // [tile], one arrival per softmax warp
    uint64_t* pfull = sfree + 2;          // [tile], one arrival per softmax warp
    uint64_t* pvdone = pfull + 2;         // [tile]
    uint64_t* ofree = pvdone + 2;         // [tile], per segment, one arrival per softmax warp: O has been read
    uint64_t* turn = ofree + 2;           // [tile][quadrant]: the tile's warp may take its exponentials
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(turn + 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int s_begin = p.cta_seg[blockIdx.x], s_end = p.cta_seg[blockIdx.x + 1];

    if (threadIdx.x == 0) {
        for (int s = 0; s < kCStages; ++s) {
            mbar_init(&kfull[s], 1);
            mbar_init(&kempty[s], 2);
            mbar_init(&vfull[s], 1);
            mbar_init(&vempty[s], 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&qfull[t], 1);
            mbar_init(&qempty[t], 1);
            mbar_init(&sfull[t], 1);
            mbar_init(&sfree[t], 4);
            mbar_init(&pfull[t], 4);
            mbar_init(&pvdone[t], 1);
            mbar_init(&ofree[t], 4);
            for (int q = 0; q < 4; ++q) mbar_init(&turn[4 * t + q], 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t smem_base = smem_u32(smem);
    auto ph = [](int n) { return static_cast<uint32_t>(n / kCStages) & 1u; };

    if (warp <= 1) {
        // ---- producers: warp 0 K tiles and queries, warp 1 V tiles. Lane b knows the first slot of part
        // b of the next tile (a block, or 64 keys of a larger one) before the ring has room for it, and
        // one lane issues the tile's copies: from 16 lanes of one warp, K and V together, they took 1300
        // clocks a tile and were what the whole kernel waited for.
        const bool is_v = warp == 1;
        const int part = min(p.bs, kCKeys), parts = kCKeys / part;  // at most 4
        const CUtensorMap* map = is_v ? &tmv : &tmk;
        uint8_t* ring = smem + (is_v ? kCOffV : kCOffK);
        uint64_t* full = is_v ? vfull : kfull;
        uint64_t* empty = is_v ? vempty : kempty;
        if (lane == 0) prefetch_tensormap(map);
        bool ok = true;
        int n = 0, nq = 0;
        for (int si = s_begin; si < s_end && ok; ++si) {
            const Segment sg = load_segment(p, si);
            const int seq = p.w_seq[p.w_pair[2 * sg.pair]];
            const int32_t* tbl = p.ids + p.indptr[seq];
            const int nblk = p.indptr[seq + 1] - p.indptr[seq];
            // past the table's end: its last block, masked
            auto slot_of = [&](int jt) {
                const int key = sg.tile(jt) * kCKeys + (lane & 3) * part;
                const int blk = min(key >> p.bs_shift, nblk - 1);
                return static_cast<int>(p.layer_slot0 + static_cast<int64_t>(__ldg(tbl + blk)) * p.bs + (key & (p.bs - 1)));
            };
            int slot = slot_of(sg.t0);
            for (int jt = sg.t0; jt < sg.t1; ++jt, ++n) {
                ok = __all_sync(0xffffffffu, mbar_wait_fast(&empty[n % kCStages], ph(n) ^ 1u));
                if (!ok) break;
                int part_slot[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) part_slot[b] = __shfl_sync(0xffffffffu, slot, b);
                uint8_t* dst = ring + (n % kCStages) * kCKvTile;
                uint64_t* bar = &full[n % kCStages];
                if (elect_one()) {
                    mbar_arrive_expect_tx(bar, kCKvTile);
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (b < parts) {
                            tma_load_4d(dst + b * part * 128, map, 0, part_slot[b], sg.kvhead, 0, bar);
                            tma_load_4d(dst + b * part * 128 + kCKeys * 128, map, 0, part_slot[b], sg.kvhead, 1, bar);
                        }
                }
                __syncwarp();
                if (jt + 1 < sg.t1) slot = slot_of(jt + 1);
                if (!is_v && jt == sg.t0) {
                    // the segment's queries, once the last one's S are done with theirs
                    if (nq > 0) {
                        const uint32_t par = static_cast<uint32_t>((nq - 1) & 1);
                        ok = __all_sync(0xffffffffu, mbar_wait_fast(&qempty[0], par, &qempty[1], par));
                        if (!ok) break;
                    }
                    if (lane == 0) {
                        for (int t = 0; t < 2; ++t) {
                            const int item = p.w_pair[2 * sg.pair + t];
                            if (item >= 0) {
                                mbar_arrive_expect_tx(&qfull[t], kTile);
                                load_query_tile<IO16>(&tmq, smem + kCOffQ + t * kTile, &qfull[t], p, item, sg.kvhead);
                            } else {
                                mbar_arrive(&qfull[t]);  // no second item: whatever is there, its rows are dead
                            }
                        }
                    }
                    __syncwarp();
                    ++nq;
                }
            }
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            atomicExch(p.err, kErrTimeout);
        }
        // never leave the CTA with copies still landing in its shared memory
        if (lane == 0) {
            if (nq > 0)
                for (int t = 0; t < 2; ++t) mbar_wait_bounded(&qfull[t], static_cast<uint32_t>((nq - 1) & 1));
            for (int t = max(0, n - kCStages); t < n; ++t)
                mbar_wait_bounded(&full[t % kCStages], static_cast<uint32_t>(t / kCStages) & 1u);
        }
    } else if (warp <= 3) {
        // ---- one issuer per query tile: S(n + 1) once the scores of n have been read, P.V(n) once P is
        // there; n counts the CTA's key tiles
        const int t = warp - 2;
        const uint64_t qd0 = smem_desc(smem_base + kCOffQ + t * kTile, 16, 1024);
        const uint64_t kd0 = smem_desc(smem_base + kCOffK, 16, 1024);
        const uint64_t vd0 = smem_desc(smem_base + kCOffV, kCKeys * 128, 1024);
        const uint32_t tS = tmem + t * kCKeys, tP = tmem + kColP + t * (kCKeys / 2), tO = tmem + kColO + t * kDim;
        bool ok = true;
        auto wait = [&](uint64_t* bar_a, uint32_t parity_a, uint64_t* bar_b, uint32_t parity_b) {
            ok = __all_sync(0xffffffffu, mbar_wait_fast(bar_a, parity_a, bar_b, parity_b));
            return ok;
        };
        auto issue_s = [&](int n, bool last) {  // last: the segment's, after which Q is free
            tc_fence_after();
            const uint64_t kd = kd0 + ((n % kCStages) * (kCKvTile >> 4));
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kDim / 16; ++kk)
                    umma_bf16(tS, qd0 + (((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4),
                              kd + (((kk >> 2) * (kCKeys * 128) + (kk & 3) * 32) >> 4), kIdescS64, kk > 0 ? 1u : 0u);
                umma_commit(&sfull[t]);
                umma_commit(&kempty[n % kCStages]);
                if (last) umma_commit(&qempty[t]);
            }
            __syncwarp();
        };
        int n = 0;
        for (int si = s_begin; si < s_end && ok; ++si) {
            const Segment sg = load_segment(p, si);
            const int k = si - s_begin, nt = sg.t1 - sg.t0;
            if (!wait(&qfull[t], static_cast<uint32_t>(k & 1), &kfull[n % kCStages], ph(n))) break;
            if (n > 0 && !wait(&sfree[t], static_cast<uint32_t>((n - 1) & 1), &sfree[t], static_cast<uint32_t>((n - 1) & 1))) break;
            issue_s(n, nt == 1);
            for (int i = 0; i < nt; ++i, ++n) {
                if (i + 1 < nt) {
                    if (!wait(&kfull[(n + 1) % kCStages], ph(n + 1), &sfree[t], static_cast<uint32_t>(n & 1))) break;
                    issue_s(n + 1, i + 2 == nt);
                }
                if (!wait(&vfull[n % kCStages], ph(n), &pfull[t], static_cast<uint32_t>(n & 1))) break;
                // the first P.V of a segment overwrites the last one's O
                if (i == 0 && k > 0 && !wait(&ofree[t], static_cast<uint32_t>((k - 1) & 1), &ofree[t], static_cast<uint32_t>((k - 1) & 1)))
                    break;
                tc_fence_after();
                const uint64_t vd = vd0 + ((n % kCStages) * (kCKvTile >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kCKeys / 16; ++kk)
                        umma_bf16_ts(tO, tP + kk * 8, vd + ((kk * 16 * 128) >> 4), kIdescO, (i > 0 || kk > 0) ? 1u : 0u);
                    umma_commit(&pvdone[t]);
                    umma_commit(&vempty[n % kCStages]);
                }
                __syncwarp();
            }
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            atomicExch(p.err, kErrTimeout);
        }
    } else {
        const int tile = (warp - 4) >> 2;
        const int q4 = warp & 3;  // TMEM lanes 32 * q4 .. + 31
        const int r = 32 * q4 + lane;
        const uint32_t trow = tmem + (static_cast<uint32_t>(32 * q4) << 16);
        const uint32_t tS = trow + tile * kCKeys;
        const uint32_t tP = trow + kColP + tile * (kCKeys / 2);
        const uint32_t tO = trow + kColO + tile * kDim;
        const uint64_t scale2 = pack_f32x2(p.sscale, p.sscale);
        float* stg = reinterpret_cast<float*>(smem + kCOffStage + (tile * 4 + q4) * 4096);
        auto stg4 = [&](int row, int i) { return reinterpret_cast<float4*>(stg + row * 32 + 4 * (i ^ (row & 7))); };
        const int t_row = r / p.g;
        bool ok = true;
        int n = 0;  // the CTA's key tiles so far
        for (int si = s_begin; si < s_end && ok; ++si) {
            const Segment sg = load_segment(p, si);
            const int item = p.w_pair[2 * sg.pair + tile];
            const int ntok = item >= 0 ? p.w_ntok[item] : 0;
            const int tok0 = item >= 0 ? p.w_tok0[item] : 0;
            const bool live = t_row < ntok;
            const int kv_end = p.pair_kend[sg.pair];
            const int last_tile = (kv_end - 1) / kCKeys;
            const int qlim = live ? p.tok_pos[tok0] + t_row : -1;  // last key of the row; consecutive tokens
            const int qlo = live ? qlim - p.window : -1;  // keys up to it and not among the sinks are past the window
            const size_t oidx = static_cast<size_t>(p.tok_row[tok0] + (live ? t_row : 0)) * p.H + sg.kvhead * p.g + r % p.g;
            float m = -INFINITY, l = 0.f;
            for (int jt = sg.t0; jt < sg.t1; ++jt, ++n) {
                const bool first = jt == sg.t0;
                const int k0 = sg.tile(jt) * kCKeys;
                ok = __all_sync(0xffffffffu, mbar_wait_fast(&sfull[tile], static_cast<uint32_t>(n & 1)));
                if (!ok) break;
                tc_fence_after();
                float sv[kCKeys];
                tmem_ld32(tS, sv);
                tmem_ld32(tS + 32, sv + 32);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sfree[tile]);
                if (k0 + kCKeys - 1 > qlim || (k0 <= qlo && k0 + kCKeys > p.sinks)) {
#pragma unroll
                    for (int i = 0; i < kCKeys; ++i)
                        if (k0 + i > qlim || (k0 + i <= qlo && k0 + i >= p.sinks)) sv[i] = -INFINITY;
                }
                float mx8[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    mx8[k] = sv[k];
#pragma unroll
                    for (int i = k + 8; i < kCKeys; i += 8) mx8[k] = fmaxf(mx8[k], sv[i]);
                }
                const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                                       fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]))) * p.sscale;
                // Lazy rescale: the base of earlier tiles stays unless this tile's maximum exceeds it by
                // more than 8 (P stays <= 2^8). P enters the second product in bf16, V's type (half a step,
                // 2^-8 at most, of each probability); l and O are fp32.
                const float mnew = (m == -INFINITY || mx > m + 8.f) ? mx : m;
                const float base = mnew == -INFINITY ? 0.f : mnew;
                const float corr = m == -INFINITY ? 0.f : ex2_approx(m - base);
                const uint64_t base2 = pack_f32x2(-base, -base);
                // The two tiles' warps of an SM sub-partition take turns at its exponential unit: left
                // alone they fall into step, both in exponentials or both between them (measured: 2240
                // clocks per 64 keys of 256 rows).
                if (tile == 1 || n > 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait_fast(&turn[4 * tile + q4], static_cast<uint32_t>((tile == 1 ? n : n - 1) & 1)));
                    if (!ok) break;
                }
                uint64_t s2[4] = {0, 0, 0, 0};  // the row sum, two lanes and four chains
                uint32_t pk[kCKeys / 2];
#pragma unroll
                for (int i = 0; i < kCKeys / 2; ++i) {
                    float a, b;
                    unpack_f32x2(fma_f32x2(pack_f32x2(sv[2 * i], sv[2 * i + 1]), scale2, base2), a, b);
                    a = ex2_approx(a);
                    b = ex2_approx(b);
                    s2[i & 3] = add_f32x2(s2[i & 3], pack_f32x2(a, b));
                    pk[i] = pack_bf16(a, b);
                    // the other tile's turn; the (always true) condition on what has been summed keeps the
                    // exponentials before it from being scheduled behind it
                    if (i == kTurnAfter - 1) {
                        float x, y;
                        unpack_f32x2(add_f32x2(add_f32x2(s2[0], s2[1]), add_f32x2(s2[2], s2[3])), x, y);
                        if (__any_sync(0xffffffffu, !(x + y < 0.f)) && lane == 0) mbar_arrive(&turn[4 * (tile ^ 1) + q4]);
                    }
                }
                float a, b;
                unpack_f32x2(add_f32x2(add_f32x2(s2[0], s2[1]), add_f32x2(s2[2], s2[3])), a, b);
                l = l * corr + (a + b);
                m = mnew;
                // P.V of the previous tile is done with P's columns (and with O, should it be rescaled)
                if (!first) {
                    ok = __all_sync(0xffffffffu, mbar_wait_fast(&pvdone[tile], static_cast<uint32_t>((n - 1) & 1)));
                    if (!ok) break;
                    tc_fence_after();
                }
                tmem_st32u(tP, pk);
                if (!first && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
                    for (int c = 0; c < kDim / 32; ++c) {
                        float o[32];
                        tmem_ld32(tO + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= corr;
                        tmem_st32(tO + c * 32, o);
                    }
                }
                tmem_wait_st();
                // V rows that no row of the pair sees - past the context in the last tile, or between the
                // sinks and the first row's window - are zeroed so that P = 0 meets 0. Each query tile
                // does it for its own product: the two are issued in either order.
                const int za = max(0, p.sinks - k0), zb = min(kCKeys, sg.lo - k0);
                const bool tail = k0 == last_tile * kCKeys && kv_end < k0 + kCKeys;
                if (tail || za < zb) {
                    const int s = n % kCStages;
                    ok = __all_sync(0xffffffffu, mbar_wait_fast(&vfull[s], ph(n)));
                    if (!ok) break;
                    uint8_t* vd = smem + kCOffV + s * kCKvTile;
                    auto zero_rows = [&](int from, int end) {
                        for (int x = threadIdx.x & 127; x < (end - from) * 16; x += 128) {
                            const int key = from + x / 16;
                            *reinterpret_cast<uint4*>(vd + ((x / 8) & 1) * (kCKeys * 128) + sw128(key, x & 7)) = make_uint4(0, 0, 0, 0);
                        }
                    };
                    if (tail) zero_rows(kv_end - k0, kCKeys);
                    if (za < zb) zero_rows(za, zb);
                    fence_proxy_async_smem();  // the zeros (generic writes) before the MMA reads them
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[tile]);
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait_fast(&pvdone[tile], static_cast<uint32_t>((n - 1) & 1)));
            if (!ok) break;
            // ---- the segment's rows: O / l, or, where the pair's list is cut, O as it is with (m, l). They
            // leave TMEM one per thread, 32 columns at a time, and go to global memory through the warp's
            // staging area, so that a store covers pieces of 4 rows; float4 slot i of staging row r sits
            // at i ^ (r & 7): conflict-free.
            tc_fence_after();
            const bool whole = sg.slot < 0;
            const float wo = whole ? (live ? 1.f / l : 0.f) : 1.f;
            const size_t prow = (static_cast<size_t>(whole ? 0 : sg.slot) * 2 + tile) * kRows;
            if (!whole) {
                p.part_ml[(prow + r) * 2] = m;
                p.part_ml[(prow + r) * 2 + 1] = l;
            } else if (p.row_lse != nullptr && item >= 0) {
                p.row_lse[(static_cast<size_t>(item) * p.kvh + sg.kvhead) * kRows + r] = live ? -(m + log2f(l)) : -INFINITY;
            }
            const int sub = lane >> 3, cq = lane & 7;  // transposed: row 4 * k + sub, 4 columns at 4 * cq
            const unsigned rows_live = __ballot_sync(0xffffffffu, live);
            uint32_t ridx[8];  // this lane's rows in the output, in units of 128 elements (row * H + head)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                ridx[k] = whole ? __shfl_sync(0xffffffffu, static_cast<uint32_t>(oidx), 4 * k + sub)
                                : static_cast<uint32_t>(prow + 32 * q4 + 4 * k + sub);
#pragma unroll 1
            for (int c = 0; c < kDim / 32; ++c) {
                float o[32];
                tmem_ld32(tO + c * 32, o);
                tmem_wait_ld();
                if (c == kDim / 32 - 1) {  // all of O is out
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ofree[tile]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *stg4(lane, i) = make_float4(o[4 * i] * wo, o[4 * i + 1] * wo, o[4 * i + 2] * wo, o[4 * i + 3] * wo);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int row = 4 * k + sub;
                    const float4 x = *stg4(row, cq);
                    if (!(rows_live >> row & 1u)) continue;
                    const size_t off = static_cast<size_t>(ridx[k]) * kDim + c * 32 + 4 * cq;
                    if (!whole)
                        *reinterpret_cast<float4*>(p.part_o + off) = x;
                    else if constexpr (IO16)
                        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + off) =
                            make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
                    else
                        *reinterpret_cast<float4*>(p.out + off) = x;
                }
                __syncwarp();
            }
        }
        if (!ok) {
            *abort_flag = 1;
            if (lane == 0) atomicExch(p.err, kErrTimeout);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the partials of the (pair, KV head)s whose tile lists are cut between CTAs, in slot order: one
// warp per row, lane = 4 dims. split = [nsplit][4] pair, KV head, first slot, slots.
template <bool IO16>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const WideParams p, const int32_t* __restrict__ split, int nsplit) {
    const int wid = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int e = wid / (2 * kRows), tile = (wid / kRows) & 1, r = wid % kRows;
    if (e >= nsplit) return;
    const int pair = split[4 * e], h = split[4 * e + 1], s0 = split[4 * e + 2], ns = split[4 * e + 3];
    const int item = p.w_pair[2 * pair + tile];
    if (item < 0) return;
    const int t = r / p.g;
    const bool live = t < p.w_ntok[item];
    float* lse = p.row_lse != nullptr ? p.row_lse + (static_cast<size_t>(item) * p.kvh + h) * kRows + r : nullptr;
    if (!live) {
        if (lse != nullptr && lane == 0) *lse = -INFINITY;
        return;
    }
    auto row = [&](int s) { return (static_cast<size_t>(s) * 2 + tile) * kRows + r; };
    float mx = -INFINITY;
    for (int s = s0; s < s0 + ns; ++s) mx = fmaxf(mx, p.part_ml[row(s) * 2]);
    float den = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = s0; s < s0 + ns; ++s) {
        const float ms = p.part_ml[row(s) * 2];
        const float f = ms == -INFINITY ? 0.f : exp2f(ms - mx);
        const float4 x = reinterpret_cast<const float4*>(p.part_o + row(s) * kDim)[lane];
        den = fmaf(f, p.part_ml[row(s) * 2 + 1], den);
        a.x = fmaf(f, x.x, a.x);
        a.y = fmaf(f, x.y, a.y);
        a.z = fmaf(f, x.z, a.z);
        a.w = fmaf(f, x.w, a.w);
    }
    const float inv = 1.f / den;
    if (lse != nullptr && lane == 0) *lse = -(mx + log2f(den));
    const size_t off = (static_cast<size_t>(p.tok_row[p.w_tok0[item]] + t) * p.H + h * p.g + r % p.g) * kDim + 4 * lane;
    if constexpr (IO16)
        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + off) =
            make_uint2(pack_bf16(a.x * inv, a.y * inv), pack_bf16(a.z * inv, a.w * inv));
    else
        *reinterpret_cast<float4*>(p.out + off) = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
}

// ---------------------------------------------------------------- weights
// Attention weight of every key of a 128-key tile: a[j] = sum over query rows c of
// 2^(s[j, c] - lse[c]), with the rows' log-sum-exp of chunk_attn_kernel, stored negated (one float per
// column: with maximum and 1 / sum kept apart, reading them from shared memory took half of its
// bandwidth). The score tile is computed
// transposed, S^T = K . Q^T with keys as the MMA rows, so that a thread owns one key and sums its
// row alone: no reduction across threads, and a fixed order. A CTA takes one piece: a key tile of
// one KV head against consecutive query items [i0, i1); the pieces of a tile are added in order by
// weight_pieces_kernel. Q tiles stream through a 2-slot ring, their statistics through an 8-slot one
// (slot x + 8 is filled after the MMA of x + 6, which waited until the epilogue had taken S^T of
// x + 4, so it was done with x), and S^T through two TMEM buffers; at 106 KB of shared memory and 256
// TMEM columns two CTAs share an SM, so that one's exponentials run beside the other's loads and
// MMAs. Bound: one exponential per score, 16 per clock and SM, twice the MMA's time; 63 % of that rate
// (85 us for 2048 rows of 32 heads behind 2048 tokens; with the column masks in every tile and four epilogue
// warps 108, the integer pipe busier than the exponentials).
constexpr int kGThreads = 320;  // producer, MMA issuer, 8 epilogue warps: two per 32 keys, 64 columns each
constexpr int kGOffK = 0;
constexpr int kGOffQ = kGOffK + kTile;
constexpr int kGOffStat = kGOffQ + 2 * kTile;               // [8][128] log-sum-exp
constexpr int kGOffBar = kGOffStat + 8 * kRows * 4;
constexpr int kGSmem = kGOffBar + 256 + 1024;

template <bool IO16>
__global__ void __launch_bounds__(kGThreads, 2)
    chunk_weight_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmq,
                        const __grid_constant__ WideParams p, const int4* __restrict__ pieces, float* __restrict__ part) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ float halves[2][kKeys];
    const float* stat = reinterpret_cast<const float*>(smem + kGOffStat);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + kGOffBar);
    uint64_t* qfull = kfull + 1;    // [2]
    uint64_t* qempty = qfull + 2;   // [2]
    uint64_t* sfull = qempty + 2;   // [2]
    uint64_t* sempty = sfull + 2;   // [2]
    uint64_t* stfull = sempty + 2;  // [8]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stfull + 8);
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
            mbar_init(&sempty[b], 8);
        }
        for (int b = 0; b < 8; ++b) mbar_init(&stfull[b], 1);
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
                mbar_arrive_expect_tx(&stfull[x & 7], kRows * 4);
                bulk_load(smem + kGOffStat + (x & 7) * kRows * 4, p.row_lse + (static_cast<size_t>(i0 + x) * p.kvh + head) * kRows,
                          kRows * 4, &stfull[x & 7]);
                mbar_arrive_expect_tx(&qfull[x & 1], kTile);
                load_query_tile<IO16>(&tmq, smem + kGOffQ + (x & 1) * kTile, &qfull[x & 1], p, i0 + x, head);
                issued = x + 1;
            }
            // never leave the CTA with copies still landing in its shared memory
            mbar_wait_bounded(kfull, 0u);
            for (int x = max(0, issued - 2); x < issued; ++x) mbar_wait_bounded(&qfull[x & 1], (x >> 1) & 1u);
            for (int x = max(0, issued - 8); x < issued; ++x) mbar_wait_bounded(&stfull[x & 7], (x >> 3) & 1u);
        }
    } else if (warp == 1) {
        const uint64_t kd0 = smem_desc(smem_base + kGOffK, 16, 1024);
        const uint64_t qd0 = smem_desc(smem_base + kGOffQ, 16, 1024);
        bool ok = __all_sync(0xffffffffu, mbar_wait_fast(kfull, 0u));
        for (int x = 0; x < n && ok; ++x) {
            const int b = x & 1;
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&qfull[b], (x >> 1) & 1u) && mbar_wait_bounded(&sempty[b], ((x >> 1) & 1u) ^ 1u));
            if (!ok) break;
            tc_fence_after();
            const uint64_t qd = qd0 + b * (kTile >> 4);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kDim / 16; ++kk) {
                    const uint32_t off = ((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4;
                    umma_bf16(tmem + b * kKeys, kd0 + off, qd + off, kIdescS, kk > 0 ? 1u : 0u);
                }
                umma_commit(&sfull[b]);
                umma_commit(&qempty[b]);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            atomicExch(p.err, kErrTimeout);
        }
    } else {
        const int q4 = warp & 3;  // TMEM lanes 32 * q4 .. + 31
        const int half = (warp - 2) >> 2;  // of the columns
        const int key = 32 * q4 + lane;
        const int j = kt * kKeys + key;
        const uint32_t trow = tmem + (static_cast<uint32_t>(32 * q4) << 16) + half * (kRows / 2);
        // items hold tpt = 128 / g consecutive tokens, all but a sequence's last one exactly
        const int tpt = kRows / p.g;
        const int pos_i0 = p.tok_pos[p.w_tok0[i0]];
        const int ntok_last = p.w_ntok[i0 + n - 1];
        uint64_t sum2[2] = {0, 0};
        const uint64_t scale2 = pack_f32x2(p.sscale, p.sscale);
        bool ok = true;
        for (int x = 0; x < n && ok; ++x) {
            const int b = x & 1;
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&stfull[x & 7], (x >> 3) & 1u) && mbar_wait_bounded(&sfull[b], (x >> 1) & 1u));
            if (!ok) break;
            tc_fence_after();
            const float* st = stat + (x & 7) * kRows + half * (kRows / 2);
            // token t of the item, at position pos0 + t, sees key j for t in [j - pos0, j - pos0 + window)
            // (without the upper limit when j is a sink); its columns are g * t .. g * t + g - 1
            const int pos0 = pos_i0 + x * tpt, ntok = x == n - 1 ? ntok_last : tpt;
            const int rel = j - pos0;
            const int t_lo = max(0, rel);
            const int t_hi = j < p.sinks || rel > INT32_MAX - p.window ? ntok : min(ntok, rel + p.window);
            // (columns of this warp's half)
            const int c_lo = t_lo * p.g - half * (kRows / 2), c_hi = t_hi * p.g - half * (kRows / 2);
            const bool whole = __all_sync(0xffffffffu, c_lo <= 0 && c_hi >= kRows / 2);
            float sv[2][32];
            tmem_ld32(trow + b * kKeys, sv[0]);
            tmem_ld32(trow + b * kKeys + 32, sv[1]);
            tmem_wait_ld();
            tc_fence_before();  // S^T is in registers
            __syncwarp();
            if (lane == 0) mbar_arrive(&sempty[b]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float* v = sv[c];
                const ulonglong2* lsep = reinterpret_cast<const ulonglong2*>(st + 32 * c);
                // two columns at a time; masks only where some key does not see all of the rows
                auto add_columns = [&](auto masked) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const ulonglong2 nl = lsep[i];
                        float e[4];
                        unpack_f32x2(fma_f32x2(pack_f32x2(v[4 * i], v[4 * i + 1]), scale2, nl.x), e[0], e[1]);
                        unpack_f32x2(fma_f32x2(pack_f32x2(v[4 * i + 2], v[4 * i + 3]), scale2, nl.y), e[2], e[3]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            e[k] = ex2_approx(e[k]);
                            if constexpr (decltype(masked)::value) {
                                const int col = 32 * c + 4 * i + k;
                                e[k] = col >= c_lo && col < c_hi ? e[k] : 0.f;
                            }
                        }
                        sum2[0] = add_f32x2(sum2[0], pack_f32x2(e[0], e[1]));
                        sum2[1] = add_f32x2(sum2[1], pack_f32x2(e[2], e[3]));
                    }
                };
                if (whole) add_columns(std::false_type{});
                else add_columns(std::true_type{});
            }
        }
        if (!ok) {
            *abort_flag = 1;
            if (lane == 0) atomicExch(p.err, kErrTimeout);
        }
        float a, c;
        unpack_f32x2(add_f32x2(sum2[0], sum2[1]), a, c);
        halves[half][key] = a + c;
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x < kKeys && !*abort_flag)
        part[(static_cast<size_t>(blockIdx.x) * p.kvh + head) * kKeys + threadIdx.x] = halves[0][threadIdx.x] + halves[1][threadIdx.x];
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

cudaError_t launch_chunk_attention(const CUtensorMap* tmk2, const CUtensorMap* tmv2, const CUtensorMap* tmq,
                                   const WideParams& p, const int32_t* split, int nsplit, cudaStream_t st) {
    if (p.nctas <= 0) return cudaSuccess;
    auto kern = p.io16 ? chunk_attn_kernel<true> : chunk_attn_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kCSmem);
    if (e != cudaSuccess) return e;
    kern<<<p.nctas, kCThreads, kCSmem, st>>>(*tmk2, *tmv2, *tmq, p);
    if ((e = cudaGetLastError()) != cudaSuccess || nsplit <= 0) return e;
    auto merge = p.io16 ? chunk_merge_kernel<true> : chunk_merge_kernel<false>;
    merge<<<nsplit * 2 * kRows / 8, 256, 0, st>>>(p, split, nsplit);
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

// Internal declarations shared by the libpagekv translation units.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace pk {

// Most query columns (query token x head-in-group) one tensor-core warp carries.
constexpr int kMaxCols = 16;
// Largest number of KV heads the tensor-core kernel maps to warps of one CTA.
constexpr int kTcMaxKvHeads = 8;
// Largest head_dim of bounded steps and evictions (a row of 16-, 4- or 2-byte words).
constexpr int kMaxBoundedDim = 512;
constexpr int kChunkKeys = 64;  // keys per tile of the bounded chunk kernel
constexpr int kWideKeys = 128;  // keys per tile of the wide-tile kernel (a multiple of block_size)

// Parameters of the split-KV tensor-core attention kernel (bf16 pool).
// Head-sharded output exchange fused into the split-KV kernel (n > 0): every output row goes
// to out[0..n) - each rank's result buffer, already offset to this rank's first query head,
// rows out_H heads apart - and when every consumer warp of the launch has stored its rows
// (a system-scope fence, then a count in `done`), the last one writes `epoch` into flag word
// `rank` of every rank (flag_of) and waits, for at most the wait limit, until every rank's
// flag word here (flags) holds it; a timeout sets *err.
constexpr int kMaxOutPeers = 8;
struct PeerOut {
    int n;
    int out_H;
    int rank;
    unsigned int epoch;
    float* out[kMaxOutPeers];
    unsigned int* flag_of[kMaxOutPeers];
    unsigned int* flags;
    unsigned int* done;  // zero between launches; the last warp resets it
    int* err;
};

// A "unit" is a window of at most kMaxCols / g query tokens of one sequence; every unit
// reads the blocks holding positions 0 .. unit_ctx-1 of its sequence. Units' blocks are
// laid end to end and cut into ncta equal ranges, one per CTA.
struct TcParams {
    const float* q;        // [rows][H][D]
    float* out;            // [rows][H][D]
    // [segments][kvh] blocks of kMaxCols * D floats: un-normalised partial sums in fragment
    // order interleaved by lane (accumulator quad j = mt * NT + nt of lane L is float4
    // j * 32 + L of the block)
    float* part_o;
    float* part_ml;        // [segments][kvh][kMaxCols][2]  (running max, sum), log2 domain
    int* err;              // device error word
    const int32_t* indptr;  // [nseq+1] block-table CSR
    const int32_t* ids;     // block ids
    const int32_t* starts;  // [nseq]
    const int32_t* offsets; // [nseq+1] first row of each sequence
    const int32_t* u_seq;   // [nu] sequence of each unit
    const int32_t* u_t0;    // [nu] first query token of the unit within its sequence
    const int32_t* u_n;     // [nu] query tokens in the unit
    const int32_t* u_blk;   // [nu+1] prefix sum of the units' block counts
    // [nu] first block of the sequence the unit reads (blocks before it - a prefix shared
    // with other sequences - are attended by the wide-tile kernel); NULL = all 0.
    const int32_t* u_kb0;
    // [rows][H] log2-domain log-sum-exp of each output row (max + log2(sum)); NULL = not
    // written. The shared-prefix pass merges its partial with the row through it.
    float* lse;
    // [ncta + 1] first block of each CTA's range; NULL = equal ranges [c*T/ncta, (c+1)*T/ncta)
    const int32_t* cta_blk;
    // [nu][2] first and last CTA whose range holds blocks of each unit; NULL = searched in
    // cta_blk (read only by the in-kernel merge)
    const int32_t* u_cta;
    // [nu] packed unit records, two int4 each: {t0, n, kb0, row0}, {qpos0, blk0, blk1, tbase}
    // (row0 = offsets[seq] + t0, qpos0 = starts[seq] + t0, blk0/blk1 = u_blk[u]/u_blk[u + 1],
    // tbase = indptr[seq] + kb0 - blk0, so that block j's id is ids[tbase + j]); NULL =
    // gathered from the arrays above
    const int4* u_meta;
    int nu;
    int total_blocks;
    int ncta;
    int kvh;
    int g;
    int H;
    int bs;
    int stages;
    int virt;              // virtual CTAs per CTA (0 or 1: one); kvh * virt <= kTcMaxKvHeads
    int per_head_layout;   // 0: one TMA box per K/V block, 1: one box per (block, head)
    int64_t layer_slot0;   // first slot of the layer in the flat [layers*num_blocks*bs] axis
    float qscale;          // log2(e) / sqrt(D)
    // In-kernel merge (NULL counters: leave the partials to merge_kernel): zero-initialised
    // counters per (partial slot, KV head) for the first-level groups of a unit's CTAs, and per
    // (unit, KV head) for the second level; both left at zero by the kernel.
    int* counters;
    int* unit_counters;
    // Fused append: fp32 rows [rows][kvh][D] of this step and the layer's bf16 pool bases;
    // NULL k_new = attention only.
    const float* k_new;
    const float* v_new;
    __nv_bfloat16* pool_k;
    __nv_bfloat16* pool_v;
    PeerOut peer;  // n == 0: rows go to `out` (H heads per row)
    // Bounded modes. q, out, k_new and v_new point at bf16 rows in kTcBounded16.
    const int4* u_bound;  // [nu] {head, skip, score lo, score hi}: see UnitBound in the kernel
    int window;           // >= 1; INT32_MAX without a window
    int sinks;
    float* score;         // masked log2-domain scores per (unit, KV head), or NULL
    float2* ml;           // [rows][H] (max, 1 / sum) of each output row, log2 domain, or NULL
};

enum TcMode { kTcPlain = 0, kTcBounded = 1, kTcBounded16 = 2 };

struct MergeParams {
    float* out;
    const float* part_o;
    const float* part_ml;
    const int32_t* offsets;
    const int32_t* u_seq;
    const int32_t* u_t0;
    const int32_t* u_n;
    const int32_t* split_u;   // [nsplit] unit of each split entry
    const int32_t* split_c0;  // first CTA that worked on it
    const int32_t* split_c1;  // last CTA that worked on it
    int kvh;
    int g;
    int H;
    int D;
    int nt;  // n8 tiles of the attention launch that wrote the partials (fragment layout)
};

// CUDA-core attention for any pool dtype / head_dim (float32 pools, odd shapes).
struct GenericParams {
    const float* q;
    float* out;
    const void* pool_k;  // layer base
    const void* pool_v;
    const int32_t* row_seq;
    const int32_t* indptr;
    const int32_t* ids;
    const int32_t* starts;
    const int32_t* offsets;
    const int32_t* rows;  // rows to process (indices into q/out)
    // Fused append (NULL: off): keys at positions >= the sequence's start are read from these
    // fp32 rows [step rows][kvh][D] (rounded to the pool type), and the CTA of (row, first
    // query head of a KV head) stores its row to the pool (pool_k / pool_v layer bases).
    const float* k_new;
    const float* v_new;
    int nrows;
    int H;
    int kvh;
    int D;
    int bs;
    float scale;  // 1/sqrt(D)
};

// Tensor-core (tcgen05) wide-tile attention: one CTA per (work item, KV head); a work
// item is 128 query rows (= 128/g tokens) of one sequence.
struct WideParams {
    const float* q;
    float* out;
    int* err;
    const int32_t* indptr;
    const int32_t* ids;
    const int32_t* w_seq;   // [nitems] sequence whose block table the item reads
    const int32_t* w_tok0;  // [nitems] first entry of the item's query tokens in tok_row/tok_pos
    const int32_t* w_ntok;  // [nitems] query tokens in the item (<= 128/g)
    const int32_t* w_kend;  // [nitems] keys 0..kend-1 of the table are attended
    const int32_t* tok_row; // query/output row of each token
    const int32_t* tok_pos; // absolute position of each token (causal limit)
    // Shared-prefix pass: NULL = write the normalised output; else merge this partial with
    // the output row already written (and its log2-domain log-sum-exp [rows][H] here).
    const float* lse;
    const int32_t* w_pair;     // [pairs][2] items of a pair (second = -1: none), same table
    const int32_t* pair_kend;  // [pairs] keys of the pair (the larger kend of its items)
    const int32_t* cta_seg;    // [nctas+1] this launch's CTAs: segment ranges
    const int32_t* seg;        // [segments][6] pair, head, first/end key tile, slot (-1 whole), pair-head
    float* part_o;             // [slots][2][128][128] un-normalised partial O
    float* part_ml;            // [slots][2][128][2] (max, sum), log2 domain
    // [items * kvh + 1][32 KB] query tiles packed by launch_wide_q_pack (bf16, scaled,
    // in the shared-memory image the MMA reads); tile item * kvh + head, the last all zero
    const uint8_t* qpk;
    int q_zero_tile;
    int nctas;
    int H;
    int kvh;
    int g;
    int bs;
    int64_t layer_slot0;
    float qscale;
    // Bounded chunk items (chunk_attn_kernel, chunk_weight_kernel).
    const int4* pair_bound;  // [pairs] {head, skip, lo, tiles}: see PairBound in the kernels
    int window;              // >= 1; INT32_MAX without a window
    int sinks;
    float sscale;            // applied to the scores: 1 when the packed queries are scaled, else qscale
    int io16;                // q and out hold bf16
    int bs_shift;            // log2 of bs (a power of two: it divides 128)
    float* row_lse;          // [items][kvh][128] minus the log-sum-exp of each query row, log2 domain (dead rows: -inf), or NULL
};

// Windowed attention on the CUDA cores: any pool, rows of `q` / `out` in the pool's input type.
// A row at position p sees the keys j <= p with j < sinks or j > p - window.
struct BoundedParams {
    const void* q;   // [rows][H][D], float or bf16
    void* out;
    const void* pool_k;  // layer base
    const void* pool_v;
    const int32_t* row_seq;
    const int32_t* indptr;
    const int32_t* ids;
    const int32_t* starts;
    const int32_t* offsets;
    const int32_t* rows;  // rows to process (indices into q / out)
    float2* ml;  // [rows][H] softmax statistics of each row: (max, 1 / sum), log2 domain; NULL = not kept
    int nrows;
    int H;
    int kvh;
    int D;
    int bs;
    int window;  // >= 1; INT32_MAX without a window
    int sinks;
    float qscale;  // log2(e) / sqrt(D)
};

// Windowed attention on the CUDA cores for rows of 4-element multiples (cc_attn_kernel).
struct CcParams {
    const void* q;       // [rows][H][D], float or bf16 as k_new, v_new and out
    void* out;
    const void* pool_k;  // layer base
    const void* pool_v;
    const void* k_new;   // fused append: the step's rows [rows][kvh][D]; NULL = off
    const void* v_new;
    const int32_t* ids;
    const int4* meta;    // [nrows][2] {row, first table entry, position, sequence start}, {sequence's first row, ..}
    float2* ml;          // [rows][H] (max, 1 / sum), log2 domain, or NULL
    float* weights;      // fused weights of the layer, or NULL
    float* part;         // [nrows][grid.y][nsplit][G][D + 2] partials (nsplit > 1)
    int* counters;       // [nrows][grid.y], zero between launches
    int nrows;
    int nsplit;
    int max_vis;         // most visible keys of a row (fused weights)
    int H;
    int kvh;
    int D;
    int bs;
    int bs_shift;        // log2 of bs, or -1
    int window;          // >= 1; INT32_MAX without a window
    int sinks;
    int add;
    float qscale;        // log2(e) / sqrt(D)
};
// Query heads of a KV head that a CTA of cc_attn_kernel takes together.
inline int cc_group(int g) { return g == 1 ? 1 : g == 2 ? 2 : 4; }

// Windowed attention on the CUDA cores in tiles of kTileCols columns - (token, head) pairs of a sequence
// and KV head - by kTileKeys keys (tile_attn_kernel), for sequences with kTileMinCols columns and more.
constexpr int kTileCols = 64, kTileKeys = 64, kTileMinCols = 32, kTileMaxDim = 256;
// Columns from which tile_weight_kernel sums a sequence's weights; more than the 4 heads of a KV head up
// to which a decode row's are summed inside cc_attn_kernel. Weights of 7 verify rows of 2 heads, 15
// contexts up to 1886: 306 us with the attention by rows, 218 here; decode rows of 8 heads 214 and 220,
// of 5 heads 597 and 702.
constexpr int kTileMinWeightCols = 8;
struct TileParams {
    const void* q;       // [rows][H][D], float or bf16
    void* out;
    const void* pool_k;  // layer base
    const void* pool_v;
    const int32_t* ids;
    const int4* meta;    // [nunits] {first row, first table entry, its position, tokens}
    float2* ml;          // [rows][H] (max, 1 / sum), log2 domain, or NULL
    float* part;         // [nunits][kvh][nsplit][kTileCols][D + 4] partials (nsplit > 1)
    int* counters;       // [nunits][kvh], zero between launches
    int nunits;
    int nsplit;
    int H;
    int kvh;
    int D;
    int bs;
    int bs_shift;        // log2 of bs, or -1
    int window;          // >= 1; INT32_MAX without a window
    int sinks;
    float qscale;        // log2(e) / sqrt(D)
};
// Their weights (tile_weight_kernel): tiles of kTileKeys consecutive slots of a sequence's touched blocks.
struct TileWeightParams {
    float* weights;
    const int4* meta;      // [ntiles][2] {first row, first table entry, start, rows} of the sequence,
                           // {its first touched block, their number, first slot of the tile, 0}
    const int32_t* t_blk;  // touched blocks: table index
    float* part;           // [ntiles][kvh][nparts][kTileKeys] (nparts > 1)
    int* counters;         // [ntiles][kvh], zero between launches
    int ntiles;
    int nparts;            // CTAs of a tile and KV head
    int add;
};

// The touched blocks of a step - those with a key that some row sees - and the layer's
// accumulated weights [num_blocks][kvh][bs].
struct WeightParams {
    float* weights;
    const int32_t* t_seq;  // [ntouched] sequence
    const int32_t* t_blk;  // [ntouched] block of its table
    int ntouched;
    int add;  // add to the weights of tokens cached before the step (else store)
    int max_rows;  // most new rows of a touched sequence
};

// Weights from the scores that a bounded split-KV launch kept, one warp per touched block.
struct ScoreWeightParams {
    WeightParams w;
    const int4* t_meta;     // [ntouched][2] {block id, table index, first and end unit of the sequence},
                            // {first new position, context, first slot of the part, 0}
    const float* score;
    const float2* ml;
    const int4* u_meta;     // units as in TcParams
    const int4* u_bound;
    int kvh;
    int g;
    int H;
    int bs;
    int bs_shift;           // log2 of bs, or -1
    int block;              // slots of a block (bs, or more: entries are parts of blocks)
    int window;
    int sinks;
    int max_units;          // most units of a sequence
};

struct EvictParams {
    void* pool_k;
    void* pool_v;
    float* weights;        // [layers][num_blocks][kvh][bs]
    const int32_t* lengths;  // [nseq]
    const int32_t* indptr;   // block tables before and after
    const int32_t* ids;
    const int32_t* new_indptr;
    const int32_t* new_ids;
    int32_t* kept;         // [layers][nseq][kvh][budget] kept positions, ascending, -1 behind the last
    const int32_t* items;  // [nitems][3] sequence, first and end new position
    int64_t num_blocks;
    int nitems;
    int nseq;
    int layer0;  // the launch's layers: layer0 .. layer0 + layers - 1 (kept: the first is layer0's)
    int layers;
    int kvh;
    int bs;
    int row_bytes;  // bytes of one (slot, KV head) row of K or V
    int budget;
    int sinks;
    int recent;
    // set by launch_evict: sequences up to this length keep their weights in shared memory; words of
    // a row; logarithms of bs and row_words (-1: no power of two)
    int cache_cap;
    int row_words;
    int bs_shift;
    int words_shift;
};

// Read-only view of a pool's fields for entry points outside pk_api.cu.
struct PoolView {
    int device;
    int n_layers;
    int64_t num_blocks;
    int block_size;
    int kvh;
    int d;
    int dtype;
    int num_sms;
    bool tc_ok;
    int tc_per_head;
    int tc_stages;
    int tc_virt;
    size_t tc_smem;
    const CUtensorMap* tmk;
    const CUtensorMap* tmv;
};

cudaError_t launch_tc_attention(int D, int NT, int mode, const CUtensorMap* tmk, const CUtensorMap* tmv,
                                const TcParams& p, size_t smem, cudaStream_t st);
size_t tc_smem_bytes(int D, int bs, int kvh, int stages, int virt);
// Shared memory a launch with the fused head exchange needs beyond tc_smem_bytes (each consumer
// warp's staging of 4 output rows, and alignment slack).
size_t tc_peer_stage_bytes(int D);
cudaError_t launch_merge(const MergeParams& p, int nsplit, cudaStream_t st);
size_t wide_smem_bytes();
cudaError_t launch_wide_attention(const CUtensorMap* tmk1, const CUtensorMap* tmv1, const WideParams& p,
                                  cudaStream_t st);
// Bytes of one packed query tile of the wide-tile kernel (128 rows x 128 dims, bf16).
constexpr int kWideQTileBytes = 128 * 128 * 2;
// Packs the query tiles of `nitems` wide-tile items (all KV heads) plus the zero tile into
// p.qpk-sized memory at `qpk`.
cudaError_t launch_wide_q_pack(const WideParams& p, int nitems, uint8_t* qpk, cudaStream_t st);
// Append of chunk rows into a bf16 pool, slots resolved from the block table.
struct WideAppend {
    __nv_bfloat16* pool_k;
    __nv_bfloat16* pool_v;
    const float* k;
    const float* v;
    const int32_t *row_seq, *offsets, *starts, *indptr, *ids;
    const int32_t* rows;  // [n] the step rows to append
    const int64_t* slots; // [n] their pool slots (layer 0); NULL = looked up from the tables
    int64_t n;
    int rowlen;           // kvh * head_dim
    int bs;
};
// launch_wide_q_pack and the append of `a` in one launch (a.n == 0: pack only).
cudaError_t launch_wide_prep(const WideParams& p, int nitems, uint8_t* qpk, const WideAppend& a, cudaStream_t st);
// Combines the partial slots of (pair, head)s cut between wide-kernel CTAs:
// split = [nsplit][4] pair, head, first slot, slots.
cudaError_t launch_wide_merge(const WideParams& p, const int32_t* split, int nsplit, cudaStream_t st);
cudaError_t launch_generic_attention(int dtype, const GenericParams& p, cudaStream_t st);
cudaError_t launch_plan_rows(const int32_t* row_seq, const int32_t* offsets, const int32_t* starts,
                             const int32_t* indptr, const int32_t* ids, int bs, int64_t nrows,
                             int64_t* positions, int64_t* slots, cudaStream_t st);
cudaError_t launch_append(int dtype, void* pool_k_layer, void* pool_v_layer, const float* k,
                          const float* v, const int64_t* slots, const int32_t* rows, int64_t n,
                          int rowlen, cudaStream_t st);
// The same with each row's slot resolved from the block table (row -> sequence -> position
// -> block id), with no per-row slots array.
cudaError_t launch_append_table(int dtype, void* pool_k_layer, void* pool_v_layer, const float* k,
                                const float* v, const int32_t* row_seq, const int32_t* offsets,
                                const int32_t* starts, const int32_t* indptr, const int32_t* ids, int bs,
                                const int32_t* rows, int64_t n, int rowlen, cudaStream_t st);
cudaError_t launch_copy_blocks(void* k, void* v, const int64_t* pairs, int64_t npairs, int layers,
                               int64_t layer_bytes, int64_t block_bytes, cudaStream_t st);
// The accumulated weights of copied blocks: pairs as in launch_copy_blocks, `block` floats each.
cudaError_t launch_copy_weights(float* weights, const int64_t* pairs, int64_t npairs, int layers, int64_t layer_floats,
                                int block, cudaStream_t st);
// Zeroes one layer's accumulated weights of n tokens: at `slots`, or (NULL) of the step's rows by the block table.
cudaError_t launch_clear_weights(float* weights, const int64_t* slots, const int32_t* row_seq, const int32_t* offsets,
                                 const int32_t* starts, const int32_t* indptr, const int32_t* ids, int bs, int kvh,
                                 int64_t n, cudaStream_t st);
cudaError_t launch_bounded_wait_selftest(int* err, unsigned long long limit_ns, cudaStream_t st);
// Three device-addressable host arrays (float counts multiples of 4, 16-byte aligned) into
// device buffers, one launch.
cudaError_t launch_h2d_gather(const float* a_src, float* a_dst, int64_t a_floats, const float* b_src, float* b_dst,
                              int64_t b_floats, const float* c_src, float* c_dst, int64_t c_floats, cudaStream_t st);
// src [world][rows][row_floats] -> dst [rows][world][row_floats]; row_floats % 4 == 0, both
// pointers 16-byte aligned.
cudaError_t launch_interleave_heads(const float* src, float* dst, int world, int64_t rows, int64_t row_floats,
                                    cudaStream_t st);
cudaError_t launch_slot_mapping(const int32_t* table, int64_t table_len, const int64_t* positions,
                                int64_t n, int bs, int64_t* slots, int32_t* err, cudaStream_t st);

cudaError_t launch_cc_attention(int dtype, bool io16, const CcParams& p, cudaStream_t st);
cudaError_t launch_tile_attention(int dtype, bool io16, const TileParams& p, cudaStream_t st);
cudaError_t launch_tile_weights(int dtype, bool io16, const TileParams& p, const TileWeightParams& w, cudaStream_t st);
cudaError_t launch_bounded_rows(int dtype, bool io16, const BoundedParams& p, cudaStream_t st);
cudaError_t launch_weight_rows(int dtype, bool io16, const BoundedParams& p, const WeightParams& w, cudaStream_t st);
// Chunk items of a bounded step: p.nctas CTAs over the segments of p.cta_seg / p.seg, then the merge
// of the `nsplit` (pair, KV head)s cut between CTAs. tmq: the tensor map of bf16 queries
// (p.io16; unread otherwise); tmk2 / tmv2: boxes of min(block_size, kChunkKeys) slots.
size_t chunk_smem_bytes();
cudaError_t launch_chunk_attention(const CUtensorMap* tmk2, const CUtensorMap* tmv2, const CUtensorMap* tmq,
                                   const WideParams& p, const int32_t* split, int nsplit, cudaStream_t st);
// Their weights: pieces {sequence, key tile, first and end query item} scored into
// part[npieces][kvh][128], then added up into the touched blocks of `w` (t_piece: first piece of
// each block's key tile and how many).
cudaError_t launch_chunk_weights(const CUtensorMap* tmk1, const CUtensorMap* tmq, const WideParams& p, const int4* pieces,
                                 int npieces, float* part, const WeightParams& w, const int32_t* starts,
                                 const int32_t* offsets, const int2* t_piece, cudaStream_t st);
cudaError_t launch_weight_scores(const ScoreWeightParams& p, cudaStream_t st);
// launch_append_table for rows given as bf16 (bf16 pools).
cudaError_t launch_append_rows16(void* pool_k_layer, void* pool_v_layer, const void* k, const void* v,
                                 const int32_t* row_seq, const int32_t* offsets, const int32_t* starts,
                                 const int32_t* indptr, const int32_t* ids, int bs, const int32_t* rows, int64_t n,
                                 int rowlen, cudaStream_t st);
// Chooses the tokens that stay and moves them (two launches); max_len: the longest sequence.
cudaError_t launch_evict(const EvictParams& p, int max_len, cudaStream_t st);

}  // namespace pk

struct pk_pool;
// Fills *out from `pool`; false if pool is NULL.
bool pk_pool_view(const pk_pool* pool, pk::PoolView* out);
struct pk_peer_gather;
// The exchange of the next step of `g` for slices of [rows][row_floats] floats (row_floats =
// heads x d of one rank): bumps the step epoch and fills *po (d: floats per head); *result is
// this rank's [rows][world * row_floats] result buffer of that step. PK_OK or an error code.
int pk_peer_gather_step(pk_peer_gather* g, int64_t rows, int64_t row_floats, int d, pk::PeerOut* po,
                        float** result);
// Sets the message pk_last_error() returns on this thread.
void pk_set_last_error(const char* msg);

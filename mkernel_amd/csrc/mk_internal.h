// mk_internal.h — kernel parameter blocks and launchers shared between the
// HIP translation units of libmk (not part of the C-ABI).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mk_map.h"
#include "mk_plan.h"
#include "mk_product_plan.h"

namespace mk {

enum Epilogue : int { kEpiStore = 0, kEpiSwiGLU = 1, kEpiReduce = 2 };
enum PermMode : int { kPermNone = 0, kPermArrival = 1, kPermOwnedSpread = 2, kPermPeerArrival = 3 };
constexpr int kMaxTilesM = 512;
constexpr int kMaxSplitListTiles = 4096;  // K-split with a permuted tile order: at most this many tiles
constexpr int kMaxRounds = 64;   // cooperative staging between rounds: at most this many rounds
constexpr int kMaxTopk = 32;     // choices per token of the router and of the combine's gradient
constexpr int kMaxExperts = 1024; // experts of the router
constexpr int kPieces = 16;  // cooperative staging: pieces per 128-row block

struct GemmKParams {
  // operands
  const uint16_t* A;
  const uint16_t* B;
  uint16_t* C;
  int64_t lda, ldb, ldc;
  int64_t b_expert_stride;  // elements between experts' B matrices
  int M, N, K;
  int tiles_m, tiles_n;
  int group_m;
  // 128-row grouped GEMMs: walk each expert's run of row tiles column by
  // column (one expert's tiles consecutive) instead of the grouped order
  int expert_order;
  // grid roles
  int n_prod, n_cons;
  int xcd_remap;
  int waves;                // 4 (one wave per SIMD) or 8 (two per SIMD)
  // grouped GEMM: expert of each BM row tile (nullptr = dense)
  const int* rb_expert;
  const int* expert_rows;   // padded rows per expert (used when rb_expert is null)
  const int* rb_rows;       // real rows per 128-row tile (null: every row is real)
  // fused dispatch: A is the token buffer [gather_rows, K], row r of the
  // GEMM reads the token the pull table names (null: A rows are the rows)
  const int* gather_pull;
  int64_t gather_rows;
  int gather_tps, gather_devs;
  int n_experts;
  // SwiGLU: width I of the gate half of B's columns
  int swiglu_I;
  // consumer A-row gate (AllGather side)
  const uint32_t* a_flags;
  const int* a_stage_order;
  int perm_mode;
  // reduce epilogue (ReduceScatter side)
  int rs_own_row0, rs_own_rows, rs_npeers;
  const uint16_t* rs_recv;
  uint16_t* rs_out;
  const uint32_t* rs_flags;
  uint32_t* ar_done;        // all-reduce: per output tile, epoch once its reduced bytes are visible
  // producer staging: block b (128 rows of st_cols) copied st_src -> st_dst
  const uint16_t* st_src;
  uint16_t* st_dst;
  int st_cols, st_nblocks;
  // Blocks at index >= st_split_at (when st_src2 is set) form a second
  // staging set: block st_split_at + b copies st_src2 block b to st_dst2
  // block b, or b + st_dst2_skip from block st_dst2_skip_at on (the
  // all-gather half of a two-shot all-reduce: the other slices' reduced
  // rows into C_final, around this rank's own slice).
  const uint16_t* st_src2;
  uint16_t* st_dst2;
  int st_split_at, st_dst2_skip_at, st_dst2_skip;
  int st_present;           // stage positions < st_present hold blocks already in st_dst: published, not copied
  const int* st_order;
  uint32_t* st_flags;
  uint32_t* st_counters;    // cooperative staging: pieces completed per block (mod kPieces)
  int st_coop;              // 1: even share, 2: alternating halves, 3: claimed (co-resident staging kernel)
  // st_coop 3: [0] the next unclaimed piece, shared with the staging kernel;
  // [1] claimers checked out; the last of st_claimers compute workgroups +
  // st_stage_waves staging waves to check out zeroes both
  uint32_t* st_claim;
  int st_claimers, st_stage_waves;
  int st_batch;             // pieces per release after the first (1..8)
  // K-split of the tail round: tiles >= sk_full are split sk_split ways along
  // K (sk_split <= 1: no split); partials go through sk_ws with sk_flags
  float* sk_ws;
  uint32_t* sk_flags;
  int sk_full, sk_split;
  // Device row count (128-row grouped GEMMs launched at a row capacity
  // before the routed row count is known on the host): *rows_dev rows are
  // real, tiles past them are not walked, and with sk_dev the tail round's
  // K-split is planned on the device by the host's rule (sk_ws / sk_flags
  // then hold n_cons partial tiles).
  const int64_t* rows_dev;
  int sk_dev;
  int spread_dev;           // with rows_dev: spread an unsplittable tail over fewer consumers (host rule)
  // flag protocol: the epoch is *epoch_ptr when that is set (read once per
  // use at run time, written by an earlier launch), else `epoch`
  const uint32_t* epoch_ptr;
  uint32_t epoch;
  uint32_t spin_limit;
  uint32_t* err;
};

hipError_t launch_gemm(const GemmKParams& p, int bm, int epi, hipStream_t stream, int bn = 256);
// Expert GEMM with a device row count, which the tile width follows
// (few_row_blocks); p.tiles_n counts 512-column tiles.
hipError_t launch_gemm_expert(const GemmKParams& p, int epi, hipStream_t stream);
// Co-resident staging: the one-wave staging kernel (waves_per_cu per CU)
// followed by a register-capped 256 x 256 GEMM that may start while the
// staging kernel runs; both claim pieces through p.st_claim.
hipError_t launch_gemm_costaged(const GemmKParams& p, int epi, int n_stage_waves, hipStream_t stream);
hipError_t launch_epoch_advance(uint32_t* epoch_ptr, hipStream_t stream);
// The staging of p's blocks alone (st_* fields).
hipError_t launch_stage_all(const GemmKParams& p, int grid, hipStream_t stream);

// Dense GEMM on small tiles (mk_gemm_small.hip).
struct GemmSmallParams {
  const uint16_t* A;
  const uint16_t* B;
  uint16_t* C;
  int64_t lda, ldb, ldc;
  int K;
  int tiles_m, tiles_n, group_m;
  int nk;            // 64-deep K stages of a tile
  int split;         // parts of a tile along K (1: whole)
  // zero between launches: a ticket per tile and a header per workgroup of a
  // K-split; with done flags, the finished parts of each
  uint32_t* words;
  float* ws;         // an fp32 tile per workgroup
  // reduce epilogue: rows rs_own_row0 .. + rs_own_rows are folded with the
  // peers' staged partials into rs_out, the others are stored to C
  int rs_own_row0, rs_own_rows, rs_npeers;
  const uint16_t* rs_recv;
  uint16_t* rs_out;
  // flags of the folded rows' 256 x 256 tiles, row by row (null: none), each
  // set to the epoch once all of its tile is visible at agent scope
  uint32_t* done;
  int done_cols;
  const uint32_t* epoch_ptr;
  uint32_t epoch;
};
hipError_t launch_gemm_small(const GemmSmallParams& p, const GemmSmallPlan& plan, bool reduce, hipStream_t stream);

struct PermuteKParams {
  const uint16_t* tokens;
  const int* pull;
  uint16_t* post;
  int64_t R_pad, H, n_src_rows;
  int tokens_per_src, devs_per_node;
  const int64_t* rows_dev;  // device row count (rows at or past it are skipped), or null
};
hipError_t launch_permute(const PermuteKParams& p, hipStream_t stream);

struct CombineKParams {
  const void* y_expert;
  const float* row_weight;
  const int* owner_offset;
  const int* slot_to_row;
  void* y_out;
  int64_t num_tokens, H;
  int out_dtype;
  int f32_rows;             // y_expert holds fp32
  uint32_t rows;            // rows of y_expert: others contribute nothing; 0: no table of rows is read
};
hipError_t launch_combine(const CombineKParams& p, hipStream_t stream);
hipError_t launch_tile_rows(const int* pull, int64_t R_pad, int* rb_rows, hipStream_t stream);

// Gradient of the combine (mk_moe.hip).
struct CombineBwdKParams {
  const void* dy;
  const uint16_t* y_expert;
  const int* ids;
  const float* row_weight;
  const int* owner_offset;
  const int* slot_to_row;
  const int* rb_rows;
  uint16_t* dy_expert;      // null: not computed
  float* dgates;
  int64_t T, H, R_pad;
  int k, e0, n_local;
  int dy_dtype;
  const int64_t* rows_dev;
  int pad_blocks;           // set by the launch
};
hipError_t launch_combine_backward(CombineBwdKParams p, hipStream_t stream);

// Router (mk_route.hip).
struct RouteKParams {
  const void* logits;
  const uint8_t* mask;
  int* ids;
  float* gates;
  int64_t T, ld;
  int E, k, bf16, renorm;
  // balance sums (part_sum null: none)
  int* counts;
  float* prob_sum;
  int* tokens;
  float* loss;
  float coef;
  double* shares;      // an expert group's share of the loss, per workgroup of the second kernel
  uint32_t* ticket;
  float* part_sum;     // [workgroups][E]
  int* part_cnt;       // [workgroups][E]
  int* part_live;      // [workgroups]
};
struct RouteBwdKParams {
  const void* logits;
  const uint8_t* mask;
  const int* ids;
  const float* dgates;
  const float* dloss;
  const int* counts;
  const int* tokens;
  void* dlogits;
  int64_t T, ld, ld_out;
  int E, k, bf16, renorm;
  float coef;
};
int64_t route_workspace_bytes(int64_t T, int E);
// ws null: no balance sums
hipError_t launch_route(RouteKParams p, void* ws, hipStream_t stream);
hipError_t launch_route_backward(const RouteBwdKParams& p, hipStream_t stream);

// Products with 4-bit weights (mk_w4.hip).
struct W4Weights {
  const unsigned char* packed;   // [E][tile pairs][blocks] of two tiles' codes, scales and zero points
  int64_t K, N;
  int group, E;
  bool zeros;                    // whether there are zero points (else 8)
};
enum W4Out : int { kW4F32 = 0, kW4Bf16 = 1, kW4Pair = 2 };
struct W4KParams {
  W4Weights w;
  const uint16_t* A;
  void* C;
  int64_t lda, ldc, M;      // elements; M: rows of A (dense) or of the tables
  int tile_cols;            // output column tiles of 16
  int swiglu;
  int parts;                // 2: a row of A is two bf16 rows of K whose sum it stands for
  int out_type;             // W4Out; a pair is two bf16 rows of the result's width
  uint32_t passes;          // set by the launch: row passes,
  int split;                // and waves that share an item's K (dense)
  // experts (rb_expert null: one dense product)
  const int* rb_expert;
  const int* rb_rows;
  const int* gather_pull;
  int64_t gather_rows;
  int gather_tps, gather_devs;
  const int64_t* rows_dev;
};
int64_t w4_packed_bytes(int64_t K, int64_t N, int64_t E, int group, bool zeros);
hipError_t launch_w4(const W4KParams& p, int cus, hipStream_t stream);
hipError_t launch_w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int64_t K, int64_t N,
                          int64_t E, int group, unsigned char* packed, hipStream_t stream);
hipError_t launch_w4_quantize(const uint16_t* W, int64_t K, int64_t N, int64_t E, int group, uint8_t* codes,
                              uint16_t* scales, hipStream_t stream);

// Products with what follows them (mk_product.h, mk_product.hip).
enum ProductEpilogue : int { kProdStore = 0, kProdSwiglu = 1, kProdSwigluGrad = 2, kProdStats = 3, kProdDlogits = 4,
                             kProdPlain = 5, kProdPlain32 = 6,  // kProdStore without anything but bf16 or fp32 results
                             kProdDlogits3 = 7 };  // three parts of the logits' gradient
enum ProductOrder : int { kProdForward = 0, kProdLeftGrad = 1, kProdRightGrad = 2 };
enum ProductAct : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };
// which rows of the epilogue start at 16-byte boundaries
enum ProductVec : int { kVecC = 1, kVecRes = 2, kVecPre = 4, kVecBias = 8 };
struct ProductParams {
  const uint16_t* A;
  const uint16_t* B;
  int64_t lda, ldb;
  int64_t M, N, K;          // of C; with ragged 1 M, with ragged 2 K is the rows of the buffers
  int64_t b_cols;           // valid columns of a k-strided B
  // groups
  const int* counts;
  int E, ragged;            // 0 none, 1 rows of A and C, 2 rows of A and B
  int64_t b_stride, c_stride;  // elements between groups' B (ragged 1) and C (ragged 2), or the parts of a gradient
  // tiles
  int tiles_m, tiles_n, group_m;
  int whole, split;         // tiles from `whole` on are cut into `split` parts along K
  uint32_t* tickets;        // one per cut tile, kTicketStride words apart, zero between launches
  float* parts;             // a tile per part
  // epilogue
  int vec, act;
  void* C;                  // SwiGLU: [M, N]; its gradient: [M, 2 N]
  int64_t ldc;
  int c_f32;
  const void* bias;
  int bias_f32;
  const void* res;          // added behind the activation (may be C); SwiGLU's gradient: [M, 2 N] gate | up
  int64_t ldr;
  int res_f32;
  uint16_t* pre;            // store: sum + bias; SwiGLU: [M, 2 N] gate | up
  int64_t ldp;
  int up;                   // SwiGLU: B's first up column
  // vocabulary
  const void* labels;
  int labels64;
  int64_t ignore, label0, vocab, first_col;
  float2* stats;            // [column tiles][M]
  float* target;
  const float* lse;
  const float* dloss;
  const float* scale;       // one number that dloss is divided by and the gradients' sums multiplied with, or null
};
hipError_t launch_product_forward(const ProductParams& p, int epi, int tile, int64_t grid, hipStream_t stream);
hipError_t launch_product_left_grad(const ProductParams& p, int epi, int tile, int64_t grid, hipStream_t stream);
hipError_t launch_product_right_grad(const ProductParams& p, int epi, int tile, int64_t grid, hipStream_t stream);
// Forward, plain epilogue, one row or two: operands of any alignment.
hipError_t launch_product_few_rows(const ProductParams& p, hipStream_t stream);
// Rows of bf16 into rows of a multiple of 8 elements, zeros behind the last: `parts` pieces of `cols` columns each,
// one behind the other, every piece filled up to `width`; groups (counts, E) that have no rows are left out.
// labels: rows whose label is `ignore` become zeros.
struct RepackParams {
  const uint16_t* src;
  uint16_t* dst;
  int64_t rows, cols, ld, src_stride, dst_stride;  // strides between the groups' matrices
  int64_t width;
  int parts, E;
  const int* counts;
  const void* labels;
  int labels64;
  int64_t ignore;
  const float* dloss;       // with labels: `scale` gets 1 <= the significand < 2 of the largest finite |dloss| there
  float* scale;
};
hipError_t launch_repack(const RepackParams& p, hipStream_t stream);
// dpre = dC * act'(pre), bf16 rows of `width` (null: not kept; in `terms` parts, M * width elements apart, that add up
// to it), and the columns' sums of it
struct ActGradParams {
  const uint16_t* dC;
  const uint16_t* pre;
  uint16_t* dpre;
  int64_t M, N, ldc, ldp, width;
  int act, vec_c, vec_p, terms;
  float* part;              // [row_blocks][N], null: no sums
  float* dbias;
  int accumulate;
  int64_t row_blocks;       // set by act_grad_blocks
};
int64_t act_grad_blocks(int64_t M, int64_t N);
hipError_t launch_act_grad(const ActGradParams& p, hipStream_t stream);
struct VocabJoinParams {
  const float2* stats;
  int64_t groups, T;
  const void* labels;
  int labels64;
  int64_t ignore, label0, vocab;
  float* target;
  float* lse;
  float* loss;
};
hipError_t launch_vocab_join(const VocabJoinParams& p, hipStream_t stream);

int64_t index_workspace_bytes(int T, int topk, int n_local);
hipError_t launch_mfma_ceiling(int64_t iters, int n_wg, uint32_t seed, float* sink, uint64_t* clocks,
                               hipStream_t stream);
int probe_threads();
hipError_t launch_invert_slots(const int* row_to_slot, const int* row_to_owner, int64_t R_pad, int owner,
                               int64_t slot_capacity, int* slot_to_row, uint32_t* err, hipStream_t stream);

}  // namespace mk

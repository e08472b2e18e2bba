/*
 * mk.h — C-ABI of libmk, the MI355X (gfx950) compute core behind mKernel's
 * fused operators at one GPU's share of the work.
 *
 * Plain pointers and sizes only; no torch types.  Every device pointer is a
 * HIP device address; `stream` is a hipStream_t passed as void* (NULL = the
 * default stream).  All tensors are caller-owned and row-major.  bf16 buffers
 * are raw 16-bit storage (IEEE bfloat16).
 *
 * Return codes: 0 = ok, negative = argument/shape error (MK_E*), positive =
 * a hipError_t from a launch.  mk_last_error_string() describes the last
 * non-zero return on the calling thread.
 *
 * Each entry point names the reference interface it replaces (file:line in
 * uccl-project/mKernel).
 */
#ifndef MK_H_
#define MK_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MK_OK 0
#define MK_EINVAL (-1)   /* null pointer / bad enum */
#define MK_ESHAPE (-2)   /* shape not supported by the tiling */
#define MK_EDEVICE (-3)  /* no usable device / wrong architecture */
#define MK_ETIMEOUT (-4) /* a bounded flag wait expired (error word set) */
#define MK_EWORKSPACE (-5) /* the workspace is too small: nothing was queued (mk_gemm_act and the entry points behind it) */

#define MK_ROW_BLOCK 128 /* flag / expert-padding granularity (rows) */

/* ------------------------------------------------------------------------ */
/* Plain persistent bf16 GEMM: C[M,N] = A[M,K] @ B[K,N], fp32 accumulate,
 * bf16 (round-to-nearest-even) output.
 * Replaces the compute role shared by ag_gemm / gemm_rs
 * (reference src/gemm_rs.cu:36-114 compute_tile_impl,
 *  src/ag_gemm.cu:265-461 fused_comp_sm).
 * Requires M % 128 == 0, N % 256 == 0, K % 32 == 0, ld* >= row width and
 * ld* % 8 == 0. */
typedef struct mk_gemm_args {
  const void* A;  /* bf16 [M, lda] */
  const void* B;  /* bf16 [K, ldb] */
  void* C;        /* bf16 [M, ldc] */
  int64_t M, N, K;
  int64_t lda, ldb, ldc;
  int32_t num_cus; /* persistent grid size; 0 = every CU of the device; at most the CU count */
  int32_t tile_m;  /* 0 = auto; 128 or 256: the persistent kernel's tile height.  With
                      tile_m, waves and num_cus all 0 the library chooses between that
                      kernel and one on tiles of 64 x 64 to 128 x 256 */
  int32_t waves;   /* waves per workgroup: 0 = auto, 4 (one per SIMD) or 8 (two per SIMD) */
  void* split_ws;          /* optional K-split workspace (see mk_query_workspace_bytes);
                              zero-filled before its first use, left zeroed by every
                              launch; NULL = no tile is split along K (neither the
                              tail round's nor a small problem's) */
  int64_t split_ws_bytes;
} mk_gemm_args;
int mk_gemm(const mk_gemm_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* Flag-gated AllGather+GEMM consumer with an in-GPU producer role.
 * C[M,N] = A_full[M,K] @ B[K,N].  A_full is assembled from `world` row
 * shards: `num_producers` producer workgroups copy 128-row tiles of
 * A_shards into A_full in the order `stage_order` and release-store
 * flags[tile] = epoch after each tile; compute workgroups acquire-poll the
 * flags of the rows they are about to read (s_sleep between polls).
 * Replaces ag_gemm_multinode::entrypoint
 * (reference include/operators/ag_gemm/ag_gemm.cuh:362-509) with the
 * intra_comm_sm gather role (src/ag_gemm.cu:31-215) and the per-chunk flag
 * wait of fused_comp_sm (src/ag_gemm.cu:374-377).
 *   gated == 0             : plain GEMM on A_full, no flags read (baseline)
 *   gated, producers == 0  : flags are published by someone else
 *   gated, producers  > 0  : that many producer workgroups run inside the
 *                            launch beside the compute workgroups
 *   gated, producers == -1 : cooperative staging — the compute workgroups
 *                            copy 128 KB pieces (in stage order) between
 *                            their tile rounds, counting pieces per tile in
 *                            stage_counters; the workgroup that completes a
 *                            tile publishes its flag.  Before round 0 every
 *                            workgroup copies what round 0 waits for; after
 *                            that the two halves of the grid (XCDs 0-3 and
 *                            4-7) take turns: one copies ahead for the next
 *                            round while the other computes
 *   gated, producers == -2 : cooperative staging with every workgroup
 *                            copying an even share before every round
 *                            (both: with num_cus == 0 the library may instead
 *                            queue a copy kernel on every CU that stages and
 *                            publishes all blocks, then the GEMM, where that
 *                            is faster; same outputs, flags and counters)
 *   gated, producers <= -3 : wave-specialised producer: a staging kernel of
 *                            (-2 - producers) one-wave workgroups per
 *                            compute workgroup (1..4) runs beside a GEMM
 *                            capped at 224 VGPRs (room for one 64-VGPR
 *                            staging wave per SIMD) on a library side
 *                            stream, forked from and joined back into
 *                            `stream`; pieces are claimed in stage order
 *                            from a word in split_ws (required), the
 *                            compute workgroups claiming what a round
 *                            still lacks.  Under graph capture the call
 *                            stages cooperatively (-1) instead.  Needs
 *                            stage_counters. */
typedef struct mk_ag_gemm_args {
  const void* A_shards;  /* bf16 [M, K]: shards stacked in rank order (source) */
  void* A_full;          /* bf16 [M, K]: gathered A (destination / GEMM input) */
  const void* B;         /* bf16 [K, N] */
  void* C;               /* bf16 [M, N] */
  int64_t M, N, K;
  uint32_t* flags;              /* [M/128] epoch-stamped ready flags */
  const int32_t* stage_order;   /* [M/128] device; NULL = ascending */
  uint32_t epoch;               /* value a ready flag must hold (never 0) */
  int32_t gated;
  int32_t num_producers;
  int32_t num_cus;              /* total workgroups (producers + compute); 0 = all CUs; never more
                                   than the device's CUs (every workgroup must be resident) */
  uint32_t spin_limit;          /* polls before a wait gives up; 0 = unbounded */
  uint32_t* error_word;         /* optional device word, bit0 set on timeout */
  uint32_t* stage_counters;     /* [M/128] piece counters for producers == -1; zero once, never reset */
  void* split_ws;          /* optional K-split workspace (see mk_query_workspace_bytes);
                              zero-filled before its first use, left zeroed by every
                              launch; NULL = no K-split of the tail round */
  int64_t split_ws_bytes;
  /* Optional device word holding the epoch: when set, the launch reads the
   * epoch from it (never 0) instead of `epoch`, so a HIP graph that records
   * mk_epoch_advance and this launch gates every replay on a new epoch with
   * no host work.  NULL = use `epoch`. */
  const uint32_t* epoch_ptr;
  /* Number of leading stage_order positions whose 128-row blocks are
   * already in A_full (this rank's own shard, written there by the caller
   * as the reference bench does, bench/ag_gemm_bench.py:364-372): the
   * staging publishes their flags without copying them, and A_shards is
   * not read for them.  0 = every block is copied.  Needs stage_order when
   * non-zero. */
  int32_t n_present;
} mk_ag_gemm_args;
int mk_ag_gemm(const mk_ag_gemm_args* args, void* stream);

/* mk_ag_gemm without any allocation.  No counterpart in the reference: it
 * is for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  The
 * K-split workspace and the cooperative-staging piece counters come from a
 * static device array of mk_ag_gemm_noalloc_scratch_bytes() bytes (about
 * 32 MB, one copy per GPU, held until the process ends); split_ws,
 * split_ws_bytes and stage_counters must be NULL / 0.  Limits: M/128 <=
 * 16384 row blocks (larger M returns MK_ESHAPE); a tail round whose K-split
 * would need more than 128 partial tiles runs unsplit; num_producers <= -3
 * (the co-resident staging kernel, whose side stream and events the library
 * creates on first use) stages cooperatively (-1) instead.  Each call checks
 * every argument, then clears the counters, split flags and claim words it
 * uses on `stream` (a small kernel), then launches mk_ag_gemm's kernels.  Every call on one GPU shares that
 * GPU's array: calls that overlap in time on one GPU (different streams)
 * race and must not be issued. */
int mk_ag_gemm_noalloc(const mk_ag_gemm_args* args, void* stream);
int64_t mk_ag_gemm_noalloc_scratch_bytes(void);

/* ------------------------------------------------------------------------ */
/* GEMM + reduce-scatter epilogue at one rank's share.
 * P = A[M,K] @ B[K,N] (this rank's partial over all M rows).  Rows owned by
 * `rank` ([rank*M/world, (rank+1)*M/world)) are folded in the epilogue:
 *   output = bf16( P_owned + sum_{p<world-1} peer_recv[p] )   (fp32 adds)
 * after acquire-waiting the flags of each peer tile; every other row is the
 * would-be send and is written to workspace.  The producer role copies
 * peer_src into peer_recv tile by tile and release-stores the flags.
 * Replaces gemm_rs_multinode::entrypoint_fused
 * (reference include/operators/gemm_rs/gemm_rs.cuh:510-935): compute_tile_impl
 * (src/gemm_rs.cu:36-114) + reduce_tiles_ws (src/gemm_rs.cu:685-845). */
typedef struct mk_gemm_rs_args {
  const void* A;          /* bf16 [M, K] */
  const void* B;          /* bf16 [K, N] */
  void* workspace;        /* bf16 [M, N]; non-owned rows written */
  void* output;           /* bf16 [M/world, N] owned slice */
  const void* peer_src;   /* bf16 [world-1, M/world, N] partials to stage */
  void* peer_recv;        /* bf16 [world-1, M/world, N] staged partials */
  int64_t M, N, K;
  int32_t world, rank;
  uint32_t* flags;              /* [(world-1) * (M/world)/128] */
  const int32_t* stage_order;   /* [(world-1) * (M/world)/128]; NULL = ascending */
  uint32_t epoch;
  int32_t gated;
  int32_t num_producers;        /* as in mk_ag_gemm; -1 and -2 = cooperative staging, even share
                                   (or staged first by a copy kernel, with num_cus == 0);
                                   <= -3 = co-resident staging kernel (needs split_ws) */
  int32_t num_cus;
  uint32_t spin_limit;
  uint32_t* error_word;
  uint32_t* stage_counters;     /* [(world-1) * (M/world)/128] for producers == -1 */
  void* split_ws;          /* optional K-split workspace (see mk_query_workspace_bytes);
                              zero-filled before its first use, left zeroed by every
                              launch; NULL = no K-split of the tail round */
  int64_t split_ws_bytes;
  /* Optional device word holding the epoch: when set, the launch reads the
   * epoch from it (never 0) instead of `epoch`, so a HIP graph that records
   * mk_epoch_advance and this launch gates every replay on a new epoch with
   * no host work.  NULL = use `epoch`. */
  const uint32_t* epoch_ptr;
} mk_gemm_rs_args;
int mk_gemm_rs(const mk_gemm_rs_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* GEMM + all-reduce at one rank's share.
 *   C_final = bf16( A @ B + sum_{p < world-1} peer_recv[p] )   (fp32 adds, p ascending)
 * over all M rows: the reduce epilogue of mk_gemm_rs with every row owned.
 * The producer role (or cooperative staging, num_producers = -1) copies
 * peer_src into peer_recv in 128-row blocks, flags[(p * M/128) + block] =
 * epoch, in the order stage_order; compute follows the arrival order of each
 * row tile's last peer block.  When done_flags is set, each finished
 * 256x256 output tile t = row_tile * (N/256) + col_tile is published as
 * done_flags[t] = epoch after its bytes are visible at agent scope (the hand-off
 * the reference's broadcast step reads); a copy kernel that stages first
 * (num_producers -1 or -2) delays the first of them by its own time.
 * Replaces gemm_ar_multinode::entrypoint
 * (reference include/operators/gemm_ar/session.cuh:188-215,
 * src/gemm_ar.cu:1-33 compute + intra-AR roles; the reference checks
 * C_final against all_reduce(matmul), bench/gemm_ar_bench.py:510-514). */
typedef struct mk_gemm_ar_args {
  const void* A;          /* bf16 [M, K] */
  const void* B;          /* bf16 [K, N] */
  void* C_final;          /* bf16 [M, N] */
  const void* peer_src;   /* bf16 [world-1, M, N] partials to stage */
  void* peer_recv;        /* bf16 [world-1, M, N] staged partials */
  int64_t M, N, K;
  int32_t world;
  uint32_t* flags;              /* [(world-1) * M/128] */
  const int32_t* stage_order;   /* [(world-1) * M/128]; NULL = ascending, no arrival order */
  uint32_t epoch;
  int32_t gated;
  int32_t num_producers;        /* as in mk_ag_gemm; -1 and -2 = cooperative staging, even share
                                   (or staged first by a copy kernel, with num_cus == 0);
                                   <= -3 = co-resident staging kernel (needs split_ws) */
  int32_t num_cus;
  uint32_t spin_limit;
  uint32_t* error_word;
  uint32_t* stage_counters;     /* [(world-1) * M/128] for producers == -1 */
  uint32_t* done_flags;         /* [(M/256) * (N/256)] or NULL */
  void* split_ws;               /* as in mk_gemm_rs; also counts the parts of done_flags' tiles where
                                   those are computed in smaller ones (a product of few tiles takes
                                   longer with done_flags and no split_ws) */
  int64_t split_ws_bytes;
  /* Optional device word holding the epoch: when set, the launch reads the
   * epoch from it (never 0) instead of `epoch`, so a HIP graph that records
   * mk_epoch_advance and this launch gates every replay on a new epoch with
   * no host work.  NULL = use `epoch`. */
  const uint32_t* epoch_ptr;
} mk_gemm_ar_args;
int mk_gemm_ar(const mk_gemm_ar_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* GEMM + all-reduce at one rank's share, two-shot: this rank reduces only
 * its own row slice and receives the other slices already reduced by their
 * owners (reduce-scatter, then all-gather), so each output row is reduced
 * once across the node — the work split of the reference's multicast
 * all-reduce, where each tile is reduced once for all GPUs
 * (reference src/gemm_ar.cu:9-32, intra-AR role with multimem reduction;
 * include/operators/gemm_ar/session.cuh:188-215).  With s = M/world rows
 * per slice and r = rank:
 *   C_final[r*s .. (r+1)*s)  = bf16( (A @ B)[own rows] + sum_p peer_recv[p] )
 *                              (fp32 adds, p ascending; the reduce epilogue)
 *   C_final[other slices]    = peer_reduced, staged in 128-row blocks
 *   sends[rows outside r's]  = bf16( (A @ B)[those rows] )  (this rank's pushes)
 * One launch: flags / stage_counters / stage_order cover 2*(world-1)*s/128
 * blocks, first the partial blocks of this rank's slice (peer_src ->
 * peer_recv, as mk_gemm_rs), then the reduced blocks (peer_reduced ->
 * C_final, flags[(world-1)*s/128 + b] = epoch once block b is in place).
 * done_flags (optional, [(M/256)*(N/256)]): each finished tile of this rank's
 * slice, as in mk_gemm_ar.  num_producers as in mk_gemm_rs; 0 = everything
 * was staged by someone else (flags published; peer_reduced unread). */
typedef struct mk_gemm_ar2_args {
  const void* A;            /* bf16 [M, K] */
  const void* B;            /* bf16 [K, N] */
  void* C_final;            /* bf16 [M, N] */
  void* sends;              /* bf16 [M, N]; rows outside this rank's slice written */
  const void* peer_src;     /* bf16 [world-1, M/world, N]: peers' partials of this rank's slice, rank order without r */
  void* peer_recv;          /* bf16 [world-1, M/world, N] staged partials */
  const void* peer_reduced; /* bf16 [world-1, M/world, N]: the other slices, reduced, slice order without r */
  int64_t M, N, K;
  int32_t world, rank;
  uint32_t* flags;              /* [2 * (world-1) * (M/world)/128] */
  const int32_t* stage_order;   /* permutation of those blocks; NULL = ascending */
  uint32_t epoch;
  int32_t gated;
  int32_t num_producers;
  int32_t num_cus;
  uint32_t spin_limit;
  uint32_t* error_word;
  uint32_t* stage_counters;     /* [2 * (world-1) * (M/world)/128] */
  uint32_t* done_flags;         /* [(M/256) * (N/256)] or NULL */
  void* split_ws;               /* as in mk_gemm_rs; also counts the parts of done_flags' tiles where
                                   those are computed in smaller ones (a product of few tiles takes
                                   longer with done_flags and no split_ws) */
  int64_t split_ws_bytes;
  const uint32_t* epoch_ptr;
} mk_gemm_ar2_args;
int mk_gemm_ar_two_shot(const mk_gemm_ar2_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* MoE routing index build (host memory, host CPU).  Restates the reference's
 * host-side builders bench/dispatch_gemm_bench.py:127-188 (build_routing,
 * build_pull_indices) and bench/dispatch_gemm_glu_combine_bench.py:222-293,
 * 513-527 (build_gather_indices, local_rb_per_expert, row_expert) for one
 * rank owning experts [expert_begin, expert_begin + n_local).
 * Rows are grouped by local expert (ascending); inside an expert, source
 * tokens ascend; each expert is padded to a multiple of `row_block` with
 * pull rows (-1,-1,-1).  Tokens come from one source (node 0, dev 0). */
int mk_moe_index_sizes(const int32_t* topk_ids, int32_t num_tokens, int32_t topk,
                       int32_t expert_begin, int32_t n_local, int32_t row_block,
                       int64_t* R_out, int64_t* R_pad_out);

typedef struct mk_moe_index {
  /* all host arrays, caller-allocated */
  int32_t* padded_tokens_per_expert; /* [n_local] */
  int32_t* local_rb_per_expert;      /* [n_local] whole row blocks of real rows */
  int32_t* pull_indices;             /* [R_pad, 3] (src_node, src_dev, src_token) */
  int32_t* row_expert;               /* [R_pad] local expert of each row */
  int32_t* rb_expert;                /* [R_pad / row_block] */
  int32_t* rb_rows;                  /* [R_pad / row_block] real (non-padding) rows per row block */
  float* row_weight;                 /* [R_pad] gate of each row; 0 on padding */
  int32_t* owner_offset;             /* [num_tokens + 1] CSR over source tokens */
  int32_t* row_to_slot;              /* [R_pad] slot of each row; 0 on padding */
  int32_t* row_to_owner;             /* [R_pad] owner dev of each row; -1 on padding */
  int32_t* slot_to_row;              /* [R] inverse of row_to_slot */
} mk_moe_index;
int mk_moe_build_indices(const int32_t* topk_ids, const float* topk_gates,
                         int32_t num_tokens, int32_t topk, int32_t expert_begin,
                         int32_t n_local, int32_t row_block, const mk_moe_index* out);

/* ------------------------------------------------------------------------ */
/* The same routing index tables built on the GPU from top-k ids and gates in
 * device memory (no host round trip), bit-identical to
 * mk_moe_build_indices.  Row tables (pull_indices, row_expert, row_weight,
 * row_to_slot, row_to_owner, slot_to_row) must hold `capacity_rows` rows,
 * rb_expert / rb_rows capacity_rows / row_block entries; R and R_pad land in
 * the device word pair `sizes` when the stream reaches them.  If R_pad >
 * capacity_rows, sizes still reports it and rows past the capacity are not
 * written (capacity_rows = num_tokens * topk + n_local * (row_block - 1)
 * always suffices).  `workspace` holds mk_moe_index_workspace_bytes bytes.
 * At most 4096 local experts.
 * No counterpart in the reference, whose builders are host Python
 * (bench/dispatch_gemm_bench.py:127-188,
 * bench/dispatch_gemm_glu_combine_bench.py:222-293, 511-527). */
typedef struct mk_moe_index_dev_args {
  const int32_t* topk_ids;   /* [num_tokens, topk] device */
  const float* topk_gates;   /* [num_tokens, topk] device */
  int32_t num_tokens, topk, expert_begin, n_local, row_block;
  int64_t capacity_rows;
  void* workspace;
  int64_t workspace_bytes;
  int64_t* sizes;            /* device [2]: R, R_pad */
  mk_moe_index out;          /* device pointers; NULL skips a table */
} mk_moe_index_dev_args;
int64_t mk_moe_index_workspace_bytes(int32_t num_tokens, int32_t topk, int32_t n_local);
int mk_moe_build_indices_dev(const mk_moe_index_dev_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* Token permute into expert-contiguous rows:
 *   post[r] = tokens[src_row(r)]   (bit-exact copy), zero on padding rows,
 * src_row = (src_node * devs_per_node + src_dev) * tokens_per_src + src_token.
 * Replaces dispatch_fused (reference src/dispatch_gemm.cu:106-198). */
typedef struct mk_moe_permute_args {
  const void* tokens;           /* bf16 [n_src_rows, H] */
  const int32_t* pull_indices;  /* [R_pad, 3] device */
  void* post_tokens;            /* bf16 [R_pad, H] */
  int64_t R_pad, H;
  int64_t n_src_rows;
  int32_t tokens_per_src, devs_per_node;
  /* Optional device row count {R, R_pad} (the `sizes` pair that
   * mk_moe_build_indices_dev writes), or NULL.  When set, R_pad above is the
   * row capacity the tables and buffers were sized for, and rows at or past
   * sizes[1] are skipped, so the call needs no host read-back of the routed
   * row count (and can be recorded in a HIP graph).  No counterpart in the
   * reference, whose row counts come from its host builders. */
  const int64_t* sizes;
} mk_moe_permute_args;
int mk_moe_permute(const mk_moe_permute_args* args, void* stream);

/* Grouped GEMM over expert-contiguous rows.
 *   mode 0: out[r] = post[r] @ W[e(r)]                 (W: [E, K, N])
 *   mode 1: out[r] = silu(h[:, :I]) * h[:, I:], h = post[r] @ W[e(r)]
 *           (W: [E, K, 2I], out: [R_pad, I])   SwiGLU fused in the epilogue
 * e(r) = rb_expert[r / 128] when rb_expert is given, else the expert whose
 * padded row range [sum_{e'<e} padded[e'], sum_{e'<=e} padded[e']) holds r,
 * from padded_tokens_per_expert (the reference's own table).  Counts that sum
 * to more than R_pad are cut off there; rows past every range go to the last
 * expert.
 * Replaces group_gemm_fused (reference src/dispatch_gemm.cu:207-408),
 * gemm1_swiglu_fused (src/dispatch_gemm_glu_combine.cu:441-643) and
 * ffn_gemm2/grouped_gemm (src/dispatch_gemm_glu_combine.cu:247-429,647-651). */
typedef struct mk_moe_grouped_gemm_args {
  const void* A;              /* bf16 [R_pad, K] */
  const void* W;              /* bf16 [E, K, Nw] */
  void* out;                  /* bf16 [R_pad, N_out] */
  const int32_t* rb_expert;   /* [R_pad/128] device, or NULL */
  const int32_t* padded_tokens_per_expert; /* [E] device; used when rb_expert is NULL */
  const int32_t* rb_rows;     /* [R_pad/128] real rows per row block, or NULL; lets the
                                 kernel skip MFMAs of all-padding 32-row blocks */
  int64_t R_pad, K, Nw;       /* Nw = W's column count (2I in mode 1) */
  int32_t num_experts;
  int32_t mode;
  int32_t num_cus;
  void* split_ws;              /* optional K-split workspace, as in mk_gemm_args */
  int64_t split_ws_bytes;
  /* Fused dispatch (the reference's moe_dispatch_gemm_fused,
   * include/operators/dispatch_gemm/dispatch_gemm.cuh:238-262): when
   * gather_pull is set, A is the token buffer [n_src_rows, K] and GEMM row r
   * reads token row (src_node * devs_per_node + src_dev) * tokens_per_src +
   * src_token of pull row r (padding rows read zeros); no permuted copy is
   * made.  n_src_rows * K * 2 must stay below 2 GiB. */
  const int32_t* gather_pull;  /* [R_pad, 3] device, or NULL */
  int64_t n_src_rows;
  int32_t tokens_per_src, devs_per_node;
  int32_t tile_n;              /* output tile width: 256, 512 (Nw % 512 == 0), or 0 = library choice */
  /* Optional device {R, R_pad}, as in mk_moe_permute_args: row tiles at or
   * past sizes[1] are not computed (R_pad is the capacity) and the tail
   * round's K-split is planned on the device; the split then needs
   * split_ws to hold mk_query_workspace_bytes() bytes, else it is off. */
  const int64_t* sizes;
} mk_moe_grouped_gemm_args;
int mk_moe_grouped_gemm(const mk_moe_grouped_gemm_args* args, void* stream);

/* Top-k weighted combine back to source-token order (gather, no atomics):
 *   y[t] = sum_{s in [owner_offset[t], owner_offset[t+1])}
 *              row_weight[slot_to_row[s]] * y_expert[slot_to_row[s]]
 * products and sum in fp32; output fp32 (out_dtype 0) or bf16 (1).
 * y_expert, row_weight and slot_to_row are read only inside owner_offset's
 * ranges; with one of them NULL (no routed rows) y = 0.  Every MoE entry
 * accepts R_pad == 0 (no rows routed to this rank): permute and the grouped
 * GEMMs do nothing and need no buffers, and the layers' y_out is 0.  In the
 * layers (mk_moe_ffn_combine, mk_moe_ffn_combine_w4) slots whose row is at or
 * past R_pad add nothing.
 * Replaces combine_producer_fused + combine_gather_owner
 * (reference src/dispatch_gemm_glu_combine.cu:736-818). */
typedef struct mk_moe_combine_args {
  const void* y_expert;         /* bf16 [R_pad, H] */
  const float* row_weight;      /* [R_pad] */
  const int32_t* owner_offset;  /* [num_tokens + 1] */
  const int32_t* slot_to_row;   /* [R] */
  void* y_out;                  /* [num_tokens, H] fp32 or bf16 */
  int64_t num_tokens, H;
  int32_t out_dtype;
} mk_moe_combine_args;
int mk_moe_combine(const mk_moe_combine_args* args, void* stream);

/* Turns the reference's producer-side tables (row_to_slot, row_to_owner;
 * bench/dispatch_gemm_glu_combine_bench.py:264-279) into the gather table
 * the combine reads: slot_to_row[0 .. slot_capacity) is first set to -1,
 * then slot_to_row[row_to_slot[r]] = r for every row r with
 * row_to_owner[r] == owner.  Rows of other owners (another GPU combines
 * them) are left out, and the combine skips slots that stay -1.  A slot
 * outside [0, slot_capacity) is not written; it sets bit 1 of *error_word
 * when error_word is non-NULL. */
int mk_moe_invert_slots(const int32_t* row_to_slot, const int32_t* row_to_owner, int64_t R_pad, int32_t owner,
                        int64_t slot_capacity, int32_t* slot_to_row, uint32_t* error_word, void* stream);

/* rb_rows[b] = number of rows r in [128b, 128b+128) with pull_indices[r][0] >= 0
 * (device, from the reference's pull table). */
int mk_moe_tile_rows(const int32_t* pull_indices, int64_t R_pad, int32_t* rb_rows, void* stream);

/* The whole local MoE layer in one call: permute -> grouped GEMM1 + SwiGLU ->
 * grouped GEMM2 -> combine (four launches on `stream`).
 * Replaces moe_dispatch_gemm_glu_combine_fused
 * (reference include/operators/dispatch_gemm_glu_combine/dispatch_gemm_glu_combine.cuh:307-548). */
typedef struct mk_moe_ffn_args {
  const void* tokens;           /* bf16 [n_src_rows, H] */
  const int32_t* pull_indices;  /* [R_pad, 3] */
  const int32_t* rb_expert;     /* [R_pad/128], or NULL */
  const int32_t* padded_tokens_per_expert; /* [E]; used when rb_expert is NULL */
  const int32_t* rb_rows;       /* [R_pad/128] real rows per row block, or NULL */
  const float* row_weight;      /* [R_pad] */
  const int32_t* owner_offset;  /* [num_tokens + 1] */
  const int32_t* slot_to_row;   /* [R] */
  const void* w1;               /* bf16 [E, H, 2I] (gate | up) */
  const void* w2;               /* bf16 [E, I, H] */
  void* post_tokens;            /* bf16 [R_pad, H]  (caller scratch / output) */
  void* act;                    /* bf16 [R_pad, I] */
  void* y_expert;               /* bf16 [R_pad, H] */
  void* y_out;                  /* [num_tokens, H] fp32 or bf16 */
  int64_t num_tokens, n_src_rows, R_pad, H, I;
  int32_t num_experts;
  int32_t tokens_per_src, devs_per_node;
  int32_t out_dtype;
  int32_t num_cus;
  void* split_ws;              /* optional K-split workspace, as in mk_gemm_args */
  int64_t split_ws_bytes;
  int32_t fuse_dispatch;       /* 1: GEMM1 gathers tokens itself, post_tokens is not written */
  int32_t tile_n;              /* grouped GEMM tile width, as in mk_moe_grouped_gemm_args */
  /* Optional device {R, R_pad}, as in mk_moe_permute_args: with it the
   * whole layer (permute, both grouped GEMMs, combine) runs from the device
   * tables of mk_moe_build_indices_dev at their capacity, with no host
   * read-back between the index build and the combine. */
  const int64_t* sizes;
} mk_moe_ffn_args;
int mk_moe_ffn_combine(const mk_moe_ffn_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* Router of the MoE layer: top-k choice, gates, and (optionally) per-expert
 * counts and the balance loss, in one pass over the logits.
 *   topk_ids[t, i] = expert of the i-th largest logit of token t; equal logits
 *     (-0 equals 0) go to the lowest expert index, NaN ranks above everything
 *     and -inf is never chosen: a token with fewer than topk other logits has
 *     id -1 and gate 0 in the places left (the index build skips such ids)
 *   p[t, e]  = exp(logit - max) / sum over the token's experts   (fp32)
 *   gates[t, i] = p of the choice, divided by the sum over the token's choices
 *     when renorm is set.  A NaN or +inf among a token's logits makes all its
 *     p and gates NaN.
 * A token does not count when its token_mask byte is 0 (its logits are not
 * read) or all its logits are -inf: ids -1, gates 0, nothing added below.
 * With counts set (then all of prob_sum, tokens, loss and workspace):
 *   counts[e] = choices of e,  prob_sum[e] = sum_t p[t, e],  tokens = n = tokens that count
 *   loss = coef * num_experts / (topk * n^2) * sum_e counts[e] * prob_sum[e]
 * (coef when every expert gets the same share of both; 0 when n = 0).  Sums
 * are added in a fixed order: equal inputs give equal bits.  The workspace
 * needs no clearing and holds nothing between calls.
 * At most 1024 experts and 32 choices.  No counterpart in the reference, whose
 * benches draw their routing on the host (bench/dispatch_gemm_bench.py:103-124). */
typedef struct mk_moe_route_args {
  const void* logits;          /* [num_tokens, ld]: the first num_experts of each row */
  const uint8_t* token_mask;   /* [num_tokens] or NULL */
  int32_t* topk_ids;           /* [num_tokens, topk] */
  float* gates;                /* [num_tokens, topk] */
  int64_t num_tokens, ld;
  int32_t num_experts, topk;
  int32_t logits_dtype;        /* 0 fp32, 1 bf16 */
  int32_t renorm;
  int32_t* counts;             /* [num_experts] or NULL: no balance outputs */
  float* prob_sum;             /* [num_experts] */
  int32_t* tokens;             /* [1] */
  float* loss;                 /* [1] */
  float coef;
  void* workspace;             /* mk_moe_route_workspace_bytes bytes, 16-byte aligned */
  int64_t workspace_bytes;
} mk_moe_route_args;
int64_t mk_moe_route_workspace_bytes(int64_t num_tokens, int32_t num_experts);
int mk_moe_route(const mk_moe_route_args* args, void* stream);

/* Gradient of mk_moe_route's logits, from the gates' gradient and from the
 * balance loss (either part may be left out: dgates or counts NULL).  With the
 * forward's p and gates g of the choices c_i, recomputed here from the logits:
 *   renorm:  dlogits[j]  = sum_i [c_i = j] g_i (dgates_i - sum_l g_l dgates_l)
 *   else:    dlogits[j]  = sum_i [c_i = j] p_j dgates_i - p_j sum_l p_{c_l} dgates_l
 *   balance: dlogits[j] += dloss * coef * E / (topk n^2) * p_j (counts[j] - sum_e counts[e] p_e)
 * (the counts are constants of the loss; counts and n = tokens may be sums over
 * several ranks).  Choices outside [0, num_experts) have no gradient; tokens
 * that do not count get zeros.  dlogits has the logits' type and may be the
 * logits themselves, with the same ld, but share no other element with them. */
typedef struct mk_moe_route_backward_args {
  const void* logits;          /* as in mk_moe_route */
  const uint8_t* token_mask;
  const int32_t* topk_ids;     /* [num_tokens, topk]; read when dgates is set */
  const float* dgates;         /* [num_tokens, topk] or NULL */
  const float* dloss;          /* [1] or NULL: 1 */
  const int32_t* counts;       /* [num_experts] or NULL */
  const int32_t* tokens;       /* [1]; read when counts is set */
  void* dlogits;               /* [num_tokens, ld_out]: the first num_experts of each row are written */
  int64_t num_tokens, ld, ld_out;
  int32_t num_experts, topk;
  int32_t logits_dtype;
  int32_t renorm;
  float coef;
} mk_moe_route_backward_args;
int mk_moe_route_backward(const mk_moe_route_backward_args* args, void* stream);

/* Gradient of mk_moe_combine for one rank's experts [expert_begin,
 * expert_begin + n_local), with the tables that mk_moe_build_indices(_dev)
 * made from topk_ids at row_block 128:
 *   dy_expert[r] = row_weight[r] * dy[t(r)]         (fp32 product, bf16; zero on padding rows)
 *   dgates[t, j] = sum_h dy[t, h] * y_expert[r(t, j), h]   (fp32)
 * dgates is 0 where topk_ids names no local expert (another rank has that
 * part) or the row was not produced here (slot_to_row -1).  Rows at or past
 * R_pad (sizes[1] when sizes is set, R_pad then being the capacity) are
 * neither read nor written; with R_pad 0 every table of rows may be NULL, and
 * dgates is 0.  dy_expert may be NULL, and rb_rows then too; it may be y_expert
 * itself, whose padding rows are then zeroed as well, but shares no other memory
 * with y_expert or dy.
 * Each sum is added in a fixed order.  At most 32 choices.  No counterpart in
 * the reference, which has no backward pass. */
typedef struct mk_moe_combine_backward_args {
  const void* dy;               /* [num_tokens, H] fp32 or bf16 */
  const void* y_expert;         /* bf16 [R_pad, H] */
  const int32_t* topk_ids;      /* [num_tokens, topk] */
  const float* row_weight;      /* [R_pad] */
  const int32_t* owner_offset;  /* [num_tokens + 1] */
  const int32_t* slot_to_row;   /* [R] */
  const int32_t* rb_rows;       /* [R_pad/128] */
  void* dy_expert;              /* bf16 [R_pad, H] or NULL */
  float* dgates;                /* [num_tokens, topk] */
  int64_t num_tokens, H, R_pad;
  int32_t topk, expert_begin, n_local;
  int32_t dy_dtype;             /* 0 fp32, 1 bf16 */
  const int64_t* sizes;         /* device {R, R_pad} or NULL */
} mk_moe_combine_backward_args;
int mk_moe_combine_backward(const mk_moe_combine_backward_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* 4-bit weights with group scales:
 *   w[k, n] = (code[k, n] - zero[k / group, n]) * scale[k / group, n]
 * codes and zero points 0 .. 15 (8 where there are no zero points), scales
 * bf16, group 32, 64 or 128 rows of K, the last one shorter where K ends in
 * it; K and N up to 2^24, 2^40 weights in all.  The products read them in an order of their own, laid out once by
 * mk_w4_pack; E matrices (experts) of one shape lie one after another. */
typedef struct mk_w4_weights {
  void* packed;      /* mk_w4_packed_bytes bytes, 16-byte aligned: codes, scales and zero points */
  int64_t K, N;
  int32_t group, num_experts;
  int32_t has_zeros; /* 0: the zero point is 8 */
} mk_w4_weights;
int64_t mk_w4_packed_bytes(int64_t K, int64_t N, int32_t num_experts, int32_t group, int32_t has_zeros);

/* Lays out codes uint8 [E, K, N] (the low four bits of each byte), scales bf16
 * [E, ceil(K / group), N] and zero points uint8 of the scales' shape. */
typedef struct mk_w4_pack_args {
  const void* codes;
  const void* scales;
  const void* zeros;    /* set exactly when out.has_zeros is */
  mk_w4_weights out;
} mk_w4_pack_args;
int mk_w4_pack(const mk_w4_pack_args* args, void* stream);

/* Codes and scales of bf16 weights [E, K, N], without zero points: scale =
 * bf16(largest magnitude of the group / 7), code = round(w / scale) + 8 cut to
 * 0 .. 15 (8 where the scale is 0).  With a NaN in a group its scale is NaN, so
 * that all its weights are; with an infinity it is infinite, and the infinities
 * keep their sign. */
typedef struct mk_w4_quantize_args {
  const void* W;        /* bf16 [E, K, N] */
  void* codes;          /* uint8 [E, K, N] */
  void* scales;         /* bf16 [E, ceil(K / group), N] */
  int64_t K, N;
  int32_t group, num_experts;
} mk_w4_quantize_args;
int mk_w4_quantize(const mk_w4_quantize_args* args, void* stream);

/* C[M, N] = A[M, K] @ w (num_experts 1), fp32 sums, bf16 or fp32 output.  For
 * few rows: the weights are expanded for every 16 of them (32 where that leaves
 * work for every CU).  K % 8 == 0, lda % 8 == 0, A 16-byte aligned; C aligned to
 * its elements, apart from A (it may be other columns of the same rows); any M
 * up to 2^20 and any N.  A group's sum is that of
 * A * (16 + code) - A * (16 + zero), exact products: its fp32 roundings are
 * relative to at most 31 times the group's sum of |A|, and an infinity in a row
 * of A, or a group whose |A| sum to more than 2^123, makes that row of C NaN or
 * infinite. */
typedef struct mk_gemm_w4_args {
  const void* A;        /* bf16 [M, lda] */
  void* C;              /* [M, ldc] */
  mk_w4_weights W;
  int64_t M, lda, ldc;
  int32_t out_type;     /* 0 fp32, 1 bf16 */
} mk_gemm_w4_args;
int mk_gemm_w4(const mk_gemm_w4_args* args, void* stream);

/* mk_moe_grouped_gemm with 4-bit weights, for the few rows per expert of a
 * decode batch: out[r] = A[r] @ w[e(r)] (mode 0), or silu(h[:, :I]) * h[:, I:]
 * of h = A[r] @ w[e(r)] with I = N / 2 a multiple of 16 (mode 1).  rb_expert
 * names the expert of each 128-row block (blocks that name none are skipped);
 * only the rb_rows real rows of a block are computed, other rows of out stay as
 * they are.  out is fp32, bf16, or a bf16 pair: a row holds its values rounded
 * to bf16 and behind them what the rounding left, again in bf16 (17 bits of
 * significand: off by 2^-17 of the value at most, a 512th of a bf16 result's
 * own rounding); such rows are read with a_parts 2.  A is 16-byte aligned,
 * out to its elements, and apart from A.  gather_pull,
 * n_src_rows, tokens_per_src, devs_per_node and sizes as in
 * mk_moe_grouped_gemm_args. */
typedef struct mk_moe_grouped_gemm_w4_args {
  const void* A;               /* bf16 [R_pad, K * a_parts], or the token buffer [n_src_rows, K] */
  mk_w4_weights W;
  void* out;                   /* [R_pad, N], mode 1: [R_pad, N / 2]; twice as wide as a pair */
  const int32_t* rb_expert;    /* [R_pad/128] */
  const int32_t* rb_rows;      /* [R_pad/128], or NULL: every row is real */
  int64_t R_pad;
  int32_t mode;
  int32_t a_parts;             /* 1, or 2: A holds pairs (without gather_pull) */
  int32_t out_type;            /* 0 fp32, 1 bf16, 2 bf16 pair */
  const int32_t* gather_pull;  /* [R_pad, 3] or NULL */
  int64_t n_src_rows;          /* n_src_rows * K * 2 below 2 GiB */
  int32_t tokens_per_src, devs_per_node;
  const int64_t* sizes;        /* device {R, R_pad} or NULL */
} mk_moe_grouped_gemm_w4_args;
int mk_moe_grouped_gemm_w4(const mk_moe_grouped_gemm_w4_args* args, void* stream);

/* The local MoE layer with 4-bit expert weights: GEMM1 + SwiGLU (token rows
 * read through the pull table) -> GEMM2 -> combine, three launches.  The
 * activation goes as a bf16 pair (17 bits) and the expert rows in fp32, so
 * y_out's is the only rounding to 8 bits.  act and y_expert are written on real rows only.  act lies apart
 * from tokens, y_expert from act, y_out from y_expert (y_out may be tokens). */
typedef struct mk_moe_ffn_w4_args {
  const void* tokens;           /* bf16 [n_src_rows, H] */
  const int32_t* pull_indices;  /* [R_pad, 3] */
  const int32_t* rb_expert;     /* [R_pad/128] */
  const int32_t* rb_rows;       /* [R_pad/128], or NULL: every row is real */
  const float* row_weight;      /* [R_pad] */
  const int32_t* owner_offset;  /* [num_tokens + 1] */
  const int32_t* slot_to_row;   /* [R] */
  mk_w4_weights w1;             /* [E, H, 2I] (gate | up) */
  mk_w4_weights w2;             /* [E, I, H] */
  void* act;                    /* bf16 [R_pad, 2I] */
  void* y_expert;               /* fp32 [R_pad, H] */
  void* y_out;                  /* [num_tokens, H] fp32 or bf16 */
  int64_t num_tokens, n_src_rows, R_pad;
  int32_t tokens_per_src, devs_per_node;
  int32_t out_dtype;            /* 0 fp32, 1 bf16 */
  const int64_t* sizes;         /* device {R, R_pad} or NULL */
} mk_moe_ffn_w4_args;
int mk_moe_ffn_combine_w4(const mk_moe_ffn_w4_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* Dense products of any size with what follows them, and their gradients.
 *
 * Common to the entry points from here to mk_vocab_loss_backward: bf16
 * operands, fp32 sums, one rounding at the end.  Any sizes up to 2^25 rows (2^21
 * tokens of the loss) and row strides (of at least the row's width, at most 2^21
 * elements); operands aligned to their elements.  Operands whose rows do not start at 16-byte boundaries, or whose
 * rows' ends do not fill 16 bytes where the sum runs along them, are laid out
 * anew in the workspace first.  Results may not overlap what is read, unless
 * said otherwise.  Sums are added in an order that depends on sizes, on the
 * operands' alignment and strides and on the device's number of CUs, never on
 * timing.
 * `workspace`: mk_*_workspace_bytes(args) bytes, 16-byte aligned, holding
 * nothing between calls (the pointers in args have to be set for the question,
 * the workspace's own need not).  `tickets`: MK_PRODUCT_TICKETS 32-bit words,
 * zero before their first use, left zero by every call; launches that share
 * them must be ordered.  mk_*_ticket_words(args) is how many of them the call
 * touches: 0 where no sum is cut (any address but NULL will do then). */
#define MK_PRODUCT_TICKETS 8192

/* What lies between two products of a backward pass (dpre, dl) is held in bf16,
 * which one product takes, or as fp32's three bf16 parts (x rounded, the rest
 * rounded, the rest), a product each: three times the operations. */
#define MK_BETWEEN_RESULT 0 /* for each result as its own type: three parts for fp32 */
#define MK_BETWEEN_BF16 1
#define MK_BETWEEN_FP32 2

#define MK_ACT_NONE 0
#define MK_ACT_RELU 1
#define MK_ACT_GELU 2      /* x * Phi(x) */
#define MK_ACT_GELU_TANH 3 /* x/2 * (1 + tanh(sqrt(2/pi) * (x + 0.044715 x^3))) */
#define MK_ACT_SILU 4      /* x / (1 + e^-x) */

/* C = act(A @ B + bias) + residual; pre, where set, gets A @ B + bias (bf16) for
 * the backward pass.  residual may be C itself (same type and stride).  Where
 * nothing follows a bf16 product of whole tiles, mk_gemm is as fast or faster. */
typedef struct mk_gemm_act_args {
  const void* A;         /* bf16 [M, lda] */
  const void* B;         /* bf16 [K, ldb] */
  void* C;               /* [M, ldc] */
  const void* bias;      /* [N] or NULL */
  const void* residual;  /* [M, ldr] or NULL */
  void* pre;             /* bf16 [M, ldp] or NULL */
  int64_t M, N, K;
  int64_t lda, ldb, ldc, ldr, ldp;
  int32_t act;           /* MK_ACT_* */
  int32_t c_type, bias_type, residual_type; /* 0 fp32, 1 bf16 */
  void* workspace;
  int64_t workspace_bytes;
  void* tickets;
} mk_gemm_act_args;
int64_t mk_gemm_act_workspace_bytes(const mk_gemm_act_args* args);
int64_t mk_gemm_act_ticket_words(const mk_gemm_act_args* args);
int mk_gemm_act(const mk_gemm_act_args* args, void* stream);

/* Gradients of mk_gemm_act (the residual's is dC itself): with
 * dpre = dC * act'(pre),
 *   dA = dpre @ B^T (bf16),  dB = A^T @ dpre,  dbias = column sums of dpre (fp32).
 * Each of the three may be NULL.  pre is needed with an activation; `between`
 * says how dpre goes into the two products (matrix cores take nothing wider than
 * bf16 at their rate).  In bf16 each product is off by up to 2^-8 of itself
 * (4096 cubed, silu: error of bf16 dA and dB 0.0023 in norm, 0.0017 without),
 * which is thousands of times an fp32 result's own rounding.  dbias takes dpre as
 * it is; without an activation, and with relu, bf16 holds it exactly.
 * accumulate: dB and dbias are added to what they hold (gradients of several
 * batches). */
typedef struct mk_gemm_act_backward_args {
  const void* dC;        /* bf16 [M, lddc] */
  const void* A;         /* bf16 [M, lda]; needed for dB */
  const void* B;         /* bf16 [K, ldb]; needed for dA */
  const void* pre;       /* bf16 [M, ldp]; NULL with MK_ACT_NONE */
  void* dA;              /* bf16 [M, ldda] or NULL */
  void* dB;              /* [K, lddb] or NULL */
  float* dbias;          /* [N] or NULL */
  int64_t M, N, K;
  int64_t lddc, lda, ldb, ldp, ldda, lddb;
  int32_t act, db_type;  /* db_type 0 fp32, 1 bf16 */
  int16_t accumulate, between; /* MK_BETWEEN_* */
  void* workspace;
  int64_t workspace_bytes;
  void* tickets;
} mk_gemm_act_backward_args;
int64_t mk_gemm_act_backward_workspace_bytes(const mk_gemm_act_backward_args* args);
int64_t mk_gemm_act_backward_ticket_words(const mk_gemm_act_backward_args* args);
int mk_gemm_act_backward(const mk_gemm_act_backward_args* args, void* stream);

/* Expert products on ragged rows: the rows of expert e are the counts[e] rows
 * behind those of the experts before it (padded_tokens_per_expert of an index
 * build, at row_block 1 or any other).  Counts are read on the device; below 0
 * they count as 0, and rows from R on, which the counts may name, are not there.
 * Rows behind the last expert's are not written, and nothing that they hold is in
 * a result (where A is laid out anew they are copied with it).
 *   mode 0: out[r] = A[r] @ W[e]                        (out [R, N])
 *   mode 1: out[r] = silu(g) * u, (g | u) = A[r] @ W[e] (out [R, N/2]), and h,
 *           where set, gets (g | u) in bf16 [R, N] for the backward pass. */
typedef struct mk_moe_ragged_gemm_args {
  const void* A;          /* bf16 [R, lda] */
  const void* W;          /* bf16 [E, K, N] */
  const int32_t* counts;  /* [E] */
  void* out;              /* bf16 [R, ldo] */
  void* h;                /* bf16 [R, ldh] or NULL */
  int64_t R, K, N;
  int64_t lda, ldo, ldh;
  int32_t num_experts, mode;
  void* workspace;
  int64_t workspace_bytes;
} mk_moe_ragged_gemm_args;
int64_t mk_moe_ragged_gemm_workspace_bytes(const mk_moe_ragged_gemm_args* args);
int mk_moe_ragged_gemm(const mk_moe_ragged_gemm_args* args, void* stream);

/* Gradient of the rows: dA[r] = dy[r] @ W[e]^T ([R, K]); with h (that product's
 * A was silu(g) * u of it, h = (g | u) [R, 2K] as mode 1 gave it) the gradient of
 * h instead: out = dh [R, 2K], in one pass.  out may be h. */
typedef struct mk_moe_ragged_dgrad_args {
  const void* dy;         /* bf16 [R, lddy] */
  const void* W;          /* bf16 [E, K, N] */
  const int32_t* counts;  /* [E] */
  const void* h;          /* bf16 [R, ldh] or NULL */
  void* out;              /* bf16 [R, ldo] */
  int64_t R, K, N;
  int64_t lddy, ldh, ldo;
  int32_t num_experts;
  void* workspace;
  int64_t workspace_bytes;
} mk_moe_ragged_dgrad_args;
int64_t mk_moe_ragged_dgrad_workspace_bytes(const mk_moe_ragged_dgrad_args* args);
int mk_moe_ragged_dgrad(const mk_moe_ragged_dgrad_args* args, void* stream);

/* Gradient of the weights: dW[e] = A_e^T @ dy_e, zeros for an expert without
 * rows; accumulate: added to what dW holds. */
typedef struct mk_moe_ragged_wgrad_args {
  const void* A;          /* bf16 [R, lda] */
  const void* dy;         /* bf16 [R, lddy] */
  const int32_t* counts;  /* [E] */
  void* dW;               /* [E, K, N] */
  int64_t R, K, N;
  int64_t lda, lddy;
  int32_t num_experts;
  int32_t dw_type;        /* 0 fp32, 1 bf16 */
  int32_t accumulate;
  void* workspace;
  int64_t workspace_bytes;
} mk_moe_ragged_wgrad_args;
int64_t mk_moe_ragged_wgrad_workspace_bytes(const mk_moe_ragged_wgrad_args* args);
int mk_moe_ragged_wgrad(const mk_moe_ragged_wgrad_args* args, void* stream);

/* Cross entropy over a vocabulary, or one rank's shard [vocab_begin,
 * vocab_begin + V) of it, without keeping the logits x @ W: per token
 *   lse = log sum_v e^logit,  target = the label's logit (0 where another shard
 *   has it),  loss = lse - target.
 * Shards are joined by lse = log sum e^lse_i and the sum of the targets.  Tokens
 * whose label is ignore_index have zeros in all three, whatever their x holds (the
 * join of such zeros is for the caller to set to 0; the backward pass gives these
 * tokens zeros whatever their lse and dloss are). */
typedef struct mk_vocab_loss_args {
  const void* x;          /* bf16 [T, ldx] */
  const void* W;          /* bf16 [H, ldw] */
  const void* labels;     /* [T] int32 or int64 */
  float* lse;             /* [T] */
  float* target;          /* [T] */
  float* loss;            /* [T] or NULL */
  int64_t T, H, V;
  int64_t ldx, ldw;
  int64_t vocab_begin, ignore_index;
  int32_t labels_type;    /* 0 int32, 1 int64 */
  void* workspace;
  int64_t workspace_bytes;
  void* tickets;
} mk_vocab_loss_args;
int64_t mk_vocab_loss_workspace_bytes(const mk_vocab_loss_args* args);
int64_t mk_vocab_loss_ticket_words(const mk_vocab_loss_args* args);
int mk_vocab_loss(const mk_vocab_loss_args* args, void* stream);

/* Gradients: with dl = (e^(logit - lse) - [v = label]) * dloss (lse over all
 * shards), 0 for ignored tokens,
 *   dx = dl @ W^T (of a shard: its part of the sum),  dW = x^T @ dl.
 * Logits are computed anew, a piece of the vocabulary at a time (piece_columns, a
 * multiple of 256; 0: as many as keep dl in bf16 at 128 MB or less, at least 256);
 * dl goes through the workspace as
 * `between` says.  In bf16 each of its elements is off by up to 2^-8 of itself
 * (without the significand of the largest dloss, which the fp32 sums take back: of
 * a mean's equal dloss no common rounding stays; of several distinct ones, the
 * labels' elements of the others keep one each).  Either result may be NULL;
 * accumulate: dW is added to. */
typedef struct mk_vocab_loss_backward_args {
  const void* x;          /* bf16 [T, ldx] */
  const void* W;          /* bf16 [H, ldw] */
  const void* labels;
  const float* lse;       /* [T] */
  const float* dloss;     /* [T] */
  void* dx;               /* [T, lddx] or NULL */
  void* dW;               /* [H, lddw] or NULL */
  int64_t T, H, V;
  int64_t ldx, ldw, lddx, lddw;
  int64_t vocab_begin, ignore_index;
  int64_t piece_columns;
  int32_t labels_type, dx_type, dw_type; /* types 0 fp32, 1 bf16 */
  int16_t accumulate, between; /* MK_BETWEEN_* */
  void* workspace;
  int64_t workspace_bytes;
  void* tickets;
} mk_vocab_loss_backward_args;
int64_t mk_vocab_loss_backward_workspace_bytes(const mk_vocab_loss_backward_args* args);
int64_t mk_vocab_loss_backward_ticket_words(const mk_vocab_loss_backward_args* args);
int mk_vocab_loss_backward(const mk_vocab_loss_backward_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* K-split workspace size.  When the output tiles do not fill the last round
 * of the persistent grid (tiles % compute workgroups != 0), the GEMM entry
 * points split each tile of that tail round along K over 2-4 workgroups;
 * the parts exchange fp32 partial tiles and ready flags through `split_ws`.
 * This returns the bytes `split_ws` needs on the current device for any
 * shape and grid (4 KB of flag words plus one 256x256 fp32 tile per CU); `which`, M,
 * N and K are accepted for symmetry and do not change the answer.  A
 * workspace serves one launch at a time: launches that share it must be
 * ordered (same stream).  After a bounded wait gave up (bit 0 of the error
 * word) its first 4 KB must be zeroed before the next launch that uses it.  No counterpart in the reference, whose tail round
 * simply idles (src/ag_gemm.cu:265-461). */
int64_t mk_query_workspace_bytes(int32_t which, int64_t M, int64_t N, int64_t K);

/* Diagnostic, no counterpart in the reference (its benches price against
 * the published peak only): the MFMA throughput ceiling of the device under
 * sustained load.  num_wg workgroups of mk_probe_threads() threads each run
 * `iters` iterations of 16 independent v_mfma_f32_32x32x16_bf16 per wave
 * (32768 FLOP each) on random bf16 operands, no memory traffic.
 * sink: fp32 [num_wg * mk_probe_threads()] (keeps the work live);
 * clocks: u64 [num_wg * 2] = per workgroup (shader clock cycles, 100 MHz
 * constant-clock ticks) around the loop, whose ratio gives the engine clock
 * the matrix cores ran at.  Used by bench.py next to the roofline. */
int mk_probe_mfma_ceiling(int64_t iters, int32_t num_wg, float* sink, uint64_t* clocks, void* stream);
int32_t mk_probe_threads(void);

/* Number of compute units of the current device (0 if no device). */
int32_t mk_device_cu_count(void);

const char* mk_last_error_string(void);

/* Advances a device epoch word on the stream: *epoch_ptr += 1, skipping 0
 * (the value flags start at).  Recorded in a HIP graph before gated launches
 * that read epoch_ptr, it gives each replay a new epoch.  Device-side
 * counterpart of the reference's host epoch helpers (set_epoch /
 * prepare_epoch / commit_epoch, include/operators/ag_gemm/session.cuh:192-230). */
int mk_epoch_advance(uint32_t* epoch_ptr, void* stream);

/* ABI version, bumped on any signature change (2: split_ws fields; 4: MoE
 * `sizes`; 5: epoch_ptr; 6: mk_ag_gemm n_present, mk_moe_invert_slots owner
 * and slot capacity). */
int32_t mk_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* MK_H_ */

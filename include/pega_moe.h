/*
 * pega_moe.h -- C ABI of libpega_moe_hip.so, the MI355X (gfx950) quantized
 * MoE expert path (W4A16: INT4 group-32 symmetric weights, bf16 activations,
 * fp32 accumulation).
 *
 * Conventions (as in the reference's FFI, pegainfer-kernels/src/ffi/kimi.rs
 * and src/ffi.rs:5):
 *   - bf16 tensors are passed as uint16_t bit patterns;
 *   - all pointers are device pointers, caller-owned; no entry point
 *     allocates, synchronises or copies to the host;
 *   - `stream` is a hipStream_t (the reference passes a CUstream);
 *   - return value: 0 success, 1 invalid value, 801 not supported,
 *     719 launch failed (CUresult numbering); the reason for the last
 *     non-zero return on the calling thread is pegainfer_kernels_last_error().
 *
 * Entry points named kimi_* keep the reference's symbol names, argument order
 * and shape guards (48 local experts, top-8, group 32), so they are drop-in
 * replacements.  Entry points named pega_* have no reference counterpart:
 * they are the shape-general forms (any expert count / top-k) used for the
 * dense and DeepSeek-V2-Lite-shaped configurations, plus the routing select
 * stages the reference runs inside larger calls or on the host.
 */
#ifndef PEGA_MOE_H_
#define PEGA_MOE_H_

#include <stdbool.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* hipStream_t;

/* Reason for the last failure on this thread (never NULL).
 * Replaces: pegainfer_kernels_last_error, pegainfer-kernels/csrc/shared/ffi_last_error.cu:13 */
const char* pegainfer_kernels_last_error(void);

/* ---------------- token -> expert permutation ---------------- */

/* Replaces kimi_moe_marlin_align_block_size_cuda, pegainfer-kernels/src/ffi/kimi.rs:279-294
 * (csrc/kimi_k2/kimi_experts.cu:197-268).  Deterministic for every route count. */
int kimi_moe_marlin_align_block_size_cuda(const int32_t* topk_idx, int32_t* sorted_token_ids,
                                          int32_t* expert_ids, int32_t* num_tokens_post_padded,
                                          uint32_t* expert_offsets, uint32_t* expert_cursor,
                                          int active_tokens, int topk, int global_start,
                                          int local_experts, int block_size,
                                          int max_padded_tokens, int max_m_blocks,
                                          hipStream_t stream);

/* No reference counterpart: shape-general form of the call above (local_experts <= 512,
 * any topk). */
int pega_moe_align_block_size(const int32_t* topk_idx, int32_t* sorted_token_ids,
                              int32_t* expert_ids, int32_t* num_tokens_post_padded,
                              uint32_t* expert_offsets, uint32_t* expert_cursor,
                              int active_tokens, int topk, int global_start, int local_experts,
                              int block_size, int max_padded_tokens, int max_m_blocks,
                              hipStream_t stream);

/* Replaces kimi_deepep_build_marlin_routing_on_stream, pegainfer-kernels/src/ffi/kimi.rs:296-307
 * (csrc/kimi_k2/kimi_experts.cu:435-459). */
int kimi_deepep_build_marlin_routing_on_stream(const int32_t* psum_expert,
                                               int32_t* sorted_token_ids, int32_t* expert_ids,
                                               int32_t* num_tokens_post_padded,
                                               int num_local_experts, int alignment,
                                               int block_size, int max_padded_tokens,
                                               int max_m_blocks, hipStream_t stream);

/* ---------------- load-time weight packaging (Marlin layout, bit-exact) ---------------- */

/* Replaces kimi_marlin_int4_reorder_weight_cuda, pegainfer-kernels/src/ffi/kimi.rs:93-101. */
int kimi_marlin_int4_reorder_weight_cuda(const uint8_t* weight_packed_checkpoint,
                                         uint8_t* weight_packed_marlin, int in_dim, int out_dim,
                                         int local_experts, int group_size, hipStream_t stream);

/* Replaces kimi_marlin_int4_reorder_scale_cuda, pegainfer-kernels/src/ffi/kimi.rs:84-91. */
int kimi_marlin_int4_reorder_scale_cuda(const uint16_t* weight_scale_checkpoint,
                                        uint16_t* weight_scale_marlin, int in_dim, int out_dim,
                                        int local_experts, int group_size, hipStream_t stream);

/* Replaces kimi_marlin_int4_fuse_w13_cuda, pegainfer-kernels/src/ffi/kimi.rs:68-82. */
int kimi_marlin_int4_fuse_w13_cuda(const uint8_t* gate_weight_packed_marlin,
                                   const uint8_t* up_weight_packed_marlin,
                                   uint8_t* w13_weight_packed_marlin,
                                   const uint16_t* gate_scale_marlin,
                                   const uint16_t* up_scale_marlin, uint16_t* w13_scale_marlin,
                                   int in_dim, int intermediate_dim, int local_experts,
                                   int group_size, hipStream_t stream);

/* No reference counterpart: the three calls above for any expert count. */
int pega_marlin_int4_reorder_weight(const uint8_t* ckpt, uint8_t* marlin, int in_dim,
                                    int out_dim, int local_experts, int group_size,
                                    hipStream_t stream);
int pega_marlin_int4_reorder_scale(const uint16_t* ckpt, uint16_t* marlin, int in_dim,
                                   int out_dim, int local_experts, int group_size,
                                   hipStream_t stream);
int pega_marlin_int4_fuse_w13(const uint8_t* gate_w, const uint8_t* up_w, uint8_t* w13_w,
                              const uint16_t* gate_s, const uint16_t* up_s, uint16_t* w13_s,
                              int in_dim, int intermediate_dim, int local_experts,
                              int group_size, hipStream_t stream);

/* ---------------- grouped W4A16 GEMM ---------------- */

/* Replaces kimi_marlin_wna16_gemm_cuda, pegainfer-kernels/src/ffi/kimi.rs:131-152
 * (csrc/kimi_k2/kimi_marlin_wna16.cu:241-343,414-442).  c_tmp and workspace (locks) are
 * required as in the reference but not accessed: K is split inside each workgroup. */
int kimi_marlin_wna16_gemm_cuda(const uint16_t* input, uint16_t* output, float* c_tmp,
                                const uint8_t* b_qweight, const uint16_t* b_scales,
                                int32_t* workspace, const int32_t* sorted_token_ids,
                                const int32_t* expert_ids, const int32_t* num_tokens_post_padded,
                                const float* topk_weights, int workspace_len,
                                int sorted_token_ids_len, int moe_block_size, int top_k,
                                bool mul_topk_weights, int size_m, int size_n, int size_k,
                                int local_experts, int group_size, int sm_count,
                                hipStream_t stream);

/* No reference counterpart: shape-general form (any expert count; c_tmp / workspace unused
 * and may be NULL). */
int pega_wna16_gemm(const uint16_t* input, uint16_t* output, float* c_tmp, long long c_tmp_len,
                    const uint8_t* b_qweight, const uint16_t* b_scales, int32_t* workspace,
                    int workspace_len, const int32_t* sorted_token_ids, const int32_t* expert_ids,
                    const int32_t* num_tokens_post_padded, const float* topk_weights,
                    int sorted_token_ids_len, int moe_block_size, int top_k,
                    bool mul_topk_weights, int size_m, int size_n, int size_k, int local_experts,
                    int group_size, int sm_count, hipStream_t stream);

/* No reference counterpart: W13 GEMM fused with SwiGLU.  The reference runs
 * kimi_marlin_wna16_gemm_cuda (W13, top_k rows) then kimi_marlin_w13_swiglu_cuda over every
 * route row; here act = [size_m * top_k, intermediate_dim] bf16 gets SwiGLU of the W13 sums
 * rounded to bf16 as the W13 output is, for the routed rows only (other rows are left as they
 * are), and the W13 output never reaches HBM.  The bits are the pair's whenever both add the
 * fp32 products over the same K shares: always at block sizes 32-64 (both take the same form
 * and the same split of K), and at block sizes 8/16 when there are at least two (block, 64-column
 * tile) units per CU, counting a block per route, and K is at least 512.
 * Otherwise the shares differ, and the sums may differ from the pair's in the last fp32 bit,
 * within the same summation error bound.
 *  - Block size 8 or 16 (decode): when the (block, tile) units are too few to fill the GPU
 *    (one expert at batch 1-8), K is split across workgroups; the fp32 partials (partials:
 *    at least 2 * size_m * top_k * 2 * intermediate_dim floats for a split, more allows more
 *    shares) are summed in share order by the SwiGLU kernel, which rounds gate and up to bf16
 *    exactly as the W13 output is rounded.  Otherwise (or when partials is NULL or too small
 *    to split) a workgroup takes a gate tile and its up tile and applies SwiGLU in its
 *    epilogue.
 *  - Block size 32, 48 or 64 (prefill): the tile GEMM (128-row tiles, or 64-row tiles when
 *    the routes are few per expert), or where they are fewer still a 32-row form of the decode
 *    kernel, takes each gate tile and its up tile in one workgroup and applies SwiGLU in its
 *    epilogue; partials is not used (may be NULL, partials_len 0). */
int pega_wna16_w13_swiglu(const uint16_t* input, uint16_t* act, float* partials,
                          long long partials_len, const uint8_t* b_qweight,
                          const uint16_t* b_scales, const int32_t* sorted_token_ids,
                          const int32_t* expert_ids, const int32_t* num_tokens_post_padded,
                          int sorted_token_ids_len, int moe_block_size, int top_k, int size_m,
                          int intermediate_dim, int size_k, int local_experts, int group_size,
                          int sm_count, hipStream_t stream);

/* The same where the experts are one GPU's of ep_size (at least 1, which is the entry above)
 * that the routes are spread over: the launch rules then expect one route in ep_size to be
 * local.  The outputs are the entry's above, bit for bit.
 * kimi_marlin_wna16_gemm_cuda, whose 48 experts are one GPU's of eight, expects that by
 * itself; pega_wna16_gemm takes every route to be local, and so do both for an expert-major
 * launch (sorted_token_ids_len <= size_m * top_k). */
int pega_wna16_w13_swiglu_ep(const uint16_t* input, uint16_t* act, float* partials,
                             long long partials_len, const uint8_t* b_qweight,
                             const uint16_t* b_scales, const int32_t* sorted_token_ids,
                             const int32_t* expert_ids, const int32_t* num_tokens_post_padded,
                             int sorted_token_ids_len, int moe_block_size, int top_k, int size_m,
                             int intermediate_dim, int size_k, int local_experts, int ep_size,
                             int group_size, int sm_count, hipStream_t stream);

/* No reference counterpart; for callers that cannot allocate (code under HIP graph capture,
 * serving loops and harnesses that forbid hipMalloc): pega_wna16_w13_swiglu without the
 * partials workspace.  The K-split partials go to the library's static per-device scratch
 * (2 MiB = 524,288 floats, held until the process ends; its device address is looked up once
 * per device on the first call there).  Nothing in it needs clearing: every routed row of
 * every K share is written before the SwiGLU kernel reads it.  Calls that overlap on one
 * device race on the scratch.  The output is pega_wna16_w13_swiglu's with a partials
 * workspace of the scratch's size (partials_len = 524,288): the share count is capped by
 * what the scratch holds, and a wanted K split it cannot hold two shares of runs unsplit, as
 * the workspace entry does with a small workspace.  The current device must own `stream`
 * (status 1 otherwise). */
int pega_wna16_w13_swiglu_noalloc(const uint16_t* input, uint16_t* act, const uint8_t* b_qweight,
                                  const uint16_t* b_scales, const int32_t* sorted_token_ids,
                                  const int32_t* expert_ids, const int32_t* num_tokens_post_padded,
                                  int sorted_token_ids_len, int moe_block_size, int top_k,
                                  int size_m, int intermediate_dim, int size_k, int local_experts,
                                  int group_size, int sm_count, hipStream_t stream);

/* One problem of pega_wna16_prefill_pair: a grouped INT4 GEMM at a prefill block size (the
 * tile kernel), as pega_wna16_gemm (act NULL) or pega_wna16_w13_swiglu (act set) would run
 * it.  Plain pointers and sizes; 112 bytes on LP64. */
typedef struct pega_wna16_problem {
    const uint16_t* input;                /* bf16 [size_m, size_k], 16-byte aligned */
    uint16_t* output;                     /* bf16 [size_m * top_k, size_n] (unused with act) */
    uint16_t* act;                        /* non-NULL: SwiGLU epilogue into bf16
                                             [size_m * top_k, size_n / 2] */
    const uint8_t* b_qweight;             /* device-layout INT4 weights [local_experts] */
    const uint16_t* b_scales;             /* device-layout bf16 scales */
    const int32_t* sorted_token_ids;      /* the permutation of this problem's routes */
    const int32_t* expert_ids;
    const int32_t* num_tokens_post_padded;
    const float* topk_weights;            /* read only with mul_topk_weights */
    int sorted_token_ids_len;
    int moe_block_size;                   /* 32, 48 or 64 */
    int top_k;
    int mul_topk_weights;                 /* 0 or 1 (0 with act) */
    int size_m;
    int size_n;                           /* with act: 2 * intermediate_dim, gate then up */
    int size_k;
    int local_experts;
    int group_size;                       /* 32 */
} pega_wna16_problem;

/* No reference counterpart: two independent prefill-size GEMMs in one launch, e.g. a layer's
 * shared expert (first) and its routed experts (second).  The workgroups of the first problem
 * are dispatched first, and the second problem's fill the rest of the GPU, so one stream keeps
 * both running at once; each problem's output has the bits its own single launch gives.  When
 * a problem has too few routed rows for the tile kernel, each gets its own launch instead.
 * Returns 801 when a problem's block size is 8 or 16 (the decode kernels). */
int pega_wna16_prefill_pair(const pega_wna16_problem* first, const pega_wna16_problem* second,
                            hipStream_t stream);

/* ---------------- activation / combine / residual ---------------- */

/* Replaces kimi_marlin_w13_swiglu_cuda, pegainfer-kernels/src/ffi/kimi.rs:113-119. */
int kimi_marlin_w13_swiglu_cuda(const uint16_t* w13, uint16_t* out, int rows,
                                int intermediate_dim, hipStream_t stream);

/* Replaces kimi_marlin_w13_swiglu_expanded_cuda, pegainfer-kernels/src/ffi/kimi.rs:121-129. */
int kimi_marlin_w13_swiglu_expanded_cuda(const uint16_t* w13, uint16_t* out,
                                         const int32_t* num_tokens_post_padded, int max_rows,
                                         int intermediate_dim, int sm_count, hipStream_t stream);

/* Replaces kimi_marlin_sum_topk_rows_f32_cuda, pegainfer-kernels/src/ffi/kimi.rs:104-111. */
int kimi_marlin_sum_topk_rows_f32_cuda(const uint16_t* route_output, float* out,
                                       int active_tokens, int topk, int hidden_dim,
                                       hipStream_t stream);

/* No reference C symbol: the DeepSeek-V2-Lite weighted fp32 combine (fmaf chain in route
 * order), restating pegainfer-kernels/csrc/deepseek_v2_lite/dsv2_lite_moe.cu:131-155. */
int pega_weighted_topk_sum_f32(const uint16_t* route_output, const float* topk_weight,
                               float* out, int active_tokens, int topk, int hidden_dim,
                               hipStream_t stream);

/* No reference counterpart: the top-k combine over the routes this GPU owns only
 * (topk_idx - global_start in [0, local_experts)); the other rows of route_output are not
 * read, so the caller skips their zero-fill (moe_nccl.rs:186-188).  topk_weight NULL: plain
 * sum as kimi_marlin_sum_topk_rows_f32_cuda; non-NULL: fmaf chain as
 * pega_weighted_topk_sum_f32.  Equal bit for bit to zero-filling the skipped rows and calling
 * those (for finite weights).  hidden_dim % 8 == 0, 16-byte aligned buffers. */
int pega_moe_combine_local_f32(const uint16_t* route_output, const int32_t* topk_idx,
                               const float* topk_weight, float* out, int active_tokens, int topk,
                               int hidden_dim, int global_start, int local_experts,
                               hipStream_t stream);

/* Replaces kimi_residual_add_scaled_f32_cuda, pegainfer-kernels/src/ffi/kimi.rs:309-317. */
int kimi_residual_add_scaled_f32_cuda(const uint16_t* hidden, const uint16_t* projected,
                                      const float* routed_f32, float scale, uint16_t* out, int n,
                                      hipStream_t stream);

/* Replaces kimi_residual_add_scaled_bf16_cuda, pegainfer-kernels/src/ffi/kimi.rs:319-327. */
int kimi_residual_add_scaled_bf16_cuda(const uint16_t* hidden, const uint16_t* projected,
                                       const uint16_t* routed, float scale, uint16_t* out, int n,
                                       hipStream_t stream);

/* Replaces kimi_add_f32_bf16_to_bf16_cuda, pegainfer-kernels/src/ffi/kimi.rs:9-15. */
int kimi_add_f32_bf16_to_bf16_cuda(const float* a, const uint16_t* b, uint16_t* out, int n,
                                   hipStream_t stream);

/* Replaces f32_to_bf16_cuda, pegainfer-kernels/src/ffi/shared.rs:849-854
 * (csrc/shared/elementwise.cu:235-244,722-728): out = bf16(input), round to nearest even. */
int f32_to_bf16_cuda(const float* input, uint16_t* output, int n, hipStream_t stream);

/* Replaces add_cuda, pegainfer-kernels/src/ffi/shared.rs:27-33
 * (csrc/shared/elementwise.cu:9-21,500-507): out = bf16(f(a) + f(b)). */
int add_cuda(const uint16_t* a, const uint16_t* b, uint16_t* out, int n, hipStream_t stream);

/* No reference symbol of its own: the DeepSeek-V2-Lite routed + shared join,
 * f32_to_bf16_cuda(routed) then add_cuda(., shared) as
 * pegainfer-deepseek-v2-lite/src/nccl_backend.rs:544-545 and runtime/moe.rs:656 run them,
 * in one pass with the same two roundings: out = bf16(f(bf16(routed)) + f(shared)). */
int pega_moe_join_routed_shared_bf16(const float* routed, const uint16_t* shared, uint16_t* out,
                                     int n, hipStream_t stream);

/* No reference symbol of its own: pega_moe_combine_local_f32 then
 * pega_moe_join_routed_shared_bf16 in one pass, for a layer whose routed sum needs no
 * reduction across GPUs between the two (one GPU holds every routed expert):
 * out[t] = bf16(f(bf16(combine_t)) + f(shared[t])), where combine_t is the fp32 sum (topk_weight
 * NULL) or fmaf chain over the token's local routes, k ascending from +0 -- the same bits as
 * the two calls.  hidden_dim % 8 == 0, 16-byte aligned buffers. */
int pega_moe_combine_join_bf16(const uint16_t* route_output, const int32_t* topk_idx,
                               const float* topk_weight, const uint16_t* shared, uint16_t* out,
                               int active_tokens, int topk, int hidden_dim, int global_start,
                               int local_experts, hipStream_t stream);

/* ---------------- dense bf16 GEMM (shared expert) ----------------
 * Y[n][m] = bf16(sum_k W[m][k] * X[n][k]) with fp32 accumulation; W [M][K],
 * X [N][K], Y [N][M] bf16 row-major (the reference's cublasGemmEx(OP_T, OP_N)
 * call, pegainfer-kernels/csrc/shared/linear.cu:321-344).  Needs M % 16 == 0,
 * K % 32 == 0 and 16-byte aligned W and X (801 otherwise).  Never allocates. */

/* Replaces gemm_cuda, pegainfer-kernels/src/ffi/shared.rs:220-228. */
int gemm_cuda(const uint16_t* W, const uint16_t* X, uint16_t* Y, int M, int N, int K,
              hipStream_t stream);

/* Replaces gemm_graphsafe_cuda, pegainfer-kernels/src/ffi/shared.rs:230-238. */
int gemm_graphsafe_cuda(const uint16_t* W, const uint16_t* X, uint16_t* Y, int M, int N, int K,
                        hipStream_t stream);

/* No reference symbol of its own: gemm_graphsafe_cuda on the shared expert's gate/up weights
 * W13 [2 inter][K] (gate rows first) followed by kimi_marlin_w13_swiglu_cuda on its bf16 output,
 * as pegainfer-kimi-k2/src/runner/moe_nccl.rs:107-123 runs them, in one launch with the same
 * bits: act[n][j] = SwiGLU(bf16 gate sum, bf16 up sum).  X [N][K], act [N][inter].  Needs
 * inter % 16 == 0, K % 32 == 0 and 16-byte aligned W13 and X (801 otherwise).  Never
 * allocates. */
int pega_dense_w13_swiglu(const uint16_t* W13, const uint16_t* X, uint16_t* act, int inter, int N,
                          int K, hipStream_t stream);

/* ---------------- a whole MoE layer for a few tokens ---------------- */

enum { PEGA_SHARED_NONE = 0, PEGA_SHARED_BF16 = 1, PEGA_SHARED_INT4 = 2 };
enum { PEGA_FEW_MAX_SPLITS = 8, PEGA_FEW_COUNTERS = 512 };

/* Arguments of pega_moe_few_tokens.  INT4 weights are device packages (the layout of
 * pega_marlin_int4_*; W13 gate columns first).  Plain pointers and sizes; 224 bytes on LP64. */
typedef struct pega_moe_few {
    const uint16_t* x;           /* bf16 [tokens][hidden_dim], the normed rows */
    const float* logits;         /* router logits [tokens][n_experts] */
    const float* bias;           /* score correction [n_experts]; unused with softmax */
    const uint8_t* w13;          /* [local_experts] INT4 gate and up */
    const uint16_t* w13_scales;
    const uint8_t* w2;           /* [local_experts] INT4 down */
    const uint16_t* w2_scales;
    const void* shared_w13;      /* bf16 [2 shared_inter][hidden_dim], or an INT4 package */
    const uint16_t* shared_w13_scales; /* INT4 only */
    const void* shared_w2;       /* bf16 [hidden_dim][shared_inter], or an INT4 package */
    const uint16_t* shared_w2_scales;  /* INT4 only */
    const uint16_t* residual;    /* bf16 [tokens][hidden_dim] or NULL */
    uint16_t* out;               /* bf16 [tokens][hidden_dim]; may be residual's or x's buffer */
    float* topk_weight;          /* out: [tokens][topk] */
    int32_t* topk_idx;           /* out: [tokens][topk] */
    uint16_t* act;               /* workspace: fp16 [min(tokens topk, local_experts)][tokens][inter] */
    float* act_factors;          /* workspace: [min(tokens topk, local_experts)][inter / 64][16] */
    uint16_t* act_shared;        /* workspace: fp16 or bf16 [tokens][shared_inter] */
    float* act_shared_factors;   /* workspace, with an INT4 shared expert: [shared_inter / 64][16] */
    int32_t* slots;              /* workspace: 1 + min(tokens topk, local_experts) */
    float* partials;             /* workspace: tokens times the larger of PEGA_FEW_MAX_SPLITS *
                                    hidden_dim and 128 * PEGA_FEW_COUNTERS */
    uint32_t* counters;          /* workspace: hidden_dim / 64 + PEGA_FEW_COUNTERS, zero before the
                                    first call; every call leaves them zero */
    float route_scale;           /* of the sigmoid select (> 0); unused with softmax */
    float routed_scale;          /* factor of the routed sum */
    int softmax;                 /* 0: pega_kimi_router_select, 1: pega_dsv2_router_select */
    int shared_kind;             /* PEGA_SHARED_* */
    int tokens;                  /* 1 to 16 */
    int hidden_dim, inter, shared_inter; /* multiples of 64 */
    int n_experts, local_experts, global_start, topk;
} pega_moe_few;

/* No reference counterpart as one call: an MoE decode layer for a few tokens in two launches.
 *   topk_idx, topk_weight = the select entry's, bit for bit;
 *   out[t] = bf16(residual[t] + routed_scale * sum over t's local routes of weight *
 *            (silu(x G_e^T) * (x U_e^T)) D_e^T + the shared expert's rows).
 * INT4 weights count as (nibble - 8) * scale unrounded; x goes into the INT4 products exactly down to
 * 2^-25 of its row's largest magnitude (to 2^-40 of it below); the SwiGLU rows, times weight and
 * routed_scale, are rounded once to fp16 with a scale for each 64 (bf16 in front of a bf16 down
 * projection, whose products take bf16 rows), out once, and all sums are fp32, in an order that the
 * sizes and the routing decide.  A row of x with an infinity or a NaN gives NaN wherever an INT4 expert
 * takes it; what takes no part (an expert that is not local, no shared expert) leaves its residual as it
 * is, a bf16 shared expert gives what fp32 gives, and other rows are as without it.  Experts without a
 * route are not read.  Calls that share a workspace must not overlap (two captured graphs that may run
 * at once need one each); nothing is kept in it from one call to the next but the zeroed counters.
 * topk_weight and topk_idx are apart from every input and from out, and out from what the second launch
 * reads (residual, unless it is out itself, and the down projections).  At most 16 tokens, topk 32, 512
 * local experts, 1024 experts, sizes multiples of 64, 2 hidden_dim (2 inter + 16) bytes under 2 GiB for
 * the larger of inter and shared_inter, 16-byte aligned buffers (801 otherwise). */
int pega_moe_few_tokens(const pega_moe_few* args, hipStream_t stream);

/* ---------------- residual add + norm ---------------- */

/* No reference counterpart as one symbol: the residual add and the root-mean-square norm between
 * two blocks, for rows [rows][hidden_dim]:
 *   s = residual + x (x alone where residual is NULL); residual_out = bf16(s);
 *   y = s * weight / sqrt(mean(s^2) + eps); normed = bf16(y); mxfp8_codes / mxfp8_scales = y in
 *   MXFP8 (below).
 * x is bf16, or fp32 with x_is_f32.  Each output may be NULL, not all of them; codes and scales go
 * together.  An output may be the buffer of x or of residual (its first byte the input's); no two
 * outputs may overlap.  The sums and products are in 64 bits, and every output is their value
 * rounded once (y past fp32's range is an infinity); y is the norm of s itself, not of bf16(s).  A
 * row's result does not depend on the other rows.  hidden_dim % 8 == 0
 * (32 with MXFP8), at most 32768; 16-byte aligned buffers, scales 4-byte (801 otherwise). */
int pega_add_rmsnorm(const void* x, bool x_is_f32, const uint16_t* residual,
                     const uint16_t* weight, double eps, uint16_t* residual_out,
                     uint16_t* normed, uint8_t* mxfp8_codes, uint8_t* mxfp8_scales, int rows,
                     int hidden_dim, hipStream_t stream);

/* No reference counterpart: what stands between two blocks that are normed on both sides, for rows
 * [rows][hidden_dim]:
 *   y = x * post_weight / sqrt(mean(x^2) + eps)         (x itself where post_weight is NULL)
 *   s = residual_scale * residual + gate * y            (gate * y where residual is NULL)
 *   z = s * pre_weight / sqrt(mean(s^2) + eps)
 *   residual_out = bf16(s); normed = bf16(z); mxfp8_codes / mxfp8_scales = z in MXFP8 (below).
 * gate_kind 0: no gate; 1: bf16 [hidden_dim], one for each column; 2: bf16 [rows], one for each row;
 * 3: bf16 [rows][hidden_dim].  With unit_offset the weights are stored less one: 1 + post_weight and
 * 1 + pre_weight are meant.  pre_weight may be NULL where residual_out alone is asked for.  What
 * pega_add_rmsnorm says of x, of the outputs, of their places, of rounding and of sizes holds here; no
 * output may overlap the gate or a weight. */
int pega_sandwich_rmsnorm(const void* x, bool x_is_f32, const uint16_t* residual,
                          double residual_scale, const uint16_t* post_weight, const uint16_t* gate,
                          int gate_kind, const uint16_t* pre_weight, bool unit_offset, double eps,
                          uint16_t* residual_out, uint16_t* normed, uint8_t* mxfp8_codes,
                          uint8_t* mxfp8_scales, int rows, int hidden_dim, hipStream_t stream);

/* ---------------- dense products with 4-bit weights ----------------
 * Weights [out_dim][in_dim] of 4-bit codes q with a bf16 scale s, and where `zeros` is given a zero
 * point z, for each group of 32, 64 or 128 columns: (q - z) * s, z = 8 without zero points. */

/* No reference counterpart: a checkpoint's weight into the device layout of pega_w4_gemm.
 * packed [out_dim][in_dim / 2] bytes, the even column in the low nibble; scales bf16
 * [out_dim][in_dim / group_size]; zeros bytes of the same shape, 0 to 127, or NULL.  codes takes
 * ceil(out_dim / 16) * ceil(in_dim / 128) * 1024 bytes, meta the same number of units of
 * 16 * 128 / group_size * (zeros ? 4 : 2) bytes.  in_dim is whole groups, at most 2^20, out_dim at most
 * 2^26.  packed is
 * 4-byte aligned, codes and meta 16-byte (801 otherwise). */
int pega_w4_pack(const uint8_t* packed, const uint16_t* scales, const uint8_t* zeros,
                 uint8_t* codes, uint8_t* meta, int out_dim, int in_dim, int group_size,
                 hipStream_t stream);

/* No reference counterpart: Y[n][m] = sum_k X[n][k] * (q[m][k] - z[m][k / g]) * s[m][k / g], X [N][K]
 * bf16, Y [N][M] bf16 or, with y_is_f32, fp32; any M, N and whole groups of K.  No weight is
 * rounded: products with the codes' integers are exact, group sums and their products with the scales
 * fp32: the error is relative to sum |x| (16 + q + 16 + z) |s|.  A row of X with an infinity or a NaN
 * gives NaN; one with finite values of 2^117 and more may (2^119 where no zero point is above 15).  A
 * row's result does not depend on the other rows' values.  No workspace.  At most 2^20 columns, 2^26 features and
 * 1048560 rows; X, codes and meta 16-byte aligned, Y by its type (801 otherwise); Y overlaps no input. */
int pega_w4_gemm(const uint8_t* codes, const uint8_t* meta, bool has_zeros, int group_size,
                 const uint16_t* X, void* Y, bool y_is_f32, int M, int N, int K,
                 hipStream_t stream);

/* ---------------- next tokens ---------------- */

/* No reference counterpart: a token for each row of logits (fp32, or bf16 with logits_bf16), rows
 * row_stride elements apart:
 *   w[v] = e^((l[v] - max l) / temperature); zero where that is below e^-28 or below min_p
 *   of these the first top_k by logit (ties to the lower index) keep their weight;
 *   of these, in that order, the ones with less than top_p of their sum before them;
 *   token = the first v in index order with w[0] + .. + w[v] > uniform * (sum of w), and
 *   logprob = ln(w[token] / sum of w).
 * temperature, top_k, top_p, min_p: one value a row, or NULL (1, all, 1, 0).  temperature <= 0 takes
 * the largest logit; top_k <= 0 and top_p >= 1 leave all; the first token of the order always stays.
 * uniform is in [0, 1) (1 and more take the last kept token).  NaN logits count as -inf and are never
 * drawn; +inf ones share all weight; a row without any other logit than -inf gives token -1 and
 * logprob -inf.  Weights are rounded to 2^-44 once and summed exactly, so a row's result depends
 * on its own inputs alone.  vocab at most 2^19 (801 above).  workspace: 16-byte aligned, at least
 * pega_sample_workspace_bytes(rows, vocab) bytes, for one call at a time; it keeps nothing from one
 * call to the next.  logprobs may be NULL.  No output overlaps another or an input. */
int pega_sample_tokens(const void* logits, bool logits_bf16, long long row_stride, int rows,
                       int vocab, const float* uniform, const float* temperature,
                       const int32_t* top_k, const float* top_p, const float* min_p,
                       int32_t* tokens, float* logprobs, void* workspace,
                       long long workspace_bytes, hipStream_t stream);

/* The workspace that pega_sample_tokens needs for up to `rows` rows of up to `vocab` logits. */
long long pega_sample_workspace_bytes(int rows, int vocab);

/* ---------------- microscaled formats (MXFP8, MXFP4) ----------------
 * 32 consecutive values of a row share a scale 2^s, stored as the byte s + 127 (255: NaN).
 * format 0: E4M3 codes [rows][cols] bytes; format 1: E2M1 codes [rows][cols / 2] bytes, the even
 * column in the low nibble; scales [rows][cols / 32] bytes.  Quantisation takes the smallest s >=
 * -127 for which the block's largest magnitude rounds to a value of the format (at most 464 * 2^s
 * in E4M3, below 7 * 2^s in E2M1) and rounds to nearest, ties to even; a block with an infinity or
 * a NaN gets scale 255 and codes 0.  cols % 32 == 0; bf16 rows and codes 16-byte aligned, scales
 * 4-byte (801 otherwise).  No reference counterpart. */

/* bf16 rows [rows][cols] into codes and scales. */
int pega_mx_quantize(const uint16_t* x, uint8_t* codes, uint8_t* scales, int format, int rows,
                     int cols, hipStream_t stream);

/* kimi_marlin_w13_swiglu_cuda's bf16 values (w13 [rows][2 intermediate_dim], gate then up) into
 * codes and scales [rows][intermediate_dim], in one pass. */
int pega_mx_swiglu_quantize(const uint16_t* w13, uint8_t* codes, uint8_t* scales, int format,
                            int rows, int intermediate_dim, hipStream_t stream);

/* The values that codes and scales stand for, as bf16 [rows][cols] (exact down to bf16's smallest
 * numbers). */
int pega_mx_dequantize(const uint8_t* codes, const uint8_t* scales, uint16_t* out, int format,
                       int rows, int cols, hipStream_t stream);

/* Y[n][m] = bf16(sum_k X[n][k] * W[m][k]): W [M][K] MXFP4, X [N][K] in x_format, Y [N][M] bf16,
 * fp32 accumulation on the scaled matrix instructions (E4M3 products are aligned to the largest of
 * 128 inside an instruction: about 2^-12 of it).  M % 16 == 0, M below 2^28, K % 128 == 0, K below
 * 2^23, codes and Y 16-byte aligned, scales 4-byte, N at most 2^21 - 32 (801 otherwise), Y apart from
 * the operands (1).
 * Never allocates.  A call's bits depend on its sizes and formats alone; a block of scale 255
 * makes its row's results NaN. */
int pega_mx_gemm(const uint8_t* w_codes, const uint8_t* w_scales, const uint8_t* x_codes,
                 const uint8_t* x_scales, int x_format, uint16_t* Y, int M, int N, int K,
                 hipStream_t stream);

/* pega_wna16_gemm on microscaled operands: for every block b < ntp / block size of expert e =
 * expert_ids[b] in [0, local_experts) and every row sid of it below size_m * top_k,
 *   output[sid] = bf16(X[sid / top_k] . W[e]^T)          W [local_experts][size_n][size_k] MXFP4
 * times topk_weights[sid] before the rounding with mul_topk_weights (may be NULL otherwise).
 * Other rows of output [size_m * top_k][size_n] are left as they are.  ep_size (at least 1): GPUs
 * that the routes' experts are spread over, for the launch rules alone, which expect one route in
 * ep_size to be local; they choose the order of the fp32 sums, nothing else.  Block sizes 8, 16, 32, 48,
 * 64, at most 65535 of them; the rules of pega_mx_gemm; X under 2 GiB (801 otherwise). */
int pega_mx_grouped_gemm(const uint8_t* x_codes, const uint8_t* x_scales, int x_format,
                         uint16_t* output, const uint8_t* w_codes, const uint8_t* w_scales,
                         const int32_t* sorted_token_ids, const int32_t* expert_ids,
                         const int32_t* num_tokens_post_padded, const float* topk_weights,
                         int sorted_token_ids_len, int moe_block_size, int top_k,
                         bool mul_topk_weights, int size_m, int size_n, int size_k,
                         int local_experts, int ep_size, hipStream_t stream);

/* ---------------- routing select ---------------- */

/* Replaces kimi_k2_router_noaux_tc_cuda, pegainfer-kernels/src/ffi/kimi.rs:52-66
 * (csrc/kimi_k2/kimi_router.cu:108-187): logits [padded_tokens][n_experts] fp32 =
 * hidden [padded_tokens][hidden_dim] . gate_weight [n_experts][hidden_dim]^T (fp32
 * accumulation), then the select stage below over the first active_tokens rows.  Same
 * rejections as the reference (1: null pointers, token counts, n_experts != 384,
 * topk != 8, route_scale <= 0); 801 when hidden_dim % 32 != 0 or hidden / gate_weight are
 * not 16-byte aligned. */
int kimi_k2_router_noaux_tc_cuda(const uint16_t* hidden, const uint16_t* gate_weight,
                                 const float* e_score_correction_bias, float* logits,
                                 float* topk_weight, int32_t* topk_idx, int active_tokens,
                                 int padded_tokens, int hidden_dim, int n_experts, int topk,
                                 float route_scale, hipStream_t stream);

/* No reference symbol of its own: the select stage (sigmoid, top-k of score+bias, renormalise)
 * of kimi_k2_router_noaux_tc_cuda, pegainfer-kernels/src/ffi/kimi.rs:52-66
 * (csrc/kimi_k2/kimi_router.cu:20-91), taking precomputed fp32 logits. */
int pega_kimi_router_select(const float* logits, const float* e_score_correction_bias,
                            float* topk_weight, int32_t* topk_idx, int active_tokens,
                            int n_experts, int topk, float route_scale, hipStream_t stream);

/* No reference symbol of its own: the router's select stage followed by the token -> expert
 * permutation, in one launch (the router fused into the permutation:
 * csrc/kimi_k2/kimi_router.cu:20-91 then csrc/kimi_k2/kimi_experts.cu:197-268, the pair
 * experts.rs:508-848 issues).  Outputs equal pega_kimi_router_select followed by
 * pega_moe_align_block_size (topk_idx / topk_weight over active_tokens rows, then the
 * permutation of their active_tokens * topk routes), bit for bit, with the union of those two
 * entry points' checks (status 1), and at most 4096 routes (801 above: a decode batch).  Above
 * four tokens the select runs in several workgroups and the last to finish sorts; they count
 * themselves in on a library-wide per-device counter, so launches of this entry point or of
 * pega_dsv2_route_align that overlap on one device race. */
int pega_kimi_route_align(const float* logits, const float* e_score_correction_bias,
                          float* topk_weight, int32_t* topk_idx, int32_t* sorted_token_ids,
                          int32_t* expert_ids, int32_t* num_tokens_post_padded,
                          uint32_t* expert_offsets, uint32_t* expert_cursor, int active_tokens,
                          int n_experts, int topk, float route_scale, int global_start,
                          int local_experts, int block_size, int max_padded_tokens,
                          int max_m_blocks, hipStream_t stream);

/* No reference counterpart: the routers' e^x, y[i] = the double-precision exp of x[i] rounded
 * to fp32, computed as the router kernels compute it (a double polynomial, falling back to the
 * double exp near fp32 rounding midpoints).  For tests that check it over every float. */
int pega_exp_exact_f32(const float* x, float* y, long long n, hipStream_t stream);

/* No reference symbol of its own: the DeepSeek-V2-Lite router (softmax top-k ordered by expert
 * id: pegainfer-deepseek-v2-lite/src/host_ops.rs:388-412, csrc/dsv2_lite/dsv2_lite_moe.cu:41-129)
 * followed by the token -> expert permutation, in one launch.  Outputs equal
 * pega_dsv2_router_select followed by pega_moe_align_block_size, bit for bit; the checks and
 * limits of pega_kimi_route_align (at most 4096 routes, 801 above), and the same race between
 * overlapping launches on one device. */
int pega_dsv2_route_align(const float* logits, float* topk_weight, int32_t* topk_idx,
                          int32_t* sorted_token_ids, int32_t* expert_ids,
                          int32_t* num_tokens_post_padded, uint32_t* expert_offsets,
                          uint32_t* expert_cursor, int tokens, int n_experts, int topk,
                          int global_start, int local_experts, int block_size,
                          int max_padded_tokens, int max_m_blocks, hipStream_t stream);

/* No reference C symbol: DeepSeek-V2-Lite softmax top-k sorted by expert id, restating
 * pegainfer-deepseek-v2-lite/src/host_ops.rs:388-412. */
int pega_dsv2_router_select(const float* logits, float* topk_weight, int32_t* topk_idx,
                            int tokens, int n_experts, int topk, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* PEGA_MOE_H_ */

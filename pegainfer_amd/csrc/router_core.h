// The routers' select stages for one token by one wave, shared by the select kernels, the fused
// router + permutation (router.hip) and the few-token layer (few_tokens.hip): the scores, the
// top-k and the weights are the same bits wherever they run.
#pragma once

#include "common.h"

namespace pega {
namespace {

constexpr int kMaxPerLane = 16;  // n_experts <= 64 * 16

// Order-preserving map of a float to u32 (for non-NaN values; -0 is folded
// into +0 first, so equal floats give equal keys).  Key 0 lies below every
// real value and marks an empty or already selected slot.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A DPP lane move with no "old" operand (bound_ctrl), so that the compiler folds
// it into the consuming max/min as a DPP source.  Rows outside kRowMask are not
// written by that fused instruction and keep their value, which is the value a
// max/min of the lane with itself would give.
template <int kCtrl, int kRowMask = 0xF>
__device__ __forceinline__ uint32_t dpp_mov(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_mov_dpp(static_cast<int>(v), kCtrl, kRowMask, 0xF, true));
}

// Wave-wide reduction over DPP lane moves (quad swaps, half-row and row
// mirrors, then the row-15 and row-31 broadcasts); lane 63 ends up holding
// the result, which is read into a scalar register.
template <typename Op>
__device__ __forceinline__ uint32_t wave_reduce_u32(uint32_t v, Op op) {
  v = op(v, dpp_mov<0xB1>(v));        // quad_perm [1,0,3,2]
  v = op(v, dpp_mov<0x4E>(v));        // quad_perm [2,3,0,1]
  v = op(v, dpp_mov<0x141>(v));       // row_half_mirror
  v = op(v, dpp_mov<0x140>(v));       // row_mirror
  v = op(v, dpp_mov<0x142, 0xA>(v));  // row_bcast:15 into rows 1 and 3
  v = op(v, dpp_mov<0x143, 0xC>(v));  // row_bcast:31 into rows 2 and 3
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

struct MaxU32 {
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
struct MinU32 {
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
};

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float,
                            __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Top-k of the wave's NS x 64 keys (expert id lane + 64 j), largest first,
// equal keys to the lower id.  Returns, on lane r < topk, the r-th selected
// id; the selected keys are cleared.  A round is one DPP max-reduction of the
// lanes' best keys; the holders of the maximum are a ballot, and only when
// several lanes hold it (equal keys) does a second reduction pick the lowest
// id (a lane's own slots are scanned from j = 0, so its candidate is its
// lowest id with that key).
template <int NS>
__device__ __forceinline__ int wave_topk_ids(uint32_t (&key)[NS], int lane, int topk) {
  int my_sel = 0;
  for (int r = 0; r < topk; ++r) {
    // the lane's best key and its lowest slot holding it, found before the
    // reduction so that they overlap its DPP latencies
    uint32_t best = key[0];
    int bj = 0;
#pragma unroll
    for (int j = 1; j < NS; ++j) {
      const bool up = key[j] > best;
      best = up ? key[j] : best;
      bj = up ? j : bj;
    }
    const uint32_t top = wave_reduce_u32(best, MaxU32{});
    const bool mine = best == top;
    const uint64_t holders = __ballot(mine);
    int win;
    if (__popcll(holders) == 1) {
      const int wl = __builtin_ctzll(holders);
      win = __builtin_amdgcn_readlane(bj * 64 + lane, wl);
    } else {
      const uint32_t cand = mine ? static_cast<uint32_t>(bj * 64 + lane) : 0xffffffffu;
      win = static_cast<int>(wave_reduce_u32(cand, MinU32{}));
    }
    const int wj = win >> 6;
    if (lane == (win & 63)) {
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (j == wj) key[j] = 0;
    }
    if (lane == r) my_sel = win;
  }
  return my_sel;
}

// Token t's selection by one wave; lane l owns experts l, l+64, ... (NS slots
// per lane, NS * 64 >= n_experts).  The Kimi score of logit l is
// 1 / (1 + e^-l), e^-l rounded from a double exp.  Writes the token's top-k
// weights and returns, on lane r < topk, the r-th selected id (the caller
// stores the ids); lane r takes its expert's score from the owner lane once,
// after the rounds.
template <int NS>
__device__ __forceinline__ int kimi_select_token(const float* __restrict__ logits,
                                                 const float* __restrict__ bias,
                                                 float* __restrict__ topk_weight, int t,
                                                 int n_experts, int topk, float route_scale) {
  const int lane = threadIdx.x & 63;
  const float* row = logits + static_cast<long long>(t) * n_experts;
  // every slot's loads, then every slot's exponential side by side (the rare
  // double-precision fallbacks after), then the scores: kimi_score's bits
  float lg[NS], bi[NS], ex[NS], sc[NS];
  bool ok[NS];
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int e = lane + 64 * j;
    lg[j] = e < n_experts ? row[e] : 0.0f;
    bi[j] = e < n_experts ? bias[e] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < NS; ++j) ex[j] = exp_exact_f32_try(-lg[j], &ok[j]);
#pragma unroll
  for (int j = 0; j < NS; ++j)
    if (!ok[j]) ex[j] = exp_exact_f32(-lg[j]);
  uint32_t key[NS];
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    sc[j] = 1.0f / (1.0f + ex[j]);
    key[j] = lane + 64 * j < n_experts ? order_key(sc[j] + bi[j]) : 0u;
  }
  const int my_i = wave_topk_ids<NS>(key, lane, topk);
  // the selected expert's score, from its owner lane's slot
  float my_s = 0.0f;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const float v = __builtin_bit_cast(
        float, __builtin_amdgcn_ds_bpermute((my_i & 63) << 2, __builtin_bit_cast(int, sc[j])));
    if (j == (my_i >> 6)) my_s = v;
  }
  if (lane >= topk) my_s = 0.0f;
  // sum in selection order, as the reference's rounds add them
  float sum = 0.0f;
  for (int r = 0; r < topk; ++r) sum += lane_value(my_s, r);
  const float scale = sum > 0.0f ? route_scale / sum : 0.0f;
  if (lane < topk) topk_weight[t * topk + lane] = my_s * scale;
  return my_i;
}

// DeepSeek-V2-Lite selection of token t by one wave: softmax (max-subtracted,
// e^x rounded from a double exp, sum over experts 0, 1, 2, ... in order,
// divide), top-k by probability (equal to the lower id), then ordered by
// expert id.  Writes the weights; returns on lane r < topk the id of rank r
// in id order (lanes >= topk return 0x7fffffff).
template <int NS>
__device__ __forceinline__ int dsv2_select_token(const float* __restrict__ logits,
                                                 float* __restrict__ topk_weight, int t,
                                                 int n_experts, int topk) {
  const int lane = threadIdx.x & 63;
  float p[NS];
  uint32_t mkey = 0;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int e = lane + 64 * j;
    p[j] = e < n_experts ? logits[static_cast<long long>(t) * n_experts + e] : 0.0f;
    if (e < n_experts) mkey = max(mkey, order_key(p[j]));
  }
  mkey = wave_reduce_u32(mkey, MaxU32{});
  const float mx = __builtin_bit_cast(float, (mkey & 0x80000000u) ? (mkey & 0x7fffffffu) : ~mkey);
#pragma unroll
  for (int j = 0; j < NS; ++j)
    p[j] = (lane + 64 * j < n_experts) ? exp_exact_f32_fast(p[j] - mx) : 0.0f;
  // Sequential fp32 sum over experts 0, 1, 2, ... (the reference's order).
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < NS; ++j)
    for (int l = 0; l < 64 && 64 * j + l < n_experts; ++l) sum += lane_value(p[j], l);
  uint32_t key[NS];
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    p[j] = sum == 0.0f ? 0.0f : p[j] / sum;
    key[j] = lane + 64 * j < n_experts ? order_key(p[j]) : 0;
  }
  const int sel = wave_topk_ids<NS>(key, lane, topk);
  const int my_i = lane < topk ? sel : 0x7fffffff;
  // the selected probability, from its owner lane's slot
  float my_w = 0.0f;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const float v = __builtin_bit_cast(
        float, __builtin_amdgcn_ds_bpermute((my_i & 63) << 2, __builtin_bit_cast(int, p[j])));
    if (j == (my_i >> 6)) my_w = v;
  }
  // Order the selection by expert id: a lane's rank is the number of selected
  // ids below its own (selected ids are distinct).
  int rank = 0;
  for (int r = 0; r < topk; ++r)
    rank += __builtin_amdgcn_readlane(my_i, r) < my_i ? 1 : 0;
  if (lane < topk) topk_weight[t * topk + rank] = my_w;
  // hand rank r's id to lane r
  int by_rank = 0x7fffffff;
  for (int r = 0; r < topk; ++r) {
    const int rr = __builtin_amdgcn_readlane(rank, r);
    const int id = __builtin_amdgcn_readlane(my_i, r);
    if (lane == rr) by_rank = id;
  }
  return by_rank;
}

}  // namespace
}  // namespace pega

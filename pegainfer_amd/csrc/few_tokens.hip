// A whole mixture-of-experts layer for a few tokens (at most 16) in two launches, MI355X (gfx950):
//
//   ids, w   = router select of the logits (router_core.h: sigmoid + bias, or softmax)
//   act_e    = silu(x . G_e^T) * (x . U_e^T)            for every local expert e with a route
//   out[t]   = bf16( residual[t] + routed_scale * sum_{e of t} w[t][e] act_e[t] . D_e^T
//                    + (silu(x . Gs^T) * (x . Us^T)) [t] . Ds^T )
//
// with INT4 experts in the device layout of repack.hip (group 32, weight (nibble - 8) * scale) and
// a shared expert in bf16, in INT4, or none.  At these sizes the layer is a stream of weights cut
// into eight short launches by the general path; here
//
//   launch 1   a workgroup per gate/up tile pair of the shared expert, then of each expert slot.
//              A routed workgroup runs the select itself (every one of them: 3 to 4 us that the
//              shared expert's workgroups, which need no routing, cover), takes the slot-th distinct
//              local expert in id order, or ends.  The routing weight and routed_scale are
//              multiplied into the SwiGLU rows, which are written for all tokens: zeros where the
//              token has no route to the expert.
//   launch 2   so the second products are one sum over the concatenated rows of all slots and the
//              shared expert.  That list of 32-k groups, priced by its bytes, is cut into equal
//              shares for the waves of `splits` workgroups per 64 output columns.  With several
//              workgroups, each leaves fp32 sums and counts itself in, and the last one adds them
//              in their order.
//
// An MFMA's 16 rows are the tokens themselves, so rows are never gathered.  INT4 weights: nibble v
// of a word becomes the bf16 16 + v by a shift and one v_and_or (mantissa bits 3..6), a constant
// -24 operand takes 24 * sum(x) off in the same accumulators' start value, and the group's fp32 sum
// times its scale is added to the column's: about 1 VALU instruction a weight and no rounding of
// q * s (the general kernels round it to bf16; the results differ by that).  Where 16 * x or 8 * x
// passes fp32's range, and with infinite activations, such a sum is infinite or NaN: a wave that
// ends with one forms its sums again from (v - 8) / 256, and takes those that were not finite.
//
// Roundings: the SwiGLU rows (with their weights) once to bf16, which the matrix instructions
// take; out once.  Everything between is fp32.
#include <type_traits>

#include "common.h"
#include "pega_moe.h"
#include "router_core.h"

namespace pega {
namespace {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_t;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4_t;

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kMaxTokens = 16, kMaxTopk = 32, kMaxLocal = 512;
constexpr int kSlotDwords = 320;  // one 32-k group of a 64-column tile, as wna16.hip's slots
constexpr int kStream = 2;        // non-temporal: bytes read once

struct FewArgs {
  pega_moe_few p;
  int sh_units, tiles, splits, shared_cost;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0),
                                           static_cast<int>(bytes), 0x00020000);
}
__device__ __forceinline__ u32x4_t load16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(voff), static_cast<int>(soff), 0);
}
__device__ __forceinline__ u32x4_t load16_once(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(voff), static_cast<int>(soff), kStream);
}
__device__ __forceinline__ bf16x8_t as_bf16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  u32x4_t v = {a, b, c, d};
  return __builtin_bit_cast(bf16x8_t, v);
}
__device__ __forceinline__ floatx4_t mfma16(bf16x8_t a, bf16x8_t b, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Two bf16 of a word's nibbles at bits `kBit` and kBit + 16: 16 + v, or (v - 8) / 256 with kWide.
template <int kBit, bool kWide>
__device__ __forceinline__ uint32_t nibble_pair(uint32_t x) {
  if constexpr (kWide)
    return pack_bf16x2((static_cast<float>((x >> kBit) & 15u) - 8.0f) * 0x1p-8f,
                       (static_cast<float>((x >> (kBit + 16)) & 15u) - 8.0f) * 0x1p-8f);
  const uint32_t y = kBit < 3 ? x << (3 - kBit) : x >> (kBit - 3);
  return (y & 0x00780078u) | 0x41804180u;
}

// INT4 weights of NT 64-column tiles, and the activations, over 32-k groups [g0, g1): every lane's
// columns are 32 (lane % 16 / 8) + 8 j + lane % 8 of a tile, j = 0..3, its sums tokens
// 4 (lane / 16) .. + 3.  A wave reads whole 512-byte tiles (one 16-byte load a lane: word row
// lane % 32 of k-tile lane / 32) and transposes them through its LDS slots, a group ahead of its
// use, as wna16.hip's decode kernel does; the activations' 16 bytes (k 16 kt + 8 hf ..) swap their
// middle halves between the lanes of the two k halves to follow the words' k order.
template <int NT>
struct Int4View {
  __amdgpu_buffer_rsrc_t w, s, a;
  uint32_t w_voff[NT], s_voff[NT], a_voff;
  uint32_t w_step, s_step;
};

template <int NT>
__device__ __forceinline__ Int4View<NT> int4_view(const uint8_t* q, const uint16_t* scales, int N,
                                                  int K, const int (&tile)[NT], const uint16_t* act,
                                                  int tokens) {
  const int lane = threadIdx.x & 63;
  const int n16 = lane & 15, kb = lane >> 4;
  const uint32_t n_tiles = static_cast<uint32_t>(N) >> 6;
  Int4View<NT> v;
  v.w = make_rsrc(q, static_cast<uint32_t>(N) * static_cast<uint32_t>(K) / 2u);
  v.s = make_rsrc(scales, static_cast<uint32_t>(K >> 5) * static_cast<uint32_t>(N) * 2u);
  v.a = make_rsrc(act, static_cast<uint32_t>(tokens) * static_cast<uint32_t>(K) * 2u);
  v.w_step = n_tiles * 1024u;
  v.s_step = static_cast<uint32_t>(N) * 2u;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    v.w_voff[i] = static_cast<uint32_t>(lane >> 5) * n_tiles * 512u +
                  static_cast<uint32_t>(tile[i]) * 512u + 16u * (lane & 31);
    v.s_voff[i] = static_cast<uint32_t>(tile[i]) * 128u + 16u * (n16 & 7) + 8u * (n16 >> 3);
  }
  // rows past the last token are past the range: zeros
  v.a_voff = static_cast<uint32_t>(n16) * static_cast<uint32_t>(K) * 2u + 16u * kb;
  return v;
}

template <int NT, int D, bool kWide>
__device__ __forceinline__ void int4_groups(floatx4_t (&acc)[NT][4], const Int4View<NT>& v, int g0,
                                            int g1, uint32_t* slots /* [2][NT][kSlotDwords] */) {
  static_assert(D % 2 == 0, "the two transpose slots alternate with the ring position");
  if (g0 >= g1) return;
  const int lane = threadIdx.x & 63;
  const int c = lane & 31, h = lane >> 5;
  const int n16 = lane & 15, kb = lane >> 4;
  const int cc = n16 & 7, a2 = n16 >> 3, kt = kb >> 1, hf = kb & 1;
  uint32_t* wr = slots + h * 160 + c;
  const uint32_t* rd = slots + kt * 160 + 64 * a2 + 4 * cc + 2 * hf;
  struct Regs {
    u32x4_t w[NT];
    uint32_t s[NT][2];
    u32x4_t a;
  };
  const auto load = [&](Regs& r, int g) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      r.w[i] = load16_once(v.w, v.w_voff[i], static_cast<uint32_t>(g) * v.w_step);
      const auto s = __builtin_amdgcn_raw_buffer_load_b64(
          v.s, static_cast<int>(v.s_voff[i]), static_cast<int>(static_cast<uint32_t>(g) * v.s_step), kStream);
      r.s[i][0] = s[0];
      r.s[i][1] = s[1];
    }
    r.a = load16(v.a, v.a_voff, static_cast<uint32_t>(g) * 64u);
  };
  const auto write = [&](const Regs& r, int par) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      uint32_t* p = wr + (par * NT + i) * kSlotDwords;
      p[0] = r.w[i][0];
      p[32] = r.w[i][1];
      p[64] = r.w[i][2];
      p[96] = r.w[i][3];
    }
  };
  // -24 in every element: the 16 + v that a nibble stands for less its own v - 8
  const bf16x8_t bias = as_bf16x8(0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u);
  const auto compute = [&](const Regs& r, int par) {
    const auto x0 = __builtin_amdgcn_permlane16_swap(r.a[0], r.a[2], false, false);
    const auto x1 = __builtin_amdgcn_permlane16_swap(r.a[1], r.a[3], false, false);
    const bf16x8_t A = as_bf16x8(x0[0], x1[0], x0[1], x1[1]);
    floatx4_t start = {};
    if (!kWide) start = mfma16(A, bias, start);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint32_t* p = rd + (par * NT + i) * kSlotDwords;
      const uint32_t wa0 = p[0], wa1 = p[1], wb0 = p[32], wb1 = p[33];
      const auto frag0 = [&](uint32_t w0, uint32_t w1) {
        return as_bf16x8(nibble_pair<0, kWide>(w0), nibble_pair<0, kWide>(w1),
                         nibble_pair<4, kWide>(w0), nibble_pair<4, kWide>(w1));
      };
      const auto frag1 = [&](uint32_t w0, uint32_t w1) {
        return as_bf16x8(nibble_pair<8, kWide>(w0), nibble_pair<8, kWide>(w1),
                         nibble_pair<12, kWide>(w0), nibble_pair<12, kWide>(w1));
      };
      const floatx4_t t0 = mfma16(A, frag0(wa0, wa1), start), t1 = mfma16(A, frag1(wa0, wa1), start);
      const floatx4_t t2 = mfma16(A, frag0(wb0, wb1), start), t3 = mfma16(A, frag1(wb0, wb1), start);
      const float s0 = bf_lo(r.s[i][0]), s1 = bf_hi(r.s[i][0]), s2 = bf_lo(r.s[i][1]), s3 = bf_hi(r.s[i][1]);
      const auto add = [](float t, float s, float a) {
        return kWide ? __builtin_fmaf(t * s, 256.0f, a) : __builtin_fmaf(t, s, a);
      };
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[i][0][e] = add(t0[e], s0, acc[i][0][e]);
        acc[i][1][e] = add(t1[e], s1, acc[i][1][e]);
        acc[i][2][e] = add(t2[e], s2, acc[i][2][e]);
        acc[i][3][e] = add(t3[e], s3, acc[i][3][e]);
      }
    }
  };
  Regs slot[D];
#pragma unroll
  for (int q = 0; q < D; ++q) {
    load(slot[q], min(g0 + q, g1 - 1));
    __builtin_amdgcn_sched_barrier(0);
  }
  int g = g0;
  write(slot[0], 0);
  for (; g + D <= g1; g += D) {
#pragma unroll
    for (int q = 0; q < D; ++q) {
      write(slot[(q + 1) % D], (q + 1) & 1);
      compute(slot[q], q & 1);
      load(slot[q], min(g + q + D, g1 - 1));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int q = 0; q < D - 1; ++q) {
    if (g + q < g1) {
      if (q + 1 < D - 1 && g + q + 1 < g1) write(slot[q + 1], (q + 1) & 1);
      compute(slot[q], q & 1);
    }
  }
}

// bf16 weights: MR sets of 16 rows (their byte offsets per lane in w_voff, for row lane / 4 of the
// set, 16-byte piece lane % 4) over 32-k steps [s0, s1).  A lane quad reads 64 contiguous bytes of a
// row; ds_bpermute hands lane (c, q) row c's k 8 q ...  Activations: row lane % 16, k 8 (lane / 16).
template <int MR, int D>
__device__ __forceinline__ void bf16_steps(floatx4_t* acc, __amdgpu_buffer_rsrc_t w,
                                           const uint32_t (&w_voff)[MR], __amdgpu_buffer_rsrc_t a,
                                           uint32_t a_voff, int s0, int s1) {
  if (s0 >= s1) return;
  const int lane = threadIdx.x & 63;
  const int src = (4 * (lane & 15) + (lane >> 4)) * 4;
  struct Regs {
    u32x4_t w[MR], a;
  };
  const auto load = [&](Regs& r, int s) {
#pragma unroll
    for (int m = 0; m < MR; ++m) r.w[m] = load16(w, w_voff[m], static_cast<uint32_t>(s) * 64u);
    r.a = load16(a, a_voff, static_cast<uint32_t>(s) * 64u);
  };
  const auto compute = [&](const Regs& r) {
    const bf16x8_t A = __builtin_bit_cast(bf16x8_t, r.a);
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      u32x4_t f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(src, static_cast<int>(r.w[m][e])));
      acc[m] = mfma16(A, __builtin_bit_cast(bf16x8_t, f), acc[m]);
    }
  };
  Regs slot[D];
#pragma unroll
  for (int q = 0; q < D; ++q) {
    load(slot[q], min(s0 + q, s1 - 1));
    __builtin_amdgcn_sched_barrier(0);
  }
  int s = s0;
  for (; s + D <= s1; s += D) {
#pragma unroll
    for (int q = 0; q < D; ++q) {
      compute(slot[q]);
      load(slot[q], min(s + q + D, s1 - 1));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int q = 0; q < D - 1; ++q)
    if (s + q < s1) compute(slot[q]);
}

template <typename... F>
__device__ __forceinline__ bool wave_any_nan(F... sums) {
  float t = 0.0f;
  ((t = __builtin_fmaf(sums, 0.0f, t)), ...);
  return __ballot(t != t) != 0;
}
__device__ __forceinline__ bool any_nan(const floatx4_t (&a)[4]) {
  bool r = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) r |= wave_any_nan(a[j][0], a[j][1], a[j][2], a[j][3]);
  return r;
}

// The elements of a that are infinite or NaN, from b (a row's sums depend on that row alone, so
// the other rows keep theirs).
__device__ __forceinline__ void take_not_finite(floatx4_t (&a)[4], const floatx4_t (&b)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(__builtin_fabsf(a[j][e]) < __builtin_inff())) a[j][e] = b[j][e];
}

__device__ __forceinline__ float silu_mul(float g, float u) {
  return g / (1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f)) * u;
}

// The lane (of 64) and the element that hold token t, column col of a tile's sums.
__device__ __forceinline__ int sum_lane(int t, int col) {
  return (col & 7) + 8 * (col >> 5) + 16 * (t >> 2);
}

// ---------------------------------------------------------------- launch 1
// TR: token rows in fours (the lanes that hold them: 16 TR).
template <int NS, bool kDsv2, int TR>
__global__ __launch_bounds__(kThreads, 4) void few_w13_kernel(FewArgs f) {
  const pega_moe_few& p = f.p;
  __shared__ union {
    uint32_t tr[kWaves][2 * 2 * kSlotDwords];
    floatx4_t red[kWaves][8][16 * TR];
  } lds;
  __shared__ int s_idx[kMaxTokens * kMaxTopk];
  __shared__ float s_w[kMaxTokens * kMaxTopk];
  __shared__ uint32_t s_mask[kMaxLocal];
  __shared__ float s_tok[kMaxTokens];  // a token's factor for this slot's rows
  __shared__ bool s_in[kMaxTokens];    // whether it has a route to the slot's expert
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int T = p.tokens, H = p.hidden_dim;
  int unit = blockIdx.x;

  if (p.shared_kind == PEGA_SHARED_BF16 && unit < f.sh_units) {
    // 8 gate rows and their 8 up rows for all tokens, K shared by the waves
    const int inter = p.shared_inter, j0 = unit * 8;
    const int steps = H >> 5;
    const uint32_t lr = static_cast<uint32_t>(lane >> 2), row_bytes = static_cast<uint32_t>(H) * 2u;
    const uint16_t* W = static_cast<const uint16_t*>(p.shared_w13) + static_cast<long long>(j0) * H;
    const __amdgpu_buffer_rsrc_t wr =
        make_rsrc(W, (static_cast<uint32_t>(inter) + 8u) * row_bytes);
    const uint32_t w_voff[1] = {((lr & 7u) + (lr >> 3) * static_cast<uint32_t>(inter)) * row_bytes +
                                16u * (lane & 3)};
    const __amdgpu_buffer_rsrc_t ar = make_rsrc(p.x, static_cast<uint32_t>(T) * row_bytes);
    floatx4_t acc[1] = {};
    bf16_steps<1, 8>(acc, wr, w_voff, ar, static_cast<uint32_t>(lane & 15) * row_bytes + 16u * (lane >> 4),
                     (steps * wave) / kWaves, (steps * (wave + 1)) / kWaves);
    if (lane < 16 * TR) lds.red[wave][0][lane] = acc[0];
    __syncthreads();
    if (tid < T * 8) {
      const int t = tid >> 3, c = tid & 7;
      float g = 0.0f, u = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        g += lds.red[w][0][c + 16 * (t >> 2)][t & 3];
        u += lds.red[w][0][c + 8 + 16 * (t >> 2)][t & 3];
      }
      p.act_shared[static_cast<long long>(t) * inter + j0 + c] = f2bf(silu_mul(g, u));
    }
    return;
  }

  const uint8_t* q = static_cast<const uint8_t*>(p.shared_w13);
  const uint16_t* sc = p.shared_w13_scales;
  uint16_t* act = p.act_shared;
  int inter = p.shared_inter, tile = unit;
  if (unit < f.sh_units) {  // the shared expert in INT4: every token, weight 1
    if (tid < kMaxTokens) {
      s_tok[tid] = 1.0f;
      s_in[tid] = true;
    }
  } else {
    unit -= f.sh_units;
    const int slot = unit / f.tiles;
    tile = unit - slot * f.tiles;
    inter = p.inter;
    for (int i = tid; i < p.local_experts; i += kThreads) s_mask[i] = 0;
    for (int t = wave; t < T; t += kWaves) {
      int id;
      if constexpr (kDsv2) id = dsv2_select_token<NS>(p.logits, s_w, t, p.n_experts, p.topk);
      else id = kimi_select_token<NS>(p.logits, p.bias, s_w, t, p.n_experts, p.topk, p.route_scale);
      if (lane < p.topk) s_idx[t * p.topk + lane] = id;
    }
    __syncthreads();
    const int routes = T * p.topk;
    for (int r = tid; r < routes; r += kThreads) {
      const int e = s_idx[r] - p.global_start;
      if (e >= 0 && e < p.local_experts) atomicOr(&s_mask[e], 1u << (r / p.topk));
    }
    __syncthreads();
    // the distinct local experts in id order; this workgroup's is number `slot`
    int expert = -1, seen = 0;
    for (int base = 0; base < p.local_experts; base += 64) {
      const bool has = base + lane < p.local_experts && s_mask[base + lane] != 0;
      uint64_t m = __ballot(has);
      const int n = __popcll(m);
      if (unit == 0 && wave == 0 && has)
        p.slots[1 + seen + __popcll(m & ((1ull << lane) - 1))] = base + lane;
      if (expert < 0 && slot - seen < n) {
        for (int i = slot - seen; i > 0; --i) m &= m - 1;
        expert = base + __builtin_ctzll(m);
      }
      seen += n;
    }
    if (unit == 0) {
      if (tid == 0) p.slots[0] = seen;
      for (int r = tid; r < routes; r += kThreads) {
        p.topk_idx[r] = s_idx[r];
        p.topk_weight[r] = s_w[r];
      }
    }
    if (expert < 0) return;
    expert = __builtin_amdgcn_readfirstlane(expert);
    if (tid < kMaxTokens) {
      float w = 0.0f;
      if (tid < T)
        for (int k = 0; k < p.topk; ++k)
          if (s_idx[tid * p.topk + k] - p.global_start == expert) w += s_w[tid * p.topk + k];
      s_tok[tid] = w * p.routed_scale;
      s_in[tid] = ((s_mask[expert] >> tid) & 1u) != 0;
    }
    const long long elems = 2LL * inter * H;
    q = p.w13 + expert * (elems / 2);
    sc = p.w13_scales + expert * (elems / 32);
    act = p.act + static_cast<long long>(slot) * T * inter;
  }
  const int groups = H >> 5;
  const int pair[2] = {tile, tile + (inter >> 6)};
  const Int4View<2> v = int4_view<2>(q, sc, 2 * inter, H, pair, p.x, T);
  const int g0 = (groups * wave) / kWaves, g1 = (groups * (wave + 1)) / kWaves;
  floatx4_t acc[2][4] = {};
  int4_groups<2, 4, false>(acc, v, g0, g1, lds.tr[wave]);
  if (__builtin_expect(any_nan(acc[0]) || any_nan(acc[1]), 0)) {
    floatx4_t again[2][4] = {};
    int4_groups<2, 2, true>(again, v, g0, g1, lds.tr[wave]);
    take_not_finite(acc[0], again[0]);
    take_not_finite(acc[1], again[1]);
  }
  __syncthreads();  // the transpose slots become the sums' place
  if (lane < 16 * TR) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) lds.red[wave][4 * i + j][lane] = acc[i][j];
  }
  __syncthreads();
  for (int o = tid; o < T * 64; o += kThreads) {
    const int t = o >> 6, col = o & 63, j = (col >> 3) & 3, l = sum_lane(t, col);
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      g += lds.red[w][j][l][t & 3];
      u += lds.red[w][4 + j][l][t & 3];
    }
    act[static_cast<long long>(t) * inter + tile * 64 + col] =
        s_in[t] ? f2bf(silu_mul(g, u) * s_tok[t]) : static_cast<uint16_t>(0);
  }
}

// ---------------------------------------------------------------- launch 2
template <int TR>
__global__ __launch_bounds__(kThreads, 4) void few_w2_kernel(FewArgs f) {
  const pega_moe_few& p = f.p;
  __shared__ union {
    uint32_t tr[kWaves][2 * kSlotDwords];
    floatx4_t red[kWaves][4][16 * TR];
  } lds;
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int T = p.tokens, H = p.hidden_dim, I = p.inter;
  const int tile = blockIdx.x, split = blockIdx.y;
  const int slots = __builtin_amdgcn_readfirstlane(p.slots[0]);

  // this wave's share of the priced list: slots' groups at 1, then the shared expert's
  const int per = I >> 5, sh_groups = p.shared_kind != PEGA_SHARED_NONE ? p.shared_inter >> 5 : 0;
  const int cost = f.shared_cost;
  const int routed_end = slots * per, total = routed_end + sh_groups * cost;
  const int parts = f.splits * kWaves, part = split * kWaves + wave;
  const int lo = static_cast<int>(static_cast<long long>(total) * part / parts);
  const int hi = static_cast<int>(static_cast<long long>(total) * (part + 1) / parts);
  const int sh0 = (max(lo - routed_end, 0) + cost - 1) / cost;
  const int sh1 = (max(hi - routed_end, 0) + cost - 1) / cost;

  floatx4_t acc[1][4] = {};
  const int tiles1[1] = {tile};
  const auto run = [&](floatx4_t (&acc)[1][4], auto wide) {
    constexpr bool kWide = decltype(wide)::value;
    constexpr int D = kWide ? 2 : 4;
    for (int at = lo; at < min(hi, routed_end);) {
      const int s = at / per, g0 = at - s * per, g1 = min(per, g0 + min(hi, routed_end) - at);
      const int expert = __builtin_amdgcn_readfirstlane(p.slots[1 + s]);
      const long long elems = static_cast<long long>(H) * I;
      const Int4View<1> v =
          int4_view<1>(p.w2 + expert * (elems / 2), p.w2_scales + expert * (elems / 32), H, I,
                       tiles1, p.act + static_cast<long long>(s) * T * I, T);
      int4_groups<1, D, kWide>(acc, v, g0, g1, lds.tr[wave]);
      at += g1 - g0;
    }
    if (p.shared_kind == PEGA_SHARED_INT4) {
      const Int4View<1> v = int4_view<1>(static_cast<const uint8_t*>(p.shared_w2), p.shared_w2_scales,
                                         H, p.shared_inter, tiles1, p.act_shared, T);
      int4_groups<1, D, kWide>(acc, v, sh0, sh1, lds.tr[wave]);
    } else if (p.shared_kind == PEGA_SHARED_BF16) {
      const uint32_t row_bytes = static_cast<uint32_t>(p.shared_inter) * 2u;
      const __amdgpu_buffer_rsrc_t wr =
          make_rsrc(static_cast<const uint16_t*>(p.shared_w2) + static_cast<long long>(tile) * 64 * p.shared_inter,
                    64u * row_bytes);
      const uint32_t n = static_cast<uint32_t>(lane >> 2);  // as the INT4 tiles' columns
      uint32_t w_voff[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w_voff[j] = (32u * (n >> 3) + 8u * j + (n & 7u)) * row_bytes + 16u * (lane & 3);
      const __amdgpu_buffer_rsrc_t ar = make_rsrc(p.act_shared, static_cast<uint32_t>(T) * row_bytes);
      bf16_steps<4, 4>(acc[0], wr, w_voff, ar,
                       static_cast<uint32_t>(lane & 15) * row_bytes + 16u * (lane >> 4), sh0, sh1);
    }
  };
  run(acc, std::integral_constant<bool, false>{});
  if (__builtin_expect(any_nan(acc[0]), 0)) {
    floatx4_t again[1][4] = {};
    run(again, std::integral_constant<bool, true>{});
    take_not_finite(acc[0], again[0]);
  }
  __syncthreads();
  if (lane < 16 * TR) {
#pragma unroll
    for (int j = 0; j < 4; ++j) lds.red[wave][j][lane] = acc[0][j];
  }
  __syncthreads();
  const auto finish = [&](int t, int col, float sum) {
    const long long o = static_cast<long long>(t) * H + tile * 64 + col;
    if (p.residual) sum += bf2f(p.residual[o]);
    p.out[o] = f2bf(sum);
  };
  const auto place = [&](int s, int t, int col) {
    return p.partials + (static_cast<long long>(s) * T + t) * H + tile * 64 + col;
  };
  for (int o = tid; o < T * 64; o += kThreads) {
    const int t = o >> 6, col = o & 63, j = (col >> 3) & 3, l = sum_lane(t, col);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += lds.red[w][j][l][t & 3];
    if (f.splits == 1) finish(t, col, sum);
    else __hip_atomic_store(place(split, t, col), sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (f.splits == 1) return;
  // The sums are device-coherent stores that have completed before the arrival is counted; the
  // last arrival of the tile reads them the same way and puts the counter back to zero.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    const uint32_t prev = __hip_atomic_fetch_add(&p.counters[tile], 1u, __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT);
    s_last = prev == static_cast<uint32_t>(f.splits - 1);
    if (s_last) __hip_atomic_store(&p.counters[tile], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  for (int o = tid; o < T * 64; o += kThreads) {
    const int t = o >> 6, col = o & 63;
    float sum = 0.0f;
    for (int s = 0; s < f.splits; ++s)
      sum += __hip_atomic_load(place(s, t, col), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    finish(t, col, sum);
  }
}

template <int NS, bool kDsv2>
void launch_w13(const FewArgs& f, unsigned grid, hipStream_t stream) {
  if (f.p.tokens <= 4)
    hipLaunchKernelGGL((few_w13_kernel<NS, kDsv2, 1>), dim3(grid), dim3(kThreads), 0, stream, f);
  else
    hipLaunchKernelGGL((few_w13_kernel<NS, kDsv2, 4>), dim3(grid), dim3(kThreads), 0, stream, f);
}

template <bool kDsv2>
void launch_w13_slots(const FewArgs& f, unsigned grid, hipStream_t stream) {
  const int need = ceil_div(f.p.n_experts, 64);
  if (need <= 1) launch_w13<1, kDsv2>(f, grid, stream);
  else if (need <= 2) launch_w13<2, kDsv2>(f, grid, stream);
  else if (need <= 6) launch_w13<6, kDsv2>(f, grid, stream);
  else launch_w13<kMaxPerLane, kDsv2>(f, grid, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int few_splits(int hidden_dim) {
  const int tiles = hidden_dim / 64;
  int s = 1;
  while (s < PEGA_FEW_MAX_SPLITS && tiles * s < 256) s *= 2;
  return s;
}

}  // namespace
}  // namespace pega

using namespace pega;

// No reference counterpart as one call: the decode layer of moe_nccl.rs:98-239 without its
// collectives (and the DeepSeek-V2-Lite layer), for a few tokens.
PEGA_API int pega_moe_few_tokens(const pega_moe_few* args, hipStream_t stream) {
  if (!args) return fail(kInvalidValue, "moe_few_tokens: null arguments");
  const pega_moe_few& p = *args;
  if (!p.x || !p.logits || !p.w13 || !p.w13_scales || !p.w2 || !p.w2_scales || !p.out ||
      !p.topk_weight || !p.topk_idx || !p.act || !p.slots || !p.partials || !p.counters ||
      (!p.softmax && !p.bias))
    return fail(kInvalidValue, "moe_few_tokens: null pointer");
  if (p.shared_kind != PEGA_SHARED_NONE && p.shared_kind != PEGA_SHARED_BF16 &&
      p.shared_kind != PEGA_SHARED_INT4)
    return fail(kInvalidValue, "moe_few_tokens: shared_kind %d", p.shared_kind);
  const bool shared = p.shared_kind != PEGA_SHARED_NONE;
  if (shared && (!p.shared_w13 || !p.shared_w2 || !p.act_shared ||
                 (p.shared_kind == PEGA_SHARED_INT4 && (!p.shared_w13_scales || !p.shared_w2_scales))))
    return fail(kInvalidValue, "moe_few_tokens: null pointer of the shared expert");
  if (p.tokens <= 0 || p.hidden_dim <= 0 || p.inter <= 0 || p.local_experts <= 0 ||
      p.n_experts <= 0 || p.topk <= 0 || p.topk > p.n_experts || p.global_start < 0 ||
      p.global_start > p.n_experts - p.local_experts || (shared && p.shared_inter <= 0))
    return fail(kInvalidValue, "moe_few_tokens: bad shape tokens=%d H=%d I=%d E=%d of %d from %d topk=%d",
                p.tokens, p.hidden_dim, p.inter, p.local_experts, p.n_experts, p.global_start, p.topk);
  if (!p.softmax && !(p.route_scale > 0.0f))
    return fail(kInvalidValue, "moe_few_tokens: route_scale must be positive");
  if (p.tokens > kMaxTokens || p.topk > kMaxTopk || p.local_experts > kMaxLocal ||
      p.n_experts > 64 * kMaxPerLane)
    return fail(kNotSupported, "moe_few_tokens: at most %d tokens, top-%d, %d local experts of %d",
                kMaxTokens, kMaxTopk, kMaxLocal, 64 * kMaxPerLane);
  if (p.hidden_dim % 64 != 0 || p.inter % 64 != 0 || (shared && p.shared_inter % 64 != 0))
    return fail(kNotSupported, "moe_few_tokens: hidden and intermediate sizes must be multiples of 64");
  const long long biggest = 2LL * (shared && p.shared_inter > p.inter ? p.shared_inter : p.inter);
  if ((biggest + 16) * p.hidden_dim * 2 >= (1LL << 31))
    return fail(kNotSupported, "moe_few_tokens: a projection over 2 GiB (H=%d)", p.hidden_dim);
  const void* vecs[] = {p.x, p.w13, p.w13_scales, p.w2, p.w2_scales, p.act, shared ? p.shared_w13 : nullptr,
                        shared ? p.shared_w2 : nullptr, shared ? p.act_shared : nullptr,
                        p.shared_kind == PEGA_SHARED_INT4 ? p.shared_w13_scales : nullptr,
                        p.shared_kind == PEGA_SHARED_INT4 ? p.shared_w2_scales : nullptr};
  for (const void* v : vecs)
    if (!aligned16(v)) return fail(kNotSupported, "moe_few_tokens: buffers must be 16-byte aligned");
  FewArgs f{p, 0, p.inter / 64, few_splits(p.hidden_dim), p.shared_kind == PEGA_SHARED_BF16 ? 3 : 1};
  if (p.shared_kind == PEGA_SHARED_BF16) f.sh_units = p.shared_inter / 8;
  if (p.shared_kind == PEGA_SHARED_INT4) f.sh_units = p.shared_inter / 64;
  const int routes = p.tokens * p.topk;
  const int slots = routes < p.local_experts ? routes : p.local_experts;
  const unsigned grid = static_cast<unsigned>(f.sh_units + slots * f.tiles);
  if (p.softmax) launch_w13_slots<true>(f, grid, stream);
  else launch_w13_slots<false>(f, grid, stream);
  const int rc = launch_status("moe_few_tokens (W13)");
  if (rc != kSuccess) return rc;
  const dim3 grid2(static_cast<unsigned>(p.hidden_dim / 64), static_cast<unsigned>(f.splits));
  if (p.tokens <= 4) hipLaunchKernelGGL((few_w2_kernel<1>), grid2, dim3(kThreads), 0, stream, f);
  else hipLaunchKernelGGL((few_w2_kernel<4>), grid2, dim3(kThreads), 0, stream, f);
  return launch_status("moe_few_tokens (W2)");
}

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
//   launch 1   workgroups for the shared expert's gate/up tile pairs, and others for the routed
//              experts.  A routed one runs the select itself (each of them does: 4 to 5 us, which the
//              shared expert's workgroups, that need no routing, cover), and then takes gate/up tile
//              pairs of the distinct local experts, in id order, in turn with the others.  The routing
//              weight and routed_scale are multiplied into the SwiGLU rows, which are written for
//              the expert's tokens (of up to four tokens, for all: zeros where there is no route).
//   launch 2   so the second products are one sum over the concatenated rows of all slots and the
//              shared expert.  That list of 32-k groups, priced by its bytes, is cut into equal
//              shares for the waves of `splits` workgroups per 64 output columns.  With several
//              workgroups, each leaves fp32 sums and counts itself in, and the last one adds them
//              in their order.
//
// INT4 products without a dequantisation: a nibble masked out of its word is the fp16 v 2^-24 (or
// v 2^-20, four bits further up), so a mask a pair makes v_mfma_f32_16x16x32_f16 operands of whole
// words, 5 instructions for 8 weights.  The activations go in as fp16 scaled by a power of two (a
// row's largest to 2^14 .. 2^15; exact down to 2^-25 of it, and to 2^-40 of it below), the second half
// of a fragment's k divided by 16; a constant operand of -8 steps starts the sums, and a 32-k
// group's fp32 sum times its scale is added to the column's.  Weights count as (nibble - 8) * scale
// unrounded (the general kernels round that product to bf16; the results differ by it).
//
// An MFMA's 16 rows are the tokens, with more than four of them those that have a route to the
// expert (16 tokens bring an expert two of them at most sizes).  With up to 4 (8) rows, 4 (2) groups
// share an instruction's rows, R = 4 (8) to each: group g's instruction has the tokens in rows R g .. and zeros
// elsewhere, the sums of all of them land in one accumulator, and the scale is a lane's own group's.
// Then a scale is applied to 4 sums a lane instead of 16, and scales and activations are loaded
// once per 4 (2) groups.
//
// Roundings: the SwiGLU rows, with their weights, once to fp16 with a scale for each 64, the type that the
// nibbles' products take (2^-11 of each at most); to bf16 in front of a bf16 down projection, since an
// instruction's operands are of one type (2^-8 of each at most: one token of a Kimi share is 0.0021 off the
// formula, of which rounding out alone makes 0.0017); out once.  Everything between is fp32.  A row with an
// infinite or NaN activation gives NaN where an INT4 expert takes it.
//
// The weights' bytes bound it, below them the select in front of the routed stream (4 us, 9 from nine
// tokens on), 2 us between the launches and 3 for the last workgroups' join.  48 of 384 experts of 7168 x
// 2048 with a bf16 shared expert at 1 / 2 / 4 / 8 / 16 tokens 28 / 32 / 50 / 64 / 88 us (112 to 429 MB, 3.7 to 4.9
// TB/s); 64 experts of 2048 x 1408 with an INT4 one at 1 / 3 / 5 / 8 / 16 23 / 32 / 42 / 49 / 68 us (39 to 257 MB).
#include <type_traits>

#include "common.h"
#include "pega_moe.h"
#include "router_core.h"

namespace pega {
namespace {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_t;
typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8_t;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4_t;

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kMaxTokens = 16, kMaxTopk = 32, kMaxLocal = 512;
constexpr int kMaxShares = 4;     // of K that launch 1 cuts a tile pair into
constexpr int kSlotDwords = 320;  // one 32-k group of a 64-column tile, as wna16.hip's slots
constexpr int kStream = 2;        // non-temporal: bytes read once
constexpr uint32_t kOutOfRange = 0x80000000u;  // voffset that fails every range check

struct FewArgs {
  pega_moe_few p;
  int sh_units, tiles, splits, shared_cost;
  int routed_first, routed;  // routed workgroups before the shared expert's, and in all
};

// The base and the size in SGPRs: a resource that the compiler takes for a lane's own costs a loop
// around every load.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(a)));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32)));
  return __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>((static_cast<uint64_t>(hi) << 32) | lo), static_cast<short>(0),
      __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), 0x00020000);
}
__device__ __forceinline__ u32x4_t load16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(voff), static_cast<int>(soff), 0);
}
__device__ __forceinline__ u32x4_t load16_once(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(voff), static_cast<int>(soff), kStream);
}
__device__ __forceinline__ f16x8_t as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  u32x4_t v = {a, b, c, d};
  return __builtin_bit_cast(f16x8_t, v);
}
__device__ __forceinline__ floatx4_t mfma16(bf16x8_t a, bf16x8_t b, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx4_t mfma16(f16x8_t a, f16x8_t b, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A value that the compiler takes for a new one.
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// 2^e as a float, e in -126 .. 127.
__device__ __forceinline__ float pow2(int e) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23);
}
// The exponent of a magnitude's float bits (of an infinity or a NaN 128, of the smallest -127).
__device__ __forceinline__ int exponent(uint32_t bits) { return static_cast<int>(bits >> 23) - 127; }

// Where the bytes of a 64-column tile of an INT4 operand, and the activations that meet it, are.  Lane
// columns of the tile are 32 (lane % 16 / 8) + 8 j + lane % 8, j = 0..3.  kScaled: the activations are
// fp16 with a factor for each 64 columns and token (launch 2), which undoes their scaling and half of
// the nibbles' 2^-24, so that the sums are kUndo times too small: the whole of it passes fp32's range
// for rows of 2^118 and more, and so would a group's products before their scale.  Otherwise they are
// bf16 rows, which the lane turns into fp16 by its row's factor (launch 1).
constexpr float kUndo = 4096.0f;
struct Int4View {
  __amdgpu_buffer_rsrc_t w, s, a, f;
  uint32_t w_voff, s_voff, a_voff, f_voff;
  uint32_t w_step, s_step;
};

// R: token rows of an instruction that a group takes (4, 8 or 16).  row: of the `rows` activation
// rows, the one that the lane brings, for row (lane % 16) % R of an instruction; -1 none.
template <int R>
__device__ __forceinline__ Int4View int4_view(const uint8_t* q, const uint16_t* scales, int N, int K,
                                              int tile, const void* act, const float* factors,
                                              int row, int rows) {
  const int lane = fresh(threadIdx.x & 63);
  const int n16 = lane & 15, kb = lane >> 4;
  const uint32_t n_tiles = static_cast<uint32_t>(N) >> 6;
  Int4View v;
  v.w = make_rsrc(q, static_cast<uint32_t>(N) * static_cast<uint32_t>(K) / 2u);
  v.s = make_rsrc(scales, static_cast<uint32_t>(K >> 5) * static_cast<uint32_t>(N) * 2u);
  v.a = make_rsrc(act, static_cast<uint32_t>(rows) * static_cast<uint32_t>(K) * 2u);
  v.f = make_rsrc(factors, static_cast<uint32_t>(K >> 6) * 64u);
  v.w_step = n_tiles * 1024u;
  v.s_step = static_cast<uint32_t>(N) * 2u;
  v.w_voff = static_cast<uint32_t>(lane >> 5) * n_tiles * 512u + static_cast<uint32_t>(tile) * 512u +
             16u * (lane & 31);
  v.s_voff = static_cast<uint32_t>(tile) * 128u + 16u * (n16 & 7) + 8u * (n16 >> 3);
  v.a_voff = row >= 0 ? static_cast<uint32_t>(row) * static_cast<uint32_t>(K) * 2u + 16u * kb
                      : kOutOfRange;  // reads zeros
  v.f_voff = static_cast<uint32_t>((4 * kb) % R) * 4u;
  return v;
}

// 32-k groups [g0, g1) of a tile into acc: element e of lane (n16, q) sums, over the groups of its
// place (4 q) / R in each set of 16 / R, token (4 q) % R + e.  A wave reads whole 512-byte tiles (one
// 16-byte load a lane: word row lane % 32 of k-tile lane / 32) and transposes them through its LDS slots,
// one ahead of their use, as wna16.hip's decode kernel does; the activations' 16 bytes (k 16 kt +
// 8 hf ..) swap their middle halves between the lanes of the two k halves to follow the words' k order.
// row_factor: of the lane's activation row, without kScaled.
// D groups are in flight: eight in launch 1 took 1 to 5% longer (16 tokens 90.2 and 72.1 against 87.9 and
// 68.5 us).
template <int R, bool kScaled>
__device__ __forceinline__ void int4_groups(floatx4_t (&acc)[4], const Int4View& v, int g0, int g1,
                                            float row_factor, uint32_t* slots /* [2][kSlotDwords] */) {
  constexpr int D = 4, G = 16 / R;  // groups of a set
  static_assert(D % G == 0 && D % 2 == 0, "whole sets, and two transpose slots in turn");
  if (g0 >= g1) return;
  const int lane = fresh(threadIdx.x & 63);
  const int c = lane & 31, h = lane >> 5;
  const int n16 = lane & 15, kb = lane >> 4;
  const int cc = n16 & 7, a2 = n16 >> 3, kt = kb >> 1, hf = kb & 1;
  const int row_group = n16 / R, sum_group = (4 * kb) / R;
  uint32_t* wr = slots + h * 160 + c;
  const uint32_t* rd = slots + kt * 160 + 64 * a2 + 4 * cc + 2 * hf;
  struct Set {
    uint32_t s[2];
    u32x4_t a, f;
  };
  const auto load_words = [&](u32x4_t& w, int g) {
    w = load16_once(v.w, v.w_voff, static_cast<uint32_t>(min(g, g1 - 1)) * v.w_step);
  };
  // a set's scales and factors are those of the lane's own group; groups past the end bring the last
  // one's, and activations of zero
  const auto load_set = [&](Set& r, int g) {
    const uint32_t mine = static_cast<uint32_t>(min(g + sum_group, g1 - 1));
    const auto s = __builtin_amdgcn_raw_buffer_load_b64(
        v.s, static_cast<int>(v.s_voff + mine * v.s_step), 0, 0);
    r.s[0] = s[0];
    r.s[1] = s[1];
    const int row = g + row_group;
    r.a = load16(v.a, row < g1 ? v.a_voff + static_cast<uint32_t>(row) * 64u : kOutOfRange, 0);
    if (kScaled) r.f = load16(v.f, v.f_voff + (mine >> 1) * 64u, 0);
  };
  const auto write = [&](const u32x4_t& w, int par) {
    uint32_t* p = wr + par * kSlotDwords;
    p[0] = w[0];
    p[32] = w[1];
    p[64] = w[2];
    p[96] = w[3];
  };
  // -8 steps of 2^-24 for the first half of a fragment's k, of 2^-20 for the second
  const f16x8_t bias = as_f16x8(0x80088008u, 0x80088008u, 0x80808080u, 0x80808080u);
  // bf16 rows become fp16 (exact but for the row's smallest values, which are cut off), k 8 .. 15 of
  // each 16, which meet the v 2^-20 and come from the lanes of the second k half, divided by 16 as
  // launch 1 leaves its fp16 rows
  const float k = hf ? row_factor * 0.0625f : row_factor;
  const auto activations = [&](u32x4_t a) {
    if constexpr (!kScaled) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        a[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(bf_lo(a[i]) * k, bf_hi(a[i]) * k));
    }
    const auto x0 = __builtin_amdgcn_permlane16_swap(a[0], a[2], false, false);
    const auto x1 = __builtin_amdgcn_permlane16_swap(a[1], a[3], false, false);
    return u32x4_t{x0[0], x1[0], x0[1], x1[1]};
  };
  u32x4_t words[D];
  Set set, next;
  load_set(set, g0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int q = 0; q < D; ++q) {
    load_words(words[q], g0 + q);
    __builtin_amdgcn_sched_barrier(0);
  }
  write(words[0], 0);
  for (int g = g0; g < g1; g += D) {
#pragma unroll
    for (int q = 0; q < D; q += G) {
      if (q != 0 && g + q >= g1) break;
      const u32x4_t x = activations(set.a);
      floatx4_t start = {};
      start = mfma16(__builtin_bit_cast(f16x8_t, x), bias, start);
      floatx4_t t[4] = {start, start, start, start};
      load_set(next, g + q + G);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < G; ++u) {
        const int at = q + u;
        write(words[(at + 1) % D], (at + 1) & 1);
        f16x8_t A = __builtin_bit_cast(f16x8_t, x);
        if (G > 1) {
          const uint32_t keep = row_group == u ? ~0u : 0u;
          A = as_f16x8(x[0] & keep, x[1] & keep, x[2] & keep, x[3] & keep);
        }
        const uint32_t* p = rd + (at & 1) * kSlotDwords;
        const uint32_t wa0 = p[0], wa1 = p[1], wb0 = p[32], wb1 = p[33];
        const auto frag = [](uint32_t w0, uint32_t w1) {
          return as_f16x8(w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u);
        };
        t[0] = mfma16(A, frag(wa0, wa1), t[0]);
        t[1] = mfma16(A, frag(wa0 >> 8, wa1 >> 8), t[1]);
        t[2] = mfma16(A, frag(wb0, wb1), t[2]);
        t[3] = mfma16(A, frag(wb0 >> 8, wb1 >> 8), t[3]);
        load_words(words[at], g + at + D);
        __builtin_amdgcn_sched_barrier(0);
      }
      const float s[4] = {bf_lo(set.s[0]), bf_hi(set.s[0]), bf_lo(set.s[1]), bf_hi(set.s[1])};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t f = set.f[e];  // (a bit cast of the element itself takes element 0)
          const float sum = kScaled ? t[j][e] * __builtin_bit_cast(float, f) : t[j][e];
          acc[j][e] = __builtin_fmaf(sum, s[j], acc[j][e]);
        }
      set = next;
    }
  }
}

// work(rows of an instruction that a group takes) for that many token rows.
template <bool kGather, typename Work>
__device__ __forceinline__ void by_rows(int rows, Work work) {
  if (!kGather || rows <= 4) work(std::integral_constant<int, 4>{});
  else if (rows <= 8) work(std::integral_constant<int, 8>{});
  else work(std::integral_constant<int, 16>{});
}

// The sums of a set's groups, together: afterwards lanes 0 .. 4 R - 1 have the token rows' totals.
template <int R>
__device__ __forceinline__ void add_places(floatx4_t (&acc)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (R == 4) acc[j][e] += __shfl_xor(acc[j][e], 16);
      if (R <= 8) acc[j][e] += __shfl_xor(acc[j][e], 32);
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

// Sums between workgroups of a launch: device-coherent stores and loads (the L2 is per XCD), of
// which every store has completed before the workgroup counts itself in.  last_of: whether this
// workgroup is the last of n to do so, for all its threads; the last puts the counter back to zero.
__device__ __forceinline__ void store_coherent(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_coherent(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool last_of(uint32_t* counter, int n, int* s_last) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t prev = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *s_last = prev == static_cast<uint32_t>(n - 1);
    if (*s_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *s_last != 0;
}

__device__ __forceinline__ float silu_mul(float g, float u) {
  return g / (1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f)) * u;
}

// The lane (of 64) and the element that hold token t, column col of a tile's sums.
__device__ __forceinline__ int sum_lane(int t, int col) {
  return (col & 7) + 8 * (col >> 5) + 16 * (t >> 2);
}

// ---------------------------------------------------------------- launch 1
// The largest magnitude (its float bits) of row t of x, by one wave.
__device__ __forceinline__ uint32_t row_amax(const uint16_t* x, int t, int H) {
  const int lane = threadIdx.x & 63;
  const uint16_t* row = x + static_cast<long long>(t) * H;
  uint32_t m = 0;
  for (int v0 = lane; v0 < H / 8; v0 += 8 * 64) {  // eight loads on their way at a time
    uint4 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = *reinterpret_cast<const uint4*>(row + 8 * min(v0 + 64 * i, H / 8 - 1));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) m = max(m, max((w[k] << 16) & 0x7fff0000u, w[k] & 0x7fff0000u));
    }
  }
  return wave_reduce_u32(m, MaxU32{});
}

template <int NS, bool kDsv2, int R>
__global__ __launch_bounds__(kThreads, 4) void few_w13_kernel(FewArgs f) {
  constexpr bool kGather = R > 4;
  const pega_moe_few& p = f.p;
  __shared__ union {
    uint32_t tr[kWaves][2 * kSlotDwords];
    floatx4_t red[kWaves][4][4 * R];
  } lds;
  __shared__ int s_idx[kMaxTokens * kMaxTopk];
  __shared__ float s_w[kMaxTokens * kMaxTopk];
  __shared__ uint32_t s_mask[kMaxLocal];
  __shared__ uint16_t s_list[kMaxLocal];
  __shared__ float s_tok[kMaxTokens];   // a row's factor
  __shared__ bool s_in[kMaxTokens];     // whether its token has a route to the slot's expert
  __shared__ uint8_t s_row[kMaxTokens]; // its token
  __shared__ uint32_t s_amax[kMaxTokens];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int T = p.tokens, H = p.hidden_dim;
  // routed workgroups that start with the launch come first: their router logits are then asked
  // for before the shared expert's weights fill the memory's queues (10 against 5 us for the select)
  int unit = static_cast<int>(blockIdx.x) - f.routed_first;
  const bool shared = unit >= 0 && unit < f.sh_units;

  if (shared && p.shared_kind == PEGA_SHARED_BF16) {
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
    if (lane < 4 * R) lds.red[wave][0][lane] = acc[0];
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

  for (int t = kWaves - 1 - wave; t < T; t += kWaves) {  // the select starts from wave 0
    const uint32_t m = row_amax(p.x, t, H);
    if (lane == 0) s_amax[t] = m;
  }
  int live = 1, first = unit, step = 1 << 30;  // this workgroup's shares of tile pairs
  int shares = 1;                              // of K that a tile pair is cut into
  const int inter = shared ? p.shared_inter : p.inter;
  const int tiles = inter >> 6;
  if (!shared) {
    const int mine = unit < 0 ? static_cast<int>(blockIdx.x) : unit + f.routed_first - f.sh_units;
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
    // the distinct local experts in id order: the slots
    live = 0;
    for (int base = 0; base < p.local_experts; base += 64) {
      const bool has = base + lane < p.local_experts && s_mask[base + lane] != 0;
      const uint64_t m = __ballot(has);
      if (wave == 0 && has)
        s_list[live + __popcll(m & ((1ull << lane) - 1))] = static_cast<uint16_t>(base + lane);
      live += __popcll(m);
    }
    if (mine == 0) {
      __syncthreads();
      if (tid == 0) p.slots[0] = live;
      for (int i = tid; i < live; i += kThreads)
        p.slots[1 + i] = static_cast<int>(s_mask[s_list[i]] << 16 | s_list[i]);
      for (int r = tid; r < routes; r += kThreads) {
        p.topk_idx[r] = s_idx[r];
        p.topk_weight[r] = s_w[r];
      }
    }
    first = mine;
    step = f.routed;
    // Few tile pairs are cut along K, while a CU of its own is there for each share: a workgroup
    // streams about 35 GB/s, whatever the others leave free.  The launch has a workgroup for every tile
    // pair that the routes could need, so this is where some go to other GPUs or several to one expert;
    // with all of them here and apart there is one for each pair and no cut.
    if (live > 0) shares = max(1, min(kMaxShares, f.routed_first / (live * tiles)));
  }
  __syncthreads();
  // waves 0 to 3 share K, or the workgroup's share of it, of the gate tile, 4 to 7 of the up tile
  constexpr int kPart = kWaves / 2;
  const int groups = H >> 5, half = wave / kPart, part = wave % kPart;
  for (int at = first; at < live * tiles * shares; at += step) {
    const int pair = at / shares, share = at - pair * shares;
    const int slot = pair / tiles, tile = pair - slot * tiles;
    const int k0 = (groups * share) / shares, k1 = (groups * (share + 1)) / shares;
    const int g0 = k0 + ((k1 - k0) * part) / kPart, g1 = k0 + ((k1 - k0) * (part + 1)) / kPart;
    const uint8_t* q = static_cast<const uint8_t*>(p.shared_w13);
    const uint16_t* sc = p.shared_w13_scales;
    uint16_t* act = p.act_shared;
    float* factors = p.act_shared_factors;
    int rows = T, row_of_mine = -1, expert = 0;
    if (shared) {
      if (tid < T) {
        s_tok[tid] = 1.0f;
        s_in[tid] = true;
        s_row[tid] = static_cast<uint8_t>(tid);
      }
    } else {
      expert = s_list[slot];
      const uint32_t mask = s_mask[expert];
      if constexpr (kGather) rows = __builtin_amdgcn_readfirstlane(__popc(mask));
      const bool has = ((mask >> (tid & 31)) & 1u) != 0;
      if (tid < T && (has || !kGather)) {
        row_of_mine = kGather ? __popc(mask & ((1u << tid) - 1u)) : tid;
        s_in[row_of_mine] = has;
        s_row[row_of_mine] = static_cast<uint8_t>(tid);
      }
      const long long elems = 2LL * inter * H;
      q = p.w13 + expert * (elems / 2);
      sc = p.w13_scales + expert * (elems / 32);
      act = p.act + static_cast<long long>(slot) * T * inter;
      factors = p.act_factors + static_cast<long long>(slot) * tiles * kMaxTokens;
    }
    if (kGather) __syncthreads();
    if (row_of_mine >= 0) {
      float w = 0.0f;
      for (int k = 0; k < p.topk; ++k)
        if (s_idx[tid * p.topk + k] - p.global_start == expert) w += s_w[tid * p.topk + k];
      s_tok[row_of_mine] = w * p.routed_scale;
    }
    floatx4_t acc[4] = {};
    by_rows<kGather>(rows, [&](auto r) {
      constexpr int RU = decltype(r)::value;
      const int row = (tid & 15) % RU, token = row >= rows ? -1 : kGather ? s_row[row] : row;
      const float row_factor = token >= 0 ? pow2(min(14 - exponent(s_amax[token]), 127)) : 0.0f;
      const Int4View v = int4_view<RU>(q, sc, 2 * inter, H, tile + half * tiles, p.x, nullptr, token, T);
      int4_groups<RU, false>(acc, v, g0, g1, row_factor, lds.tr[wave]);
      add_places<RU>(acc);
    });
    __syncthreads();  // the transpose slots become the sums' place
    // the lane read anew: what is computed from it would otherwise sit in registers for the whole loop
    const int lane = fresh(tid & 63);
    if (lane < 4 * R) {
#pragma unroll
      for (int j = 0; j < 4; ++j) lds.red[wave][j][lane] = acc[j];
    }
    __syncthreads();
    // a wave finishes a row's 64 columns: SwiGLU times the row's factor, in fp16 with the
    // largest at 2^14 .. 2^15; the factor that undoes it takes 2^12 of the nibbles' 2^24 along
    const auto finish = [&](int t, float g, float u) {
      // x came in times 2^(14 - exponent), at most 2^127, and v as v 2^-24
      const int e = max(10 + exponent(s_amax[s_row[t]]), -103);
      const float a = s_in[t] ? silu_mul(__builtin_ldexpf(g, e), __builtin_ldexpf(u, e)) * s_tok[t] : 0.0f;
      const uint32_t top = wave_reduce_u32(__builtin_bit_cast(uint32_t, a) & 0x7fffffffu, MaxU32{});
      const int ae = top == 0 ? 0 : exponent(top);
      const float down = (lane & 8) ? 0.0625f : 1.0f;  // what meets the nibbles at 2^-20
      const _Float16 h = static_cast<_Float16>(a * pow2(min(14 - ae, 127)) * down);
      act[static_cast<long long>(t) * inter + tile * 64 + lane] = __builtin_bit_cast(uint16_t, h);
      if (lane == 0) factors[tile * kMaxTokens + t] = pow2(max(ae - 2, -115));
    };
    const auto place = [&](int of, int t, int up) {
      return p.partials + (((static_cast<long long>(pair) * shares + of) * T + t) * 2 + up) * 64 + lane;
    };
    for (int t = wave; t < rows; t += kWaves) {
      const int j = (lane >> 3) & 3, l = sum_lane(t, lane);
      float g = 0.0f, u = 0.0f;
#pragma unroll
      for (int w = 0; w < kPart; ++w) {
        g += lds.red[w][j][l][t & 3];
        u += lds.red[kPart + w][j][l][t & 3];
      }
      if (shares == 1) {
        finish(t, g, u);
      } else {
        store_coherent(place(share, t, 0), g);
        store_coherent(place(share, t, 1), u);
      }
    }
    if (shares > 1 && last_of(&p.counters[H / 64 + pair], shares, &s_last)) {
      for (int t = wave; t < rows; t += kWaves) {
        float g[kMaxShares], u[kMaxShares], gs = 0.0f, us = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxShares; ++i) {
          g[i] = load_coherent(place(min(i, shares - 1), t, 0));
          u[i] = load_coherent(place(min(i, shares - 1), t, 1));
        }
#pragma unroll
        for (int i = 0; i < kMaxShares; ++i) {
          gs = i < shares ? gs + g[i] : gs;
          us = i < shares ? us + u[i] : us;
        }
        finish(t, gs, us);
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- launch 2
template <int R>
__global__ __launch_bounds__(kThreads, 4) void few_w2_kernel(FewArgs f) {
  constexpr bool kGather = R > 4;
  const pega_moe_few& p = f.p;
  __shared__ uint32_t s_tr[kWaves][2 * kSlotDwords];
  __shared__ float s_sum[kWaves][R][64];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int T = p.tokens, H = p.hidden_dim, I = p.inter;
  const int tile = blockIdx.x, split = blockIdx.y;
  const int listed = p.slots[min(lane, p.tokens * p.topk < p.local_experts ? p.tokens * p.topk : p.local_experts)];
  const int slots = __builtin_amdgcn_readfirstlane(listed);

  // this wave's share of the priced list: slots' groups at 1, then the shared expert's
  const int per = I >> 5, sh_groups = p.shared_kind != PEGA_SHARED_NONE ? p.shared_inter >> 5 : 0;
  const int cost = f.shared_cost;
  const int routed_end = slots * per, total = routed_end + sh_groups * cost;
  const int parts = f.splits * kWaves, part = split * kWaves + wave;
  const int lo = static_cast<int>(static_cast<long long>(total) * part / parts);
  const int hi = static_cast<int>(static_cast<long long>(total) * (part + 1) / parts);
  const int sh0 = (max(lo - routed_end, 0) + cost - 1) / cost;
  const int sh1 = (max(hi - routed_end, 0) + cost - 1) / cost;

  // A gathered slot's rows are its own tokens: its sums go to theirs in LDS, where they wait for the
  // wave's other slots.  Otherwise rows are tokens throughout, and the sums stay in acc.
  floatx4_t acc[4] = {};
  for (int t = 0; t < R; ++t) s_sum[wave][t][lane] = 0.0f;
  const auto leave = [&](auto r, uint32_t mask) {
    constexpr int RU = decltype(r)::value;
    add_places<RU>(acc);
#pragma unroll
    for (int i = 0; i < RU; ++i) {
      const bool some = mask != 0;
      const int t = __builtin_ctz(mask | 0x10000u) & 15;
      mask &= mask - 1;
      if (some && lane >> 4 == i >> 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s_sum[wave][t][32 * ((lane >> 3) & 1) + 8 * j + (lane & 7)] += acc[j][i & 3];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = floatx4_t{};
  };
  const auto undo = [&] {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] *= kUndo;
  };
  const auto groups = [&](const uint8_t* q, const uint16_t* scales, int K, const void* act,
                          const float* factors, uint32_t mask, int g0, int g1) {
    const int rows = kGather ? __popc(mask) : T;
    by_rows<kGather>(rows, [&](auto r) {
      constexpr int RU = decltype(r)::value;
      const int row = (lane & 15) % RU;
      const Int4View v = int4_view<RU>(q, scales, H, K, tile, act, factors, row < rows ? row : -1, rows);
      int4_groups<RU, true>(acc, v, g0, g1, 1.0f, s_tr[wave]);
      if (kGather) {
        undo();
        leave(r, mask);
      }
    });
  };
  const uint32_t everyone = (1u << T) - 1u;
  for (int at = lo; at < min(hi, routed_end);) {
    const int s = at / per, g0 = at - s * per, g1 = min(per, g0 + min(hi, routed_end) - at);
    const uint32_t slot = static_cast<uint32_t>(
        s < 63 ? __builtin_amdgcn_readlane(listed, 1 + s) : __builtin_amdgcn_readfirstlane(p.slots[1 + s]));
    const long long elems = static_cast<long long>(H) * I, expert = slot & 0xffffu;
    groups(p.w2 + expert * (elems / 2), p.w2_scales + expert * (elems / 32), I,
           p.act + static_cast<long long>(s) * T * I,
           p.act_factors + static_cast<long long>(s) * (I >> 6) * kMaxTokens, slot >> 16, g0, g1);
    at += g1 - g0;
  }
  if (p.shared_kind == PEGA_SHARED_INT4 && sh0 < sh1) {
    groups(static_cast<const uint8_t*>(p.shared_w2), p.shared_w2_scales, p.shared_inter, p.act_shared,
           p.act_shared_factors, everyone, sh0, sh1);
  }
  if (!kGather) undo();
  if (p.shared_kind == PEGA_SHARED_BF16) {
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
    bf16_steps<4, 4>(acc, wr, w_voff, ar,
                     static_cast<uint32_t>(lane & 15) * row_bytes + 16u * (lane >> 4), sh0, sh1);
    if (kGather) leave(std::integral_constant<int, 16>{}, everyone);
  }
  if (!kGather) leave(std::integral_constant<int, R>{}, everyone);
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
    const int t = o >> 6, col = o & 63;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += s_sum[w][t][col];
    if (f.splits == 1) finish(t, col, sum);
    else store_coherent(place(split, t, col), sum);
  }
  if (f.splits == 1 || !last_of(&p.counters[tile], f.splits, &s_last)) return;
  for (int o = tid; o < T * 64; o += kThreads) {
    const int t = o >> 6, col = o & 63;
    float part[PEGA_FEW_MAX_SPLITS], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PEGA_FEW_MAX_SPLITS; ++i) part[i] = load_coherent(place(min(i, f.splits - 1), t, col));
#pragma unroll
    for (int i = 0; i < PEGA_FEW_MAX_SPLITS; ++i) sum = i < f.splits ? sum + part[i] : sum;
    finish(t, col, sum);
  }
}

template <int NS, bool kDsv2>
void launch_w13(const FewArgs& f, unsigned grid, hipStream_t stream) {
  if (f.p.tokens <= 4)
    hipLaunchKernelGGL((few_w13_kernel<NS, kDsv2, 4>), dim3(grid), dim3(kThreads), 0, stream, f);
  else
    hipLaunchKernelGGL((few_w13_kernel<NS, kDsv2, 16>), dim3(grid), dim3(kThreads), 0, stream, f);
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
      !p.topk_weight || !p.topk_idx || !p.act || !p.act_factors || !p.slots || !p.partials || !p.counters ||
      (!p.softmax && !p.bias))
    return fail(kInvalidValue, "moe_few_tokens: null pointer");
  if (p.shared_kind != PEGA_SHARED_NONE && p.shared_kind != PEGA_SHARED_BF16 &&
      p.shared_kind != PEGA_SHARED_INT4)
    return fail(kInvalidValue, "moe_few_tokens: shared_kind %d", p.shared_kind);
  const bool shared = p.shared_kind != PEGA_SHARED_NONE;
  if (shared && (!p.shared_w13 || !p.shared_w2 || !p.act_shared ||
                 (p.shared_kind == PEGA_SHARED_INT4 &&
                  (!p.shared_w13_scales || !p.shared_w2_scales || !p.act_shared_factors))))
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
                        p.act_factors, p.shared_kind == PEGA_SHARED_INT4 ? p.act_shared_factors : nullptr,
                        p.shared_kind == PEGA_SHARED_INT4 ? p.shared_w13_scales : nullptr,
                        p.shared_kind == PEGA_SHARED_INT4 ? p.shared_w2_scales : nullptr};
  for (const void* v : vecs)
    if (!aligned16(v)) return fail(kNotSupported, "moe_few_tokens: buffers must be 16-byte aligned");
  // The ids and weights are written while launch 1's other workgroups read, and out by launch 2's, place
  // for place over residual at most, or over what only launch 1 reads.
  struct Span {
    const void* p;
    long long bytes;
  };
  const long long rows = 2LL * p.hidden_dim * p.tokens, routes_b = 4LL * p.tokens * p.topk;
  const long long w2 = static_cast<long long>(p.local_experts) * p.hidden_dim * p.inter;  // values
  const long long s2 = shared ? static_cast<long long>(p.hidden_dim) * p.shared_inter : 0;
  const bool s4 = p.shared_kind == PEGA_SHARED_INT4;
  const Span outs[] = {{p.topk_weight, routes_b}, {p.topk_idx, routes_b}, {p.out, rows}};
  const Span second[] = {{p.residual != p.out ? p.residual : nullptr, rows}, {p.w2, w2 / 2}, {p.w2_scales, w2 / 16},
                         {shared ? p.shared_w2 : nullptr, s4 ? s2 / 2 : 2 * s2},
                         {s4 ? p.shared_w2_scales : nullptr, s2 / 16}};
  const Span first[] = {{p.x, rows}, {p.logits, 4LL * p.tokens * p.n_experts},
                        {p.softmax ? nullptr : p.bias, 4LL * p.n_experts}, {p.w13, w2}, {p.w13_scales, w2 / 8},
                        {shared ? p.shared_w13 : nullptr, s4 ? s2 : 4 * s2},
                        {s4 ? p.shared_w13_scales : nullptr, s2 / 8}, {p.residual, rows}};
  for (int o = 0; o < 3; ++o) {
    bool meets = false;
    for (const Span& in : second) meets |= overlap(outs[o].p, outs[o].bytes, in.p, in.bytes);
    if (o < 2)
      for (const Span& in : first) meets |= overlap(outs[o].p, outs[o].bytes, in.p, in.bytes);
    for (int i = 0; i < o; ++i) meets |= overlap(outs[o].p, outs[o].bytes, outs[i].p, outs[i].bytes);
    if (meets) return fail(kInvalidValue, "moe_few_tokens: buffers overlap");
  }
  const int cu = current_cu_count();
  if (cu <= 0) return fail(kInvalidValue, "moe_few_tokens: no device");
  FewArgs f{p, 0, p.inter / 64, few_splits(p.hidden_dim), p.shared_kind == PEGA_SHARED_BF16 ? 3 : 1, 0, 0};
  if (p.shared_kind == PEGA_SHARED_BF16) f.sh_units = p.shared_inter / 8;
  if (p.shared_kind == PEGA_SHARED_INT4) f.sh_units = p.shared_inter / 64;
  const int routes = p.tokens * p.topk;
  const int slots = routes < p.local_experts ? routes : p.local_experts;
  // A CU has room for two workgroups.  Where the shared expert leaves room for a routed one per CU,
  // all that fit start at once: a few that wait for the first to end run alone then (64 experts of 2048
  // x 1408 with 8 tokens: 512 beside 44 took 37 us, 468 25).  A shared expert of more workgroups is
  // done early, and its places go to a second routed workgroup per CU.
  const int room = f.sh_units < cu ? 2 * cu - f.sh_units : 2 * cu;
  f.routed = slots * f.tiles < room ? slots * f.tiles : room;
  f.routed_first = f.routed < cu ? f.routed : cu;
  const unsigned grid = static_cast<unsigned>(f.sh_units + f.routed);
  if (p.softmax) launch_w13_slots<true>(f, grid, stream);
  else launch_w13_slots<false>(f, grid, stream);
  const int rc = launch_status("moe_few_tokens (W13)");
  if (rc != kSuccess) return rc;
  const dim3 grid2(static_cast<unsigned>(p.hidden_dim / 64), static_cast<unsigned>(f.splits));
  if (p.tokens <= 4) hipLaunchKernelGGL((few_w2_kernel<4>), grid2, dim3(kThreads), 0, stream, f);
  else hipLaunchKernelGGL((few_w2_kernel<16>), grid2, dim3(kThreads), 0, stream, f);
  return launch_status("moe_few_tokens (W2)");
}

// Dense products with 4-bit weights and group scales on MI355X (gfx950):
//
//   Y[n][m] = sum_k X[n][k] * (q[m][k] - z[m][k / g]) * s[m][k / g]
//
// X [N][K] bf16, codes q in 0..15, bf16 scales s and zero points z (8 where the checkpoint has
// none) for each group of g = 32, 64 or 128 columns, Y bf16 or fp32.
//
// A code becomes a bf16 operand without arithmetic: its four bits as the top mantissa bits of
// 1.0 are the number (16 + q) / 16.  So d = sum_k x (16 + q) / 16 - sum_k x (16 + z) / 16 over a
// group is a chain of v_mfma_f32_16x16x32_bf16, the second sum with a constant operand, and
// 16 s d is the group's share of Y: products of bf16 with exact integers, fp32 sums, one scale an
// fp32 group sum.  No weight is rounded.  (16 + q and 16 + z cancel to at most two bits of the
// fp32 sums.)  An infinite or NaN activation gives NaN in its whole row.
//
// Device layout, for tiles of 16 features (the last one padded) and steps of 128 columns (the last
// one padded): per tile and step 64 lanes' 16 bytes, lane (c, h) = (lane % 16, lane / 16) holding
// feature c, word j the columns 32 j + 8 h .. + 7 of the step, the order in which the instruction
// takes them; in a word the even columns' codes are nibbles 0..3 and the odd ones' nibbles 4..7,
// rotated left by three bits, so that each pair's two operands are one masked word.  Per tile,
// step and feature the groups' scales (2 bytes each), or with zero points 4 bytes each: the scale
// and the bf16 number -(16 + z) / 16.
#include "common.h"
#include "pega_moe.h"

namespace pega {
namespace {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_t;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4_t;

constexpr int kStep = 128;                     // columns of a step
constexpr uint32_t kOutOfRange = 0x80000000u;  // voffset that fails every range check

__host__ __device__ constexpr int meta_bytes(int group, bool zeros) {  // of a feature's step
  return kStep / group * (zeros ? 4 : 2);
}

struct W4Args {
  const uint8_t* codes;
  const uint8_t* meta;
  const uint16_t* x;
  void* y;
  int M, N, K;  // features, rows of X, columns
  int f32;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0),
                                           static_cast<int>(bytes), 0x00020000);
}

// Eight codes as (16 + q) / 16.
__device__ __forceinline__ bf16x8_t expand(uint32_t w) {
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = (__builtin_amdgcn_alignbit(w, w, 4 * i) & 0x00780078u) | 0x3F803F80u;
  return __builtin_bit_cast(bf16x8_t, v);
}
__device__ __forceinline__ bf16x8_t repeat(uint32_t pair) {
  const u32x4_t v = {pair, pair, pair, pair};
  return __builtin_bit_cast(bf16x8_t, v);
}
__device__ __forceinline__ floatx4_t mfma(u32x4_t a, bf16x8_t b, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), b, c, 0, 0, 0);
}

// ---------------------------------------------------------------- device layout
__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t* __restrict__ packed,
                                                      const uint16_t* __restrict__ scales,
                                                      const uint8_t* __restrict__ zeros,
                                                      uint8_t* __restrict__ codes,
                                                      uint8_t* __restrict__ meta, int M, int K,
                                                      int group, long long units) {
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= units) return;
  const int steps = ceil_div(K, kStep);
  const int lane = static_cast<int>(at & 63), c = lane & 15, h = lane >> 4;
  const long long ts = at >> 6;
  const int s = static_cast<int>(ts % steps);
  const int m = static_cast<int>(ts / steps) * 16 + c;
  u32x4_t out = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = s * kStep + 32 * j + 8 * h;
    uint32_t q = 0;
    if (m < M && k < K)
      q = *reinterpret_cast<const uint32_t*>(packed + static_cast<long long>(m) * (K / 2) + k / 2);
    uint32_t even = q & 0x0f0f0f0fu, odd = (q >> 4) & 0x0f0f0f0fu;
    even = (even | even >> 4) & 0x00ff00ffu;  // nibbles of bytes 0, 1 and 2, 3 side by side
    odd = (odd | odd >> 4) & 0x00ff00ffu;
    even = (even | even >> 8) & 0xffffu;
    odd = (odd | odd >> 8) & 0xffffu;
    const uint32_t w = even | odd << 16;
    out[j] = w << 3 | w >> 29;
  }
  *reinterpret_cast<u32x4_t*>(codes + at * 16) = out;
  const int per = kStep / group, groups = K / group;
  if (h < per) {
    const int grp = s * per + h;
    const bool ok = m < M && grp < groups;
    const long long from = static_cast<long long>(m) * groups + grp;
    const uint16_t scale = ok ? scales[from] : 0;
    const long long to = (ts * 16 + c) * per + h;
    if (zeros) {
      const float z = ok ? static_cast<float>(zeros[from]) : 0.0f;
      reinterpret_cast<uint32_t*>(meta)[to] =
          scale | static_cast<uint32_t>(f2bf(-(16.0f + z) * 0.0625f)) << 16;
    } else {
      reinterpret_cast<uint16_t*>(meta)[to] = scale;
    }
  }
}

// ---------------------------------------------------------------- few rows
// A workgroup per 16 MR features and 16 RB rows; its waves share K's steps.  x is the
// instruction's first operand, so a lane's sums are of its own feature and it needs that feature's
// scales alone.  D steps are in flight.
template <int G, bool kZeros, int MR, int RB>
struct W4Step {
  static constexpr int kWords = (meta_bytes(G, kZeros) + 3) / 4;
  u32x4_t w[MR];
  uint32_t meta[MR][kWords];
  u32x4_t x[RB][4];
};

template <int G, bool kZeros, int MR, int RB, int WV, int D>
__global__ __launch_bounds__(64 * WV) void w4_stream_kernel(W4Args p) {
  constexpr int kPer = kStep / G, kMeta = meta_bytes(G, kZeros);
  using Step = W4Step<G, kZeros, MR, RB>;
  __shared__ __align__(16) floatx4_t s_red[WV][MR * RB][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, h = lane >> 4;
  const int K = p.K, steps = ceil_div(K, kStep);
  const int tiles = ceil_div(p.M, 16), t0 = blockIdx.x * MR, n0 = blockIdx.y * (16 * RB);
  const int live = min(MR, tiles - t0), rows = min(16 * RB, p.N - n0);
  const uint32_t w_tile = static_cast<uint32_t>(steps) * 1024u;
  const uint32_t m_tile = static_cast<uint32_t>(steps) * (16u * kMeta);
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(p.codes + static_cast<long long>(t0) * w_tile, live * w_tile);
  const __amdgpu_buffer_rsrc_t mr_ = make_rsrc(p.meta + static_cast<long long>(t0) * m_tile, live * m_tile);
  const uint32_t x_row = static_cast<uint32_t>(K) * 2u;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x + static_cast<long long>(n0) * K, rows * x_row);

  const auto load_step = [&](Step& r, int s) {
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      r.w[m] = __builtin_amdgcn_raw_buffer_load_b128(
          wr, static_cast<int>(16u * lane + m * w_tile), s * 1024, 0);
      const int at = static_cast<int>(static_cast<uint32_t>(c * kMeta) + m * m_tile);
      const int from = s * (16 * kMeta);
      if constexpr (kMeta == 2) {
        r.meta[m][0] = __builtin_amdgcn_raw_buffer_load_b16(mr_, at, from, 0);
      } else if constexpr (kMeta == 4) {
        r.meta[m][0] = __builtin_amdgcn_raw_buffer_load_b32(mr_, at, from, 0);
      } else if constexpr (kMeta == 8) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(mr_, at, from, 0);
        r.meta[m][0] = v[0], r.meta[m][1] = v[1];
      } else {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(mr_, at, from, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.meta[m][i] = v[i];
      }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // columns past the last one are another row's
        const uint32_t at = static_cast<uint32_t>(16 * b + c) * x_row + 64u * j + 16u * h;
        r.x[b][j] = __builtin_amdgcn_raw_buffer_load_b128(
            xr, static_cast<int>(s * kStep + 32 * j < K ? at : kOutOfRange), s * (2 * kStep), 0);
      }
  };
  floatx4_t acc[MR][RB] = {};
  const auto compute = [&](const Step& r) {
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int g = 0; g < kPer; ++g) {
        float scale;
        uint32_t bias = 0xBFC0BFC0u;  // -(16 + 8) / 16
        if constexpr (kZeros) {
          const uint32_t v = r.meta[m][g];
          scale = bf_lo(v);
          bias = (v & 0xffff0000u) | v >> 16;
        } else {
          scale = g & 1 ? bf_hi(r.meta[m][g / 2]) : bf_lo(r.meta[m][g / 2]);
        }
        floatx4_t d[RB] = {};
#pragma unroll
        for (int j = g * (4 / kPer); j < (g + 1) * (4 / kPer); ++j) {
          const bf16x8_t w = expand(r.w[m][j]);
#pragma unroll
          for (int b = 0; b < RB; ++b) d[b] = mfma(r.x[b][j], repeat(bias), d[b]);
#pragma unroll
          for (int b = 0; b < RB; ++b) d[b] = mfma(r.x[b][j], w, d[b]);
        }
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][b][i] = __builtin_fmaf(scale, d[b][i], acc[m][b][i]);
      }
  };

  const int s0 = (steps * wave) / WV, s1 = (steps * (wave + 1)) / WV;
  if (s0 < s1) {
    Step slot[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      load_step(slot[j], min(s0 + j, s1 - 1));
      __builtin_amdgcn_sched_barrier(0);
    }
    int s = s0;
    for (; s + D <= s1; s += D) {
#pragma unroll
      for (int j = 0; j < D; ++j) {
        compute(slot[j]);
        load_step(slot[j], min(s + j + D, s1 - 1));  // past the share's end: fetched again, never used
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int j = 0; j < D - 1; ++j)
      if (s + j < s1) compute(slot[j]);
  }
  // the waves' sums in wave order
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int b = 0; b < RB; ++b) s_red[wave][m * RB + b][lane] = acc[m][b];
  __syncthreads();
  for (int t = wave; t < MR * RB; t += WV) {
    floatx4_t sum = s_red[0][t][lane];
#pragma unroll
    for (int w = 1; w < WV; ++w) {
      const floatx4_t v = s_red[w][t][lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += v[i];
    }
    const int m = 16 * (t0 + t / RB) + c;
    if (m >= p.M) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * (t % RB) + 4 * h + i;
      if (r >= rows) break;
      const long long at = static_cast<long long>(n0 + r) * p.M + m;
      const float v = 16.0f * sum[i];
      if (p.f32) static_cast<float*>(p.y)[at] = v;
      else static_cast<uint16_t*>(p.y)[at] = f2bf(v);
    }
  }
}

template <int G, bool kZeros, int MR, int RB, int WV, int D>
void launch_stream(const W4Args& p, hipStream_t stream) {
  hipLaunchKernelGGL((w4_stream_kernel<G, kZeros, MR, RB, WV, D>),
                     dim3(ceil_div(ceil_div(p.M, 16), MR), ceil_div(p.N, 16 * RB)), dim3(64 * WV), 0,
                     stream, p);
}

template <int G, bool kZeros>
void launch_w4(const W4Args& p, hipStream_t stream) {
  if (p.N <= 16) launch_stream<G, kZeros, 1, 1, 4, 4>(p, stream);
  else launch_stream<G, kZeros, 2, 2, 4, 2>(p, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_sizes(const char* name, int M, int K, int group) {
  if (M <= 0 || K <= 0) return fail(kInvalidValue, "%s: bad sizes (%d x %d)", name, M, K);
  if (group != 32 && group != 64 && group != 128)
    return fail(kNotSupported, "%s: groups of 32, 64 or 128 columns, got %d", name, group);
  if (K % group != 0) return fail(kInvalidValue, "%s: %d columns are not whole groups of %d", name, K, group);
  if (K > (1 << 20) || M > (1 << 28))
    return fail(kNotSupported, "%s: at most 2^20 columns and 2^28 features, got %d x %d", name, M, K);
  return kSuccess;
}

}  // namespace
}  // namespace pega

using namespace pega;

// No reference counterpart: the reference's 4-bit weights are its experts' alone.
PEGA_API int pega_w4_pack(const uint8_t* packed, const uint16_t* scales, const uint8_t* zeros,
                          uint8_t* codes, uint8_t* meta, int out_dim, int in_dim, int group_size,
                          hipStream_t stream) {
  if (const int rc = check_sizes("w4_pack", out_dim, in_dim, group_size)) return rc;
  if (!packed || !scales || !codes || !meta) return fail(kInvalidValue, "w4_pack: null pointer");
  if ((reinterpret_cast<uintptr_t>(packed) & 3u) || (reinterpret_cast<uintptr_t>(scales) & 1u) ||
      !aligned16(codes) || !aligned16(meta))
    return fail(kNotSupported, "w4_pack: packed must be 4-byte, codes and meta 16-byte aligned");
  const long long tiles = ceil_div(out_dim, 16), steps = ceil_div(in_dim, kStep);
  const long long n = static_cast<long long>(out_dim) * in_dim, units = tiles * steps * 64;
  const long long metas = tiles * steps * 16 * meta_bytes(group_size, zeros != nullptr);
  struct Span { const void* p; long long bytes; };
  const Span outs[2] = {{codes, units * 16}, {meta, metas}};
  const Span ins[3] = {{packed, n / 2}, {scales, 2 * (n / group_size)}, {zeros, n / group_size}};
  for (int o = 0; o < 2; ++o)
    for (int i = 0; i < 3; ++i)
      if (overlap(outs[o].p, outs[o].bytes, ins[i].p, ins[i].bytes))
        return fail(kInvalidValue, "w4_pack: an output overlaps an input");
  if (overlap(codes, units * 16, meta, metas)) return fail(kInvalidValue, "w4_pack: two outputs overlap");
  // 2^24 workgroups a launch: below 2^32 threads
  if (units > (1LL << 24) * 256)
    return fail(kNotSupported, "w4_pack: %d x %d weights are too many for one launch", out_dim, in_dim);
  hipLaunchKernelGGL(w4_pack_kernel, dim3(static_cast<unsigned>((units + 255) / 256)), dim3(256), 0, stream,
                     packed, scales, zeros, codes, meta, out_dim, in_dim, group_size, units);
  return launch_status("w4_pack");
}

PEGA_API int pega_w4_gemm(const uint8_t* codes, const uint8_t* meta, bool has_zeros, int group_size,
                          const uint16_t* X, void* Y, bool y_is_f32, int M, int N, int K,
                          hipStream_t stream) {
  if (const int rc = check_sizes("w4_gemm", M, K, group_size)) return rc;
  if (N < 0) return fail(kInvalidValue, "w4_gemm: %d rows", N);
  if (N == 0) return kSuccess;  // empty tensors have no address
  if (!codes || !meta || !X || !Y) return fail(kInvalidValue, "w4_gemm: null pointer");
  if (!aligned16(codes) || !aligned16(meta) || !aligned16(X) || !aligned16(Y))
    return fail(kNotSupported, "w4_gemm: buffers must be 16-byte aligned");
  if (N > 16 * 65535) return fail(kNotSupported, "w4_gemm: at most %d rows, got %d", 16 * 65535, N);
  const long long units = 1LL * ceil_div(M, 16) * ceil_div(K, kStep);
  const long long y_bytes = (y_is_f32 ? 4LL : 2LL) * N * M;
  if (overlap(Y, y_bytes, X, 2LL * N * K) || overlap(Y, y_bytes, codes, units * 1024) ||
      overlap(Y, y_bytes, meta, units * 16 * meta_bytes(group_size, has_zeros)))
    return fail(kInvalidValue, "w4_gemm: the output overlaps an input");
  const W4Args p{codes, meta, X, Y, M, N, K, y_is_f32};
  switch (group_size * 2 + has_zeros) {
    case 64: launch_w4<32, false>(p, stream); break;
    case 65: launch_w4<32, true>(p, stream); break;
    case 128: launch_w4<64, false>(p, stream); break;
    case 129: launch_w4<64, true>(p, stream); break;
    case 256: launch_w4<128, false>(p, stream); break;
    default: launch_w4<128, true>(p, stream); break;
  }
  return launch_status("w4_gemm");
}

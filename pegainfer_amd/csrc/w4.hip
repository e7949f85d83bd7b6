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
// fp32 group sum.  No weight is rounded.  What is rounded are sums of x (16 + q) and x (16 + z), so the error is
// relative to sum |x| (16 + q + 16 + z) |s|: a group whose codes all are its zero point gives about 2^-23 of that
// and not zero.  An infinite or NaN activation gives NaN in its whole row.  So may finite ones of 2^117 and more
// (2^119 where no zero point is above 15), with which sums of up to 128 |x| (16 + z) / 16 pass fp32's range.
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

// Eight codes as (16 + q) / 16.  The constants stand in registers that the compiler cannot see through: as
// literals they would cost an instruction of their own each.
struct Masks {
  uint32_t code = 0x00780078u, one = 0x3F803F80u;
  __device__ __forceinline__ Masks() { asm volatile("" : "+v"(code), "+v"(one)); }
};
__device__ __forceinline__ bf16x8_t expand(uint32_t w, const Masks& k) {
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (__builtin_amdgcn_alignbit(w, w, 4 * i) & k.code) | k.one;
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
// Once, at load time.  A load of a wave takes 16 bytes of each of 16 features: 163840 x 7168 in 339 us, 1.4 times a
// copy of its bytes.
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
// Bound by the weights' stream from memory: a lane's 16 bytes are all it needs of a step's codes, read once and
// never staged.  One row of 163840 x 7168 (606 MB): 101 us, 6.0 TB/s.  One of 4096 x 7168 (16.5 MB): 5.6 us of
// kernel, one round trip of the loads and the join, which is why eight waves share K there and few features go to a
// workgroup; with many features more of them to a workgroup read each row of X less often.
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
  const Masks masks;
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
          const bf16x8_t w = expand(r.w[m][j], masks);
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

// ---------------------------------------------------------------- many rows
// A workgroup of WM x WN waves owns 16 TM WM features x 16 TN WN rows, each wave 16 TM of the features and
// 16 TN of the rows, for all of K; a stage of the ring in LDS holds a step of X, codes and scales,
// brought in by loads straight to LDS, one barrier a step.  A row of X has its 16-byte pieces at slot
// piece ^ (row % 16), which spreads sixteen lanes' fragment reads over all 64 banks.
// sum_k x over a group (times -24 / 16 without zero points) is one more chain a row block, with a
// constant operand, which the waves share out a step ahead; its features' chains start from it.
// (A chain in every wave instead of the shared sums: 9% slower.)
// Bound by instruction issue: each code is expanded by every wave that has its features, so wide tiles, whose waves
// take many rows, spread that over more products.  4096 rows of 4096 x 7168, groups of 128, zero points: 253 us, 950
// TFLOP/s, matrix cores busy 42% and vector units 55% of the cycles.  333 rows of 9728 x 2560: 31 us, one workgroup a CU
// that reads LDS and multiplies in turn; 48 rows of 163840 x 2048: 62 us, 3.3 TB/s, two workgroups a CU.
template <int G_, bool kZeros_, int WM_, int WN_, int TM_, int TN_, int NS_>
struct W4Tile {
  static constexpr int G = G_, WM = WM_, WN = WN_, TM = TM_, TN = TN_, NS = NS_;
  static constexpr bool kZeros = kZeros_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN;
  static constexpr int kMeta = meta_bytes(G, kZeros), kMetaBytes = BM * kMeta;
  static constexpr int kXLoads = BN / 4, kWLoads = BM / 16, kMLoads = (kMetaBytes + 255) / 256;
  static constexpr int PX = (kXLoads + kWaves - 1) / kWaves;  // loads of a wave and stage
  static constexpr int PW = (kWLoads + kWaves - 1) / kWaves, PM = (kMLoads + kWaves - 1) / kWaves;
  static constexpr int P = PX + PW + PM;
  static constexpr int kX = BN * 256, kW = BM * 64;
  static constexpr int kStage = kX + kW + kMLoads * 256, kRing = NS * kStage;
  static constexpr int kSum = kStep / G * BN * 4;  // a step's group sums of X
  static constexpr int kLds = kRing + 2 * kSum;
  static_assert(NS >= 3 && kLds <= 160 * 1024, "tile shape");
};

template <typename S>
__global__ __launch_bounds__(S::kThreads) void w4_tile_kernel(W4Args p) {
  constexpr int TM = S::TM, TN = S::TN, NS = S::NS, kMeta = S::kMeta, kPer = kStep / S::G;
  __shared__ __align__(1024) uint8_t smem[S::kLds];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % S::WM, wn = wave / S::WM;
  const int c = lane & 15, h = lane >> 4;
  int tx = blockIdx.x, ty = blockIdx.y;
  xcd_tile(tx, ty, gridDim.y);
  const int K = p.K, steps = ceil_div(K, kStep);
  const int t0 = tx * (S::BM / 16), n0 = ty * S::BN;
  const int live = min(S::BM / 16, ceil_div(p.M, 16) - t0), rows = min(S::BN, p.N - n0);
  const uint32_t w_tile = static_cast<uint32_t>(steps) * 1024u;
  const uint32_t m_tile = static_cast<uint32_t>(steps) * (16u * kMeta);
  const uint32_t x_row = static_cast<uint32_t>(K) * 2u;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) uint8_t*)smem));

  u32x4_t x_rsrc = rsrc_words(p.x + static_cast<long long>(n0) * K, static_cast<uint32_t>(rows) * x_row);
  u32x4_t w_rsrc = rsrc_words(p.codes + static_cast<long long>(t0) * w_tile, static_cast<uint32_t>(live) * w_tile);
  u32x4_t m_rsrc = rsrc_words(p.meta + static_cast<long long>(t0) * m_tile, static_cast<uint32_t>(live) * m_tile);
  const uint32_t x_size = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x_rsrc[2])));
  const uint32_t w_size = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(w_rsrc[2])));
  const uint32_t m_size = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(m_rsrc[2])));
  // This wave's loads of a stage (a repeat brings the same).  Rows past the last one and tiles past the
  // last one are past their operands' ranges, and come as zeros.
  uint32_t x_voff[S::PX], w_voff[S::PW], m_voff[S::PM], x_dst[S::PX], w_dst[S::PW], m_dst[S::PM];
  int x_col[S::PX];
#pragma unroll
  for (int j = 0; j < S::PX; ++j) {
    const int i = min(wave * S::PX + j, S::kXLoads - 1);
    const int r = 4 * i + (lane >> 4), piece = (lane & 15) ^ (r & 15);
    x_dst[j] = lds0 + 1024u * static_cast<uint32_t>(i);
    x_col[j] = 8 * piece;
    x_voff[j] = static_cast<uint32_t>(r) * x_row + 16u * static_cast<uint32_t>(piece);
  }
#pragma unroll
  for (int j = 0; j < S::PW; ++j) {
    const int i = min(wave * S::PW + j, S::kWLoads - 1);
    w_dst[j] = lds0 + S::kX + 1024u * static_cast<uint32_t>(i);
    w_voff[j] = static_cast<uint32_t>(i) * w_tile + 16u * lane;
  }
#pragma unroll
  for (int j = 0; j < S::PM; ++j) {
    const int i = min(wave * S::PM + j, S::kMLoads - 1), b = i * 256 + lane * 4;
    m_dst[j] = lds0 + S::kX + S::kW + 256u * static_cast<uint32_t>(i);
    m_voff[j] = b < S::kMetaBytes ? static_cast<uint32_t>(b / (16 * kMeta)) * m_tile +
                                        static_cast<uint32_t>(b % (16 * kMeta))
                                  : kOutOfRange;
  }
  // Stages come in turn; past the last one the operands have no bytes, and zeros come that nothing uses.
  const auto stage_in = [&](int s, uint32_t at) {
    x_rsrc[2] = s < steps ? x_size : 0u;
    w_rsrc[2] = s < steps ? w_size : 0u;
    m_rsrc[2] = s < steps ? m_size : 0u;
    const int cols = K - s * kStep;  // columns past the last one are another row's
#pragma unroll
    for (int j = 0; j < S::PX; ++j)
      dma_b128(x_rsrc, x_dst[j] + at, x_col[j] < cols ? x_voff[j] : kOutOfRange, static_cast<uint32_t>(s) * 256u);
#pragma unroll
    for (int j = 0; j < S::PW; ++j)
      dma_b128(w_rsrc, w_dst[j] + at, w_voff[j], static_cast<uint32_t>(s) * 1024u);
#pragma unroll
    for (int j = 0; j < S::PM; ++j)
      dma_b32(m_rsrc, m_dst[j] + at, m_voff[j], static_cast<uint32_t>(s) * (16u * kMeta));
  };

  floatx4_t acc[TM][TN] = {};
  const Masks masks;
  struct Rows {
    u32x4_t v[4];
  };
  const auto x_rows = [&](uint32_t at, int b) {  // row block b of the workgroup's
    Rows x;
    const uint8_t* xl = smem + at + (16 * b + c) * 256;
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = *reinterpret_cast<const u32x4_t*>(xl + 16 * ((4 * j + h) ^ c));
    return x;
  };
  // a step's group sums of X, row blocks in turn by wave: block `wave` + i kWaves
  constexpr int kSumBlocks = (S::BN / 16 + S::kWaves - 1) / S::kWaves;
  const auto sum_rows = [&](uint32_t at, int i) { return x_rows(at, min(wave + i * S::kWaves, S::BN / 16 - 1)); };
  const auto sum_up = [&](const Rows& x, uint32_t sums, int i) {
    const bf16x8_t ones = repeat(S::kZeros ? 0x3F803F80u : 0xBFC0BFC0u);  // 1, or -(16 + 8) / 16
    constexpr int kJ = 4 / kPer;
    const int b = wave + i * S::kWaves;
#pragma unroll
    for (int g = 0; g < kPer; ++g) {
      floatx4_t sum = {};
#pragma unroll
      for (int j = g * kJ; j < (g + 1) * kJ; ++j) sum = mfma(x.v[j], ones, sum);
      // the same in all 16 columns, which all write it: no branch cuts the step in two
      if (S::BN / 16 % S::kWaves == 0 || b < S::BN / 16)
        *reinterpret_cast<floatx4_t*>(smem + sums + 4 * (g * S::BN + 16 * b + 4 * h)) = sum;
    }
  };
  // What a step starts with, read from LDS while the step before is computed.
  constexpr int kWords = (kMeta + 3) / 4;
  struct First {
    u32x4_t q[TM];
    uint32_t meta[TM][kWords];
    Rows x;
  };
  const auto read_first = [&](First& f, uint32_t at) {
    const uint8_t* wl = smem + at + S::kX + wm * (TM * 1024) + 16 * lane;
    const uint8_t* ml = smem + at + S::kX + S::kW + wm * (TM * 16 * kMeta) + c * kMeta;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      f.q[t] = *reinterpret_cast<const u32x4_t*>(wl + 1024 * t);
      const uint8_t* m = ml + t * (16 * kMeta);
      if constexpr (kMeta == 2) {
        f.meta[t][0] = *reinterpret_cast<const uint16_t*>(m);
      } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) f.meta[t][i] = reinterpret_cast<const uint32_t*>(m)[i];
      }
    }
    f.x = x_rows(at, wn * TN);
  };
  // A step, on the stage at `at`, with what is in f; f and the group sums for the stage at `then`.
  const auto compute = [&](First& f, uint32_t at, uint32_t sums, uint32_t then, uint32_t ahead) {
    constexpr int kJ = 4 / kPer;
    const auto sum_of = [&](int b, int g) {
      return *reinterpret_cast<const floatx4_t*>(smem + sums + 4 * (g * S::BN + 16 * (wn * TN + b) + 4 * h));
    };
    bf16x8_t w[TM][4];
    float scale[TM][kPer], zero[TM][kPer];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[t][j] = expand(f.q[t][j], masks);
#pragma unroll
      for (int g = 0; g < kPer; ++g) {
        if constexpr (S::kZeros) scale[t][g] = bf_lo(f.meta[t][g]), zero[t][g] = bf_hi(f.meta[t][g]);
        else scale[t][g] = g & 1 ? bf_hi(f.meta[t][g / 2]) : bf_lo(f.meta[t][g / 2]), zero[t][g] = 0.0f;
      }
    }
    Rows x = f.x;
    floatx4_t last[TM];  // the last group's sums of the row block before, not yet in acc
    const auto settle = [&](const floatx4_t* d, int b, int g) {
#pragma unroll
      for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][b][i] = __builtin_fmaf(scale[t][g], d[t][i], acc[t][b][i]);
    };
    floatx4_t sum = sum_of(0, 0);
    Rows ys = sum_rows(then, 0);
#pragma unroll
    for (int b = 0; b < TN; ++b) {
      Rows coming;
      if (b + 1 < TN) coming = x_rows(at, wn * TN + b + 1);
      else read_first(f, then);
#pragma unroll
      for (int g = 0; g < kPer; ++g) {
        floatx4_t d[TM];
#pragma unroll
        for (int t = 0; t < TM; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) d[t][i] = S::kZeros ? sum[i] * zero[t][g] : sum[i];
        if (g + 1 < kPer) sum = sum_of(b, g + 1);
        else if (b + 1 < TN) sum = sum_of(b + 1, 0);
#pragma unroll
        for (int j = g * kJ; j < (g + 1) * kJ; ++j)
#pragma unroll
          for (int t = 0; t < TM; ++t) d[t] = mfma(x.v[j], w[t][j], d[t]);
        if (b + g > 0) settle(last, g > 0 ? b : b - 1, g > 0 ? g - 1 : kPer - 1);
#pragma unroll
        for (int t = 0; t < TM; ++t) last[t] = d[t];
      }
      if (b + 1 < TN) x = coming;
      // behind the first products of this step, the sums of the next one
      if (b < kSumBlocks) {
        sum_up(ys, ahead, b);
        if (b + 1 < kSumBlocks) ys = sum_rows(then, b + 1);
      }
    }
    static_assert(kSumBlocks <= TN, "tile shape");
    settle(last, TN - 1, kPer - 1);
  };

  const auto next = [](uint32_t at) { return at + S::kStage == S::kRing ? 0u : at + S::kStage; };
  uint32_t in = 0, out = 0;  // where the next stage goes, and which is next to be used
  for (int s = 0; s < NS - 1; ++s) {
    stage_in(s, in);
    in = next(in);
  }
  uint32_t sums = S::kRing;
  vm_wait<(NS - 2) * S::P>();
  lds_barrier();
#pragma unroll
  for (int i = 0; i < kSumBlocks; ++i) sum_up(sum_rows(0, i), sums, i);
  First first;
  read_first(first, 0);
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    vm_wait<(NS - 3) * S::P>();  // the stage after this one
    lds_barrier();
    stage_in(s + NS - 1, in);
    in = next(in);
    const uint32_t then = next(out), ahead = 2 * S::kRing + S::kSum - sums;
    compute(first, out, sums, then, ahead);
    out = then, sums = ahead;
  }
  vm_wait<0>();
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int m = 16 * (t0 + wm * TM + t) + c;
    if (m >= p.M) continue;
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * (wn * TN + b) + 4 * h + i;
        if (r >= rows) continue;
        const long long at = static_cast<long long>(n0 + r) * p.M + m;
        const float v = 16.0f * acc[t][b][i];
        if (p.f32) static_cast<float*>(p.y)[at] = v;
        else static_cast<uint16_t*>(p.y)[at] = f2bf(v);
      }
  }
}

template <typename S>
void launch_tile(const W4Args& p, hipStream_t stream) {
  hipLaunchKernelGGL(w4_tile_kernel<S>, dim3(ceil_div(p.M, S::BM), ceil_div(p.N, S::BN)), dim3(S::kThreads), 0,
                     stream, p);
}

// ---------------------------------------------------------------- which kernel
// A call's time in us, over 1024 .. 163840 features, 2048 .. 7168 columns and 1 .. 2048 rows of each
// form alone: start + steps * (step + fill * step_rows + (more + fill * more_rows) * (w - w0)), with w
// workgroups a CU (above w0) and a workgroup's rows filled to `fill`.  The form that this puts first
// is within 3% of the fastest one on average, 34% at most (one row of 1024 x 2048, groups of 32 with zero
// points: 4.3 us where the first form takes 3.2; the streaming forms have one set of costs for all groups).  Examples,
// groups of 128: one row of 4096 x 7168 5.0 us with <1, 1, 8, 2>, 11.6 with <4, 1, 4, 2>; one of 163840 x
// 2048 35.8 with the latter, 77 with the former; 48 rows of those 62 with the tile of 48 rows, 94 with
// <4, 4, 4, 1>; 2048 rows of 4096 x 7168 132 with the tile of 256 x 128, 156 with 128 x 64, of 1024
// rows 101 and 81.  Groups of 32 take half as long again in the tile kernel, whose vector work grows with
// the groups; its widest tile would spill registers with them (with groups of 64 and zero points it spills one).
// Two streaming forms have one wave a SIMD with groups of 32, of 256 registers and a few more: <4, 1, 4, 2> with
// zero points (one row of 32768 x 2048 12.7 us, with groups of 128 10.2) and <4, 4, 4, 1> without.
struct Form {
  int bm, bn;
  bool whole;  // half of the cost is by whole rounds of workgroups
  float start, step, step_rows, more, more_rows, w0;
};
constexpr Form kForms[] = {
    {16, 16, false, 5.9f, 0.0f, 0.03f, 0.079f, 0.123f, 0.90f},    // stream <1, 1, 8, 2>
    {32, 16, false, 3.2f, 0.055f, 0.064f, 0.114f, 0.061f, 0.71f}, // stream <2, 1, 4, 2>
    {64, 16, false, 3.4f, 0.139f, 0.002f, 0.216f, 0.0f, 0.70f},   // stream <4, 1, 4, 2>
    {64, 32, false, 3.4f, 0.197f, 0.073f, 0.234f, 0.09f, 0.74f},  // stream <4, 2, 4, 1>
    {64, 64, false, 4.3f, 0.332f, 0.18f, 0.356f, 0.235f, 0.83f},  // stream <4, 4, 4, 1>
    {128, 48, false, 4.1f, 0.737f, 0.0f, 0.588f, 0.0f, 0.90f},    // tile <4, 1, 2, 3>
    {128, 64, true, 4.8f, 0.857f, 0.0f, 0.73f, 0.0f, 1.17f},      // tile <4, 1, 2, 4>
    {256, 64, true, 4.4f, 1.231f, 0.0f, 1.547f, 0.0f, 0.88f},     // tile <8, 1, 2, 4>
    {128, 128, true, 4.5f, 1.292f, 0.0f, 1.522f, 0.0f, 0.92f},    // tile <4, 2, 2, 4>
    {256, 128, true, 6.9f, 1.948f, 0.0f, 2.495f, 0.0f, 0.81f},    // tile <4, 2, 4, 4>
};
constexpr int kStreams = 5, kFormCount = sizeof(kForms) / sizeof(kForms[0]);

int choose_form(int M, int N, int K, int group) {
  int best = 0;
  float best_time = 0.0f;
  const float steps = static_cast<float>(ceil_div(K, kStep));
  for (int i = 0; i < kFormCount - (group == 32 ? 1 : 0); ++i) {
    const Form& f = kForms[i];
    const int blocks = ceil_div(N, f.bn);
    const float groups = static_cast<float>(ceil_div(M, f.bm)) * static_cast<float>(blocks) / 256.0f;
    const float w = f.whole ? 0.5f * (groups + __builtin_ceilf(groups)) : groups;
    const float fill = static_cast<float>(N) / (static_cast<float>(blocks) * static_cast<float>(f.bn));
    const float over = w > f.w0 ? w - f.w0 : 0.0f;
    const float step = f.step + fill * f.step_rows + (f.more + fill * f.more_rows) * over;
    const float time = f.start + steps * step * (group == 32 && i >= kStreams ? 1.5f : 1.0f);
    if (i == 0 || time < best_time) best = i, best_time = time;
  }
  return best;
}

template <int G, bool kZeros>
void launch_w4(const W4Args& p, hipStream_t stream) {
  switch (choose_form(p.M, p.N, p.K, G)) {
    case 0: launch_stream<G, kZeros, 1, 1, 8, 2>(p, stream); break;
    case 1: launch_stream<G, kZeros, 2, 1, 4, 2>(p, stream); break;
    case 2: launch_stream<G, kZeros, 4, 1, 4, 2>(p, stream); break;
    case 3: launch_stream<G, kZeros, 4, 2, 4, 1>(p, stream); break;
    case 4: launch_stream<G, kZeros, 4, 4, 4, 1>(p, stream); break;
    case 5: launch_tile<W4Tile<G, kZeros, 4, 1, 2, 3, 3>>(p, stream); break;
    case 6: launch_tile<W4Tile<G, kZeros, 4, 1, 2, 4, 3>>(p, stream); break;
    case 7: launch_tile<W4Tile<G, kZeros, 8, 1, 2, 4, 3>>(p, stream); break;
    case 8: launch_tile<W4Tile<G, kZeros, 4, 2, 2, 4, 3>>(p, stream); break;
    default:
      if constexpr (G != 32) launch_tile<W4Tile<G, kZeros, 4, 2, 4, 4, 3>>(p, stream);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_sizes(const char* name, int M, int K, int group) {
  if (M <= 0 || K <= 0) return fail(kInvalidValue, "%s: bad sizes (%d x %d)", name, M, K);
  if (group != 32 && group != 64 && group != 128)
    return fail(kNotSupported, "%s: groups of 32, 64 or 128 columns, got %d", name, group);
  if (K % group != 0) return fail(kInvalidValue, "%s: %d columns are not whole groups of %d", name, K, group);
  if (K > (1 << 20) || M > (1 << 26))
    return fail(kNotSupported, "%s: at most 2^20 columns and 2^26 features, got %d x %d", name, M, K);
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
  if (!aligned16(codes) || !aligned16(meta) || !aligned16(X) ||
      (reinterpret_cast<uintptr_t>(Y) & (y_is_f32 ? 3u : 1u)))
    return fail(kNotSupported, "w4_gemm: X and the weight must be 16-byte aligned, Y by its type");
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

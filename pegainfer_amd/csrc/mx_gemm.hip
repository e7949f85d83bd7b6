// Products of microscaled rows (mx_format.h) on MI355X (gfx950):
//
//   Y[n][m] = bf16( sum_k X[n][k] * W[m][k] ),   W [M][K] MXFP4, X [N][K] MXFP8 or MXFP4
//
// on v_mfma_scale_f32_16x16x128_f8f6f4, which takes codes and scale bytes as they are stored:
// 16 features (operand A) by 16 rows (operand B) by 128 k.  Lane (c, g), c = lane % 16 and
// g = lane / 16, holds row c of its operand: of E2M1 codes the 16 bytes of k 32 g .. 32 g + 31, of
// E4M3 codes the 16 bytes from k 16 g on and those from k 64 + 16 g on; its scale byte is that of
// the block k 32 g .. 32 g + 31 either way.  The lane's four sums are features 4 g .. 4 g + 3 of
// row c of X.  Sums are fp32 from one instruction to the next; inside one, products of E4M3 codes
// are aligned to the largest of the 128 and lose what lies about 2^-12 below it (measured: random
// codes 3e-4 of the largest product, normal values 8e-6 of the sum of magnitudes; E2M1 with E2M1
// products are exact to 2e-8), which is far below what the codes themselves keep.
//
// The grouped form takes its rows through the token -> expert permutation, as the INT4 GEMM does:
//   for every block b < ntp / bs of expert e = expert_ids[b], row i: sid = sorted_token_ids[b bs + i]
//   Y[sid] = X[sid / top_k] . W[e]   where sid < N top_k; other rows of Y stay as they are.
//
// Two kernels.  The streaming one serves few rows, where the weights' bytes bound the call: a
// workgroup per 16 MR features and block of rows, whose waves share K.  The tiled one serves many
// rows: both operands go straight to an LDS ring and each wave owns a part of the tile for all of K.
#include <type_traits>

#include "common.h"
#include "mx_format.h"
#include "pega_moe.h"

namespace pega {
namespace {

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8_t;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4_t;

constexpr uint32_t kOutOfRange = 0x80000000u;  // voffset that fails every range check

struct MxArgs {
  const uint8_t* wq;
  const uint8_t* ws;
  const uint8_t* xq;
  const uint8_t* xs;
  uint16_t* y;
  int M, N, K;  // features, rows of X, columns
  // grouped
  const int32_t* sorted_ids;
  const int32_t* expert_ids;
  const int32_t* ntp;
  const float* topk_w;
  int sorted_len, bs, top_k, mul, experts;
};

template <int kXFormat>
__device__ __forceinline__ floatx4_t mx_mfma(u32x4_t w, u32x4_t x0, u32x4_t x1, uint32_t sw,
                                             uint32_t sx, floatx4_t c) {
  i32x8_t a = {}, b = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = static_cast<int>(w[i]);
    b[i] = static_cast<int>(x0[i]);
    if (kXFormat == kMxE4M3) b[4 + i] = static_cast<int>(x1[i]);
  }
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      a, b, c, 4, kXFormat == kMxE4M3 ? 0 : 4, 0, static_cast<int>(sw), 0, static_cast<int>(sx));
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0),
                                           static_cast<int>(bytes), 0x00020000);
}

__device__ __forceinline__ void store4(const MxArgs& p, long long row, int m, floatx4_t v, int sid) {
  float w = 1.0f;
  if (p.mul) w = p.topk_w[sid];
  *reinterpret_cast<uint2*>(p.y + row * p.M + m) =
      make_uint2(pack_bf16x2(v[0] * w, v[1] * w), pack_bf16x2(v[2] * w, v[3] * w));
}

// ---------------------------------------------------------------- few rows
// One workgroup per (16 MR features, 16 RB rows); wave w of WV takes its share of K's steps of
// 128.  A load's lanes read 64 contiguous bytes of a row per quad (fragment order would touch a
// line per lane), and ds_bpermute hands every lane its fragment's 16 bytes.  Four steps' scales of
// 16 rows are one word per lane.  D steps are in flight.
template <int kXFormat, int MR, int RB>
struct MxStep {
  u32x4_t w[MR];
  u32x4_t x[RB][kXFormat == kMxE4M3 ? 2 : 1];
};

template <int kXFormat, int WV, int MR, int RB, int D, bool kGrouped>
__global__ __launch_bounds__(64 * WV) void mx_stream_kernel(MxArgs p) {
  constexpr int kQuads = D / 4;
  constexpr int kHalves = kXFormat == kMxE4M3 ? 2 : 1;
  constexpr int kXStep = 64 * kHalves;  // bytes of a row of X per step
  __shared__ __align__(16) floatx4_t s_red[WV][MR * RB][64];
  __shared__ int s_sid[16 * RB];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.x * (16 * MR);
  const int K = p.K, steps = K >> 7;
  long long expert = 0;
  int n0 = blockIdx.y * (16 * RB);
  if constexpr (kGrouped) {
    const int mb = blockIdx.y;
    const int limit = p.N * p.top_k;
    int sid = limit;
    if (tid < p.bs && mb * p.bs + tid < p.sorted_len) sid = p.sorted_ids[mb * p.bs + tid];
    const int e = __builtin_amdgcn_readfirstlane(p.expert_ids[mb]);
    if (min(p.ntp[0], p.sorted_len) < (mb + 1) * p.bs || e < 0 || e >= p.experts) return;
    expert = e;
    if (tid < 16 * RB) s_sid[tid] = static_cast<unsigned>(sid) < static_cast<unsigned>(limit) ? sid : -1;
    __syncthreads();
    n0 = 0;
  }
  // the row of X (and of Y) of local row i; -1 where there is none
  const auto sid_of = [&](int i) { return kGrouped ? s_sid[i] : (n0 + i < p.N ? n0 + i : -1); };
  const auto x_row = [&](int i) {
    const int sid = sid_of(i);
    return static_cast<long long>(sid < 0 ? 0 : kGrouped ? sid / p.top_k : sid);
  };

  const uint32_t w_bytes = static_cast<uint32_t>(K) / 2u, s_bytes = static_cast<uint32_t>(K) / 32u;
  const long long w_first = expert * p.M + m0;
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(p.wq + w_first * w_bytes, 16u * MR * w_bytes);
  const __amdgpu_buffer_rsrc_t sr = make_rsrc(p.ws + w_first * s_bytes, 16u * MR * s_bytes);
  const uint32_t lr = static_cast<uint32_t>(lane >> 2), lp = static_cast<uint32_t>(lane & 3);
  const uint8_t *xp[RB], *xsp[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    xp[rb] = p.xq + x_row(16 * rb + static_cast<int>(lr)) * (w_bytes * kHalves) + 16u * lp;
    xsp[rb] = p.xs + x_row(16 * rb + c) * s_bytes;
  }
  const int src = (4 * c + g) * 4;
  const auto to_fragment = [&](u32x4_t v) {
    u32x4_t f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      f[e] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(src, static_cast<int>(v[e])));
    return f;
  };

  const int s0 = (steps * wave) / WV, s1 = (steps * (wave + 1)) / WV;
  const auto load_step = [&](MxStep<kXFormat, MR, RB>& r, int s) {
    s = min(s, steps - 1);  // past the share's end: fetched again, never used
#pragma unroll
    for (int mr = 0; mr < MR; ++mr)
      r.w[mr] = __builtin_amdgcn_raw_buffer_load_b128(
          wr, static_cast<int>((16u * mr + lr) * w_bytes + 16u * lp), s * 64, 0);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        r.x[rb][h] = *reinterpret_cast<const u32x4_t*>(xp[rb] + static_cast<long long>(s) * kXStep + 64 * h);
  };
  // scales of steps s .. s + 3: lane (c, j) takes row c's word of step s + j
  struct Scales {
    uint32_t w[MR], x[RB];
  };
  const auto load_scales = [&](Scales& r, int s) {
    const int at = 4 * min(s + g, steps - 1);
#pragma unroll
    for (int mr = 0; mr < MR; ++mr)
      r.w[mr] = __builtin_amdgcn_raw_buffer_load_b32(
          sr, static_cast<int>((16u * mr + c) * s_bytes) + at, 0, 0);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) r.x[rb] = *reinterpret_cast<const uint32_t*>(xsp[rb] + at);
  };
  floatx4_t acc[MR][RB] = {};
  const auto compute = [&](const MxStep<kXFormat, MR, RB>& r, const Scales& sc, int j) {
    const int from = (c + 16 * j) * 4;
    uint32_t sx[RB];
    u32x4_t x[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      sx[rb] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(from, static_cast<int>(sc.x[rb]))) >> (8 * g);
#pragma unroll
      for (int h = 0; h < kHalves; ++h) x[rb][h] = to_fragment(r.x[rb][h]);
      if (kHalves == 1) x[rb][1] = u32x4_t{};
    }
#pragma unroll
    for (int mr = 0; mr < MR; ++mr) {
      const uint32_t sw =
          static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(from, static_cast<int>(sc.w[mr]))) >> (8 * g);
      const u32x4_t w = to_fragment(r.w[mr]);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        acc[mr][rb] = mx_mfma<kXFormat>(w, x[rb][0], x[rb][1], sw, sx[rb], acc[mr][rb]);
    }
  };

  MxStep<kXFormat, MR, RB> slot[D];
  Scales sc[kQuads];
  if (s0 < s1) {
#pragma unroll
    for (int q = 0; q < kQuads; ++q) load_scales(sc[q], s0 + 4 * q);
#pragma unroll
    for (int j = 0; j < D; ++j) {
      load_step(slot[j], min(s0 + j, s1 - 1));
      __builtin_amdgcn_sched_barrier(0);
    }
    int s = s0;
    for (; s + D <= s1; s += D) {
      Scales next[kQuads];
#pragma unroll
      for (int q = 0; q < kQuads; ++q) load_scales(next[q], s + D + 4 * q);
#pragma unroll
      for (int j = 0; j < D; ++j) {
        compute(slot[j], sc[j / 4], j % 4);
        load_step(slot[j], min(s + j + D, s1 - 1));
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int q = 0; q < kQuads; ++q) sc[q] = next[q];
    }
#pragma unroll
    for (int j = 0; j < D - 1; ++j)
      if (s + j < s1) compute(slot[j], sc[j / 4], j % 4);
  }
  // the waves' sums in wave order
#pragma unroll
  for (int mr = 0; mr < MR; ++mr)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) s_red[wave][mr * RB + rb][lane] = acc[mr][rb];
  __syncthreads();
  for (int t = wave; t < MR * RB; t += WV) {
    floatx4_t sum = s_red[0][t][lane];
#pragma unroll
    for (int w = 1; w < WV; ++w) {
      const floatx4_t v = s_red[w][t][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
    const int sid = sid_of(16 * (t % RB) + c);
    if (sid >= 0) store4(p, sid, m0 + 16 * (t / RB) + 4 * g, sum, sid);
  }
}

// ---------------------------------------------------------------- many rows
// A workgroup owns BM features x BN rows, its WM x WN waves TM x TN blocks of 16 x 16 each for all
// of K; a stage of the ring holds 128 k of both operands.  A load brings 1 KB:
// 16 rows of 64 bytes (E2M1) or 8 of 128 (E4M3), the row's 16-byte pieces at slot piece ^ (row / 2
// % 4) or piece ^ (row % 8), which spreads eight lanes' fragment reads over all banks; 64 rows'
// scales of four steps are one load.  One barrier a stage.
template <int kXFormat_, int WM_, int WN_, int TM_, int TN_, int NS_>
struct MxTile {
  static constexpr int kXFormat = kXFormat_, WM = WM_, WN = WN_, TM = TM_, TN = TN_, NS = NS_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int BM = 16 * WM * TM, BN = 16 * WN * TN;
  static constexpr int kXRow = kXFormat == kMxE4M3 ? 128 : 64;  // bytes of a row of X in a stage
  static constexpr int kXLoadRows = 1024 / kXRow;
  static constexpr int kWLoads = BM / 16, kXLoads = BN / kXLoadRows;
  static constexpr int kSLoads = BM / 64 + (BN + 63) / 64;
  static constexpr int PW = (kWLoads + kWaves - 1) / kWaves;  // loads per wave and stage
  static constexpr int PX = (kXLoads + kWaves - 1) / kWaves, P = PW + PX;
  static constexpr int PS = (kSLoads + kWaves - 1) / kWaves;  // scale loads per wave and four
  static constexpr int kX = BM * 64, kStage = kX + BN * kXRow;
  static constexpr int kFour = kSLoads * 1024;                // four steps' scales
  static constexpr int kS = NS * kStage, kLds = kS + 2 * kFour;
  static_assert(BM % 64 == 0 && BN % kXLoadRows == 0 && TN % 2 == 0, "tile shape");
  static_assert(NS >= 3 && NS <= 6 && kLds <= 160 * 1024, "tile shape");
};

// Workgroups go to the eight XCDs in turn; each XCD's are made to cover a compact part of the grid
// of tiles (runs of the order that goes down panels four feature tiles wide), so that its L2 brings
// in as few operand rows as it can.
// gy: of the grid's rows of tiles, those that are there.
__device__ __forceinline__ void xcd_tile(int& tx, int& ty, int gy) {
  const int gx = gridDim.x;
  const int total = gx * gy, id = ty * gx + tx;
  const int xcd = id & 7, each = total >> 3, more = total & 7;
  const int at = xcd * each + min(xcd, more) + (id >> 3);
  const int panel = at / (4 * gy), in = at - panel * 4 * gy;
  const int wide = min(4, gx - 4 * panel);
  ty = in / wide;
  tx = 4 * panel + in - ty * wide;
}

template <int V>
using Int = std::integral_constant<int, V>;

template <typename S, bool kGrouped>
__global__ __launch_bounds__(S::kThreads) void mx_tile_kernel(MxArgs p) {
  constexpr int BM = S::BM, BN = S::BN, NS = S::NS, TM = S::TM, TN = S::TN, P = S::P;
  constexpr bool kF8 = S::kXFormat == kMxE4M3;
  __shared__ __align__(1024) uint8_t smem[S::kLds];
  __shared__ int s_sid[kGrouped ? BN : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % S::WM, wn = wave / S::WM;
  const int c = lane & 15, g = lane >> 4;
  int tx = blockIdx.x, ty = blockIdx.y;
  int live = gridDim.y;  // blocks with rows
  if constexpr (kGrouped) {
    live = min(p.ntp[0], p.sorted_len) / p.bs;
    if (ty >= live) return;
  }
  // grouped tiles of few rows share little, and lose 2% by the mapping; wide ones gain (256 x 128, 4096
  // x 7168 over 48 experts of 341 rows: 879 and 542 us)
  if constexpr (!kGrouped || BN >= 128) xcd_tile(tx, ty, live);
  const int m0 = tx * BM;
  int n0 = ty * BN;
  const int K = p.K, steps = K >> 7;
  long long expert = 0;
  if constexpr (kGrouped) {
    // up to BN / bs blocks of one expert (an expert's blocks follow each other): this one, if the
    // number of the expert's blocks before it is a multiple of that, and those after it
    const int mb = ty, take = max(BN / p.bs, 1);
    const int limit = p.N * p.top_k;
    const int e = __builtin_amdgcn_readfirstlane(p.expert_ids[mb]);
    if (e < 0 || e >= p.experts) return;
    int before = 0, blocks = 1;
    if (take > 1) {
      for (int at = mb; at > 0;) {
        const uint64_t other = ~__ballot(lane < at && p.expert_ids[max(at - 1 - lane, 0)] == e);
        const int same = other == 0 ? 64 : __builtin_ctzll(other);
        before += same;
        at -= 64;
        if (same < 64) break;
      }
      if (before % take != 0) return;
      const uint64_t other = ~__ballot(mb + lane < live && p.expert_ids[min(mb + lane, live - 1)] == e);
      blocks = min(take, other == 0 ? 64 : __builtin_ctzll(other));
    }
    expert = e;
    for (int i = tid; i < BN; i += S::kThreads) {
      int sid = limit;
      if (i < blocks * p.bs && mb * p.bs + i < p.sorted_len) sid = p.sorted_ids[mb * p.bs + i];
      s_sid[i] = static_cast<unsigned>(sid) < static_cast<unsigned>(limit) ? sid : -1;
    }
    __syncthreads();
    n0 = 0;
  }
  const uint32_t w_bytes = static_cast<uint32_t>(K) / 2u, s_bytes = static_cast<uint32_t>(K) / 32u;
  const uint32_t x_bytes = w_bytes * (S::kXRow / 64);
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) uint8_t*)smem));
  const long long w_first = expert * p.M + m0;
  const int w_rows = min(BM, p.M - m0), x_rows = kGrouped ? p.N : min(BN, p.N - n0);

  // The offset of a row of the tile in its operand: rows past the last feature or row of X are past
  // the operand's range, and so are grouped rows without a route; they bring zeros.
  const auto row_off = [&](bool x, int r, uint32_t row_bytes) {
    if (!kGrouped || !x) return static_cast<uint32_t>(r) * row_bytes;
    const int sid = s_sid[min(r, BN - 1)];
    return sid < 0 ? kOutOfRange : static_cast<uint32_t>(sid / p.top_k) * row_bytes;
  };
  // This wave's loads of a stage (a repeat brings the same): PW of W, then PX of X.
  u32x4_t w_rsrc = rsrc_words(p.wq + w_first * w_bytes, static_cast<uint32_t>(w_rows) * w_bytes);
  u32x4_t x_rsrc = rsrc_words(p.xq + static_cast<long long>(n0) * x_bytes, static_cast<uint32_t>(x_rows) * x_bytes);
  const uint32_t w_size = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(w_rsrc[2])));
  const uint32_t x_size = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x_rsrc[2])));
  uint32_t dst[P], voff[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const bool x = j >= S::PW;
    const int i = x ? min(wave * S::PX + j - S::PW, S::kXLoads - 1) : min(wave * S::PW + j, S::kWLoads - 1);
    const int rows_per = x ? S::kXLoadRows : 16, pieces = 64 / rows_per;
    const int r = i * rows_per + lane / pieces;
    const int swz = pieces == 8 ? r & 7 : (r >> 1) & 3;
    dst[j] = lds0 + (x ? S::kX : 0) + 1024u * static_cast<uint32_t>(i);
    voff[j] = row_off(x, r, x ? x_bytes : w_bytes) + 16u * static_cast<uint32_t>((lane % pieces) ^ swz);
  }
  u32x4_t s_rsrc[S::PS];
  uint32_t s_dst[S::PS], s_voff[S::PS];
#pragma unroll
  for (int j = 0; j < S::PS; ++j) {
    const int i = min(wave * S::PS + j, S::kSLoads - 1);
    const bool x = i >= BM / 64;
    const long long first = x ? n0 : w_first;
    s_rsrc[j] = rsrc_words((x ? p.xs : p.ws) + first * s_bytes,
                           static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(
                               static_cast<int>((x ? x_rows : w_rows) * s_bytes))));
    s_dst[j] = lds0 + S::kS + 1024u * static_cast<uint32_t>(i);
    const int r = 64 * (x ? i - BM / 64 : i) + lane;
    s_voff[j] = x && r >= BN ? kOutOfRange : row_off(x, r, s_bytes);
  }
  // Stages come in turn; past the last one the operands have no bytes, and the loads bring zeros that
  // nothing reads: a branch there would cut the step in two, and the compiler moves products across it.
  uint32_t w_at = 0, x_at = 0;
  int to_come = steps;
  const auto stage_in = [&](uint32_t st) {
    w_rsrc[2] = to_come > 0 ? w_size : 0u;
    x_rsrc[2] = to_come > 0 ? x_size : 0u;
#pragma unroll
    for (int j = 0; j < P; ++j)
      dma_b128(j < S::PW ? w_rsrc : x_rsrc, dst[j] + st, voff[j], j < S::PW ? w_at : x_at);
    w_at += 64;
    x_at += S::kXRow;
    --to_come;
  };
  // Scales come for four steps at a time, 16 bytes a row (a word a step would touch as many lines
  // four times as often: 4096 x 4096 x 7168 in MXFP4 84 us instead of 68 without scale loads); the
  // last four are steps - 4 .. steps - 1, wherever that starts.
  const auto four_first = [&](int four) { return min(4 * four, steps - 4); };
  const auto scales_in = [&](int four) {
#pragma unroll
    for (int j = 0; j < S::PS; ++j)
      dma_b128(s_rsrc[j], s_dst[j] + static_cast<uint32_t>((four & 1) * S::kFour), s_voff[j],
               4u * static_cast<uint32_t>(four_first(four)));
  };
  struct WFrags {
    u32x4_t w[TM];
    uint32_t s[TM];
  };
  struct XFrag {
    u32x4_t x[kF8 ? 2 : 1];
    uint32_t s;
  };
  const uint8_t* w_rd = smem + (wm * TM * 16 + c) * 64 + 16 * (g ^ ((c >> 1) & 3));
  const uint8_t* x_rd = smem + S::kX + (wn * TN * 16 + c) * S::kXRow;
  const int x_at0 = 16 * (kF8 ? g ^ (c & 7) : g ^ ((c >> 1) & 3));
  const int x_at1 = 16 * ((4 + g) ^ (c & 7));
  const uint8_t* sw_rd = smem + S::kS + (wm * TM * 16 + c) * 16 + g;
  const uint8_t* sx_rd = smem + S::kS + (BM + wn * TN * 16 + c) * 16 + g;
  // where the scale bytes of a four's first step are
  const auto scales_at = [&](int four) {
    return (four & 1) * S::kFour + 4 * min(4 * four - four_first(four), 3);
  };
  const auto read_w = [&](WFrags& f, int t, int st, int sc) {
    f.w[t] = *reinterpret_cast<const u32x4_t*>(w_rd + st + 1024 * t);
    f.s[t] = sw_rd[sc + 256 * t];
  };
  const auto read_x = [&](XFrag& f, int j, int st, int sc) {
    f.x[0] = *reinterpret_cast<const u32x4_t*>(x_rd + st + 16 * S::kXRow * j + x_at0);
    if constexpr (kF8)
      f.x[1] = *reinterpret_cast<const u32x4_t*>(x_rd + st + 16 * S::kXRow * j + x_at1);
    f.s = sx_rd[sc + 256 * j];
  };
  floatx4_t acc[TM][TN] = {};

  scales_in(0);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) stage_in(i * S::kStage);
  vm_wait<(NS - 2) * P>();
  lds_barrier();
  int st_now = 0, st_in_now = (NS - 1) * S::kStage;
  const auto next = [](int at) { return at + S::kStage == NS * S::kStage ? 0 : at + S::kStage; };
  // Step s multiplies the rows' fragments one after another, each read while the one before it is
  // multiplied.  Half way the next stage has landed (each wave waits for its own loads, the barrier
  // for all) and every wave is past stage s - 1, which the loads of stage s + NS - 1 then fill; in
  // the second half the next stage's weight fragments and first row fragment are read.
  constexpr int kMid = TN / 2, kPer = (TM + TN - kMid - 1) / (TN - kMid);
  WFrags wa, wb;
  XFrag x[2];
#pragma unroll
  for (int t = 0; t < TM; ++t) read_w(wa, t, 0, 0);
  read_x(x[0], 0, 0, 0);
  // Steps go four at a time, whose scales lie one after another from sc on (the next four's from
  // sc_four on); with a ring of four stages every place in it is then a constant.
  const auto step = [&](auto of_four, const WFrags& w, WFrags& w_next, int four, int sc, int sc_four) {
    constexpr int Q = decltype(of_four)::value;
    const int st = NS == 4 ? Q * S::kStage : st_now, st_next = NS == 4 ? (Q + 1) % 4 * S::kStage : next(st_now);
    const int st_in = NS == 4 ? (Q + 3) % 4 * S::kStage : st_in_now;
    const int sc_now = sc + 4 * Q, sc_next = Q == 3 ? sc_four : sc + 4 * Q + 4;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      if (j == kMid) {
        // loads since the next stage's: NS - 3 stages, and scales where a four's first step is among
        // theirs (all of them have landed two steps on, before anything reads them)
        vm_wait<(NS - 3) * P + (Q >= 1 && Q <= 2 && Q <= NS - 3 ? S::PS : 0)>();
        lds_barrier();
        // the four steps after these, in whose place every wave has read to the end; after the last
        // the same again
        if constexpr (Q == 0) scales_in(four + 1);
        stage_in(static_cast<uint32_t>(st_in));
      }
      if (j + 1 < TN) read_x(x[(j + 1) & 1], j + 1, st, sc_now);
      else read_x(x[0], 0, st_next, sc_next);
      if (j >= kMid) {
#pragma unroll
        for (int t = (j - kMid) * kPer; t < (j - kMid + 1) * kPer && t < TM; ++t)
          read_w(w_next, t, st_next, sc_next);
      }
#pragma unroll
      for (int t = 0; t < TM; ++t)
        acc[t][j] = mx_mfma<S::kXFormat>(w.w[t], x[j & 1].x[0], x[j & 1].x[kF8 ? 1 : 0], w.s[t],
                                         x[j & 1].s, acc[t][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    st_now = next(st_now);
    st_in_now = next(st_in_now);
  };
  int four = 0, sc = 0;
  for (; four < steps >> 2; ++four) {
    const int sc_four = scales_at(four + 1);
    step(Int<0>{}, wa, wb, four, sc, sc_four);
    step(Int<1>{}, wb, wa, four, sc, sc_four);
    step(Int<2>{}, wa, wb, four, sc, sc_four);
    step(Int<3>{}, wb, wa, four, sc, sc_four);
    sc = sc_four;
  }
  const int left = steps & 3;
  if (left > 0) step(Int<0>{}, wa, wb, four, sc, 0);
  if (left > 1) step(Int<1>{}, wb, wa, four, sc, 0);
  if (left > 2) step(Int<2>{}, wa, wb, four, sc, 0);
  vm_wait<0>();  // nothing lands in LDS that is another workgroup's by then

#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int i = (wn * TN + j) * 16 + c;
    const int sid = kGrouped ? s_sid[i] : (n0 + i < p.N ? n0 + i : -1);
    if (sid < 0) continue;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      const int m = m0 + (wm * TM + t) * 16 + 4 * g;
      if (m < p.M) store4(p, sid, m, acc[t][j], sid);
    }
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int kMaxGridY = 65535;

int mx_gemm_checks(const char* name, const MxArgs& a, int x_format) {
  // no rows: nothing to do, and empty tensors have no address
  if (a.N != 0 && (!a.wq || !a.ws || !a.xq || !a.xs || !a.y)) return fail(kInvalidValue, "%s: null pointer", name);
  if (a.M <= 0 || a.N < 0 || a.K <= 0)
    return fail(kInvalidValue, "%s: bad shape M=%d N=%d K=%d", name, a.M, a.N, a.K);
  if (x_format != kMxE4M3 && x_format != kMxE2M1)
    return fail(kInvalidValue, "%s: format %d (0 E4M3, 1 E2M1)", name, x_format);
  if (a.M % 16 != 0 || a.K % 128 != 0)
    return fail(kNotSupported, "%s: M %% 16 and K %% 128 must be 0 (M=%d K=%d)", name, a.M, a.K);
  if (!aligned(a.wq, 16) || !aligned(a.xq, 16) || !aligned(a.y, 16) || !aligned(a.ws, 4) ||
      !aligned(a.xs, 4))
    return fail(kNotSupported, "%s: codes and output must be 16-byte aligned, scales 4-byte", name);
  // a launch has fewer than 2^32 threads a dimension, the streaming kernel 256 for 16 features
  if (a.M >= (1 << 28)) return fail(kNotSupported, "%s: M=%d is not below 2^28", name, a.M);
  // a workgroup addresses up to 256 rows of either operand through one 32-bit range
  if (256LL * a.K >= static_cast<long long>(kOutOfRange))
    return fail(kNotSupported, "%s: K=%d is over 2^23", name, a.K);
  return kSuccess;
}

// The last check, once the sizes are known to be sound.
int mx_gemm_apart(const char* name, const MxArgs& a, int x_format) {
  const long long w = static_cast<long long>(a.M) * a.K * a.experts, x = static_cast<long long>(a.N) * a.K;
  const long long y = 2LL * a.M * a.N * a.top_k;
  if (overlap(a.y, y, a.wq, w / 2) || overlap(a.y, y, a.ws, w / kMxBlock) ||
      overlap(a.y, y, a.xq, mx_code_bytes(x_format, x)) || overlap(a.y, y, a.xs, x / kMxBlock))
    return fail(kInvalidValue, "%s: the output overlaps an operand", name);
  return kSuccess;
}

template <int kXFormat, int MR, int RB, bool kGrouped, int D = 4>
void launch_stream(const MxArgs& a, int row_blocks, hipStream_t stream) {
  constexpr int WV = 4;  // eight waves take 2 to 10% longer
  hipLaunchKernelGGL((mx_stream_kernel<kXFormat, WV, MR, RB, D, kGrouped>),
                     dim3(a.M / (16 * MR), row_blocks), dim3(64 * WV), 0, stream, a);
}

template <typename S, bool kGrouped>
void launch_tile(const MxArgs& a, int row_blocks, hipStream_t stream) {
  hipLaunchKernelGGL((mx_tile_kernel<S, kGrouped>), dim3(ceil_div(a.M, S::BM), row_blocks),
                     dim3(S::kThreads), 0, stream, a);
}

// The tiled kernel's scales come four steps at a time.
constexpr int kTileMinK = 512;

// The tile shapes, smallest first, with what a step of 128 k costs a CU that has one tile, and each
// of several, and what a tile costs besides its steps (its start, and its results, which the large
// ones write while nothing else runs on their CU), in ns.  Measured with MXFP8 rows and operands that come
// from HBM, 64 x 64 to 256 x 256: 256 rows x 4096 x 7168 20 / 27 / 37 / 53 / 90 us, 1024 rows 57 / 47 / 40 / 53 /
// 89, 4096 rows 200 / 166 / 151 / 111 / 96 (15, 34 and 86 us by the chosen shapes where the last-level cache
// has the operands); MXFP4 rows 17 / 25 / 29 / 43 / 59, 46 / 39 / 32 / 44 / 59, 157 / 134 / 99 / 91 / 69.  Over 53 sizes
// each, drawn from 65 to 4096 rows, 512 to 10240 features and k 1024 to 9216, the chosen shape is within
// 0.6% (MXFP8) and 2.9% (MXFP4) of the best one, rms, and 4% and 15% at most.  Four stages make every place
// in the ring a constant; 64 x 64 tiles, whose steps are shortest, gain more from a fifth (256 rows x 4096 x
// 7168 22.2 and 18.8 us), and 256 x 256 of MXFP8 have room for three.
template <int F> using Tile64 = MxTile<F, 2, 2, 2, 2, 5>;
template <int F> using Tile128x64 = MxTile<F, 2, 2, 4, 2, 4>;
template <int F> using Tile128 = MxTile<F, 2, 2, 4, 4, 4>;
template <int F> using Tile256x128 = MxTile<F, 4, 2, 4, 4, 4>;
template <int F> using Tile256 = MxTile<F, 4, 2, 4, 8, F == kMxE4M3 ? 3 : 4>;
struct TileCost {
  int m, n, alone, each, besides;
};
constexpr TileCost kTileCosts[] = {{64, 64, 270, 215, 900},
                                   {128, 64, 385, 335, 1900},
                                   {128, 128, 570, 600, 3000},
                                   {256, 128, 840, 950, 6000},
                                   {256, 256, 1400, 1450, 9500}};

int best_tile(int M, int N, int K, int cu) {
  int best = 0;
  long long least = 0;
  for (int i = 0; i < 5; ++i) {
    const TileCost& c = kTileCosts[i];
    const long long each = (static_cast<long long>(ceil_div(M, c.m)) * ceil_div(N, c.n) + cu - 1) / cu;
    const long long t = each == 1 ? static_cast<long long>(K / 128) * c.alone + c.besides
                                  : each * (static_cast<long long>(K / 128) * c.each + c.besides);
    if (i == 0 || t < least) best = i, least = t;
  }
  return best;
}

template <int kXFormat>
int dense_launch(const MxArgs& a, hipStream_t stream, const char* name) {
  const int cu = current_cu_count();
  if (cu <= 0) return fail(kInvalidValue, "%s: no device", name);
  const long long tiles64 = static_cast<long long>(ceil_div(a.M, 64)) * ceil_div(a.N, 64);
  // The streaming kernel while 64 x 64 tiles would leave many CUs idle, since its waves share K: a
  // quarter of the CUs to 8 rows (one row x 9728 x 2560, 152 tiles: 6.5 against 7.0 us, x 14336 x 4096, 224
  // tiles: 11.9 and 10.3), half where K is long or a workgroup has all rows (64 rows x 4096 x 7168, 64
  // tiles: 10.6 against 18.4 us; 128 rows, 128 tiles: 15.1 and 18.5; 32 rows x 7168 x 2048, 112 tiles: 5.7
  // and 6.9; 16 rows x 9728 x 2560 8.9 and 7.3), else three quarters (96 rows x 2816 x 2048, 88 tiles: 7.1
  // and 6.1).
  const int most = a.N <= 8 ? 3 * cu / 4 : a.K > 4096 || a.N <= 32 ? cu / 2 : cu / 4;
  if (a.K < kTileMinK || tiles64 <= most) {
    // To 16 rows as many workgroups as there are (9728 x 2560, 16 rows: 608 of 16 features 7.8 us,
    // 304 of 32 8.1), but 32 features each where that is one for most CUs (8192 x 4096, 256: 8.7 and 6.7 us);
    // beyond, more features a workgroup, which read X less often, as long as three quarters of the CUs
    // have one (64 rows x 4096 x 7168 with 1 / 2 / 4 sets of 16: 14.2 / 10.6 / 14.3 us; 32 rows x 7168 x
    // 2048 7.9 / 5.7 / 7.9).  Four steps in flight; eight only for few MXFP8 rows of long K (one row x
    // 2560 x 9728 7.1 and 6.6 us; eight cost x 8192 x 4096 6.4 and 7.3, 64 rows x 4096 x 7168 10.4 and 11.6).
    const int blocks = ceil_div(a.N, 32);
    const auto enough = [&](int mr) {
      return a.M % (16 * mr) == 0 && 4LL * (a.M / (16 * mr)) * blocks >= 3LL * cu;
    };
    const int wide = a.M / 32;  // workgroups of 32 features
    if (a.N <= 16 && a.M % 32 == 0 && wide <= cu && 4 * wide >= 3 * cu)
      launch_stream<kXFormat, 2, 1, false>(a, 1, stream);
    else if (a.N <= 8 && kXFormat == kMxE4M3 && a.K > 4096) launch_stream<kXFormat, 1, 1, false, 8>(a, 1, stream);
    else if (a.N <= 16) launch_stream<kXFormat, 1, 1, false>(a, 1, stream);
    else if (enough(4)) launch_stream<kXFormat, 4, 2, false>(a, blocks, stream);
    else if (enough(2)) launch_stream<kXFormat, 2, 2, false>(a, blocks, stream);
    else launch_stream<kXFormat, 1, 2, false>(a, blocks, stream);
    return launch_status(name);
  }
  const auto go = [&](auto shape) {
    using S = decltype(shape);
    launch_tile<S, false>(a, ceil_div(a.N, S::BN), stream);
  };
  switch (best_tile(a.M, a.N, a.K, cu)) {
    case 0: go(Tile64<kXFormat>{}); break;
    case 1: go(Tile128x64<kXFormat>{}); break;
    case 2: go(Tile128<kXFormat>{}); break;
    case 3: go(Tile256x128<kXFormat>{}); break;
    default: go(Tile256<kXFormat>{}); break;
  }
  return launch_status(name);
}

template <int kXFormat>
int grouped_launch(const MxArgs& a, int ep_size, hipStream_t stream, const char* name) {
  const int cu = current_cu_count();
  if (cu <= 0) return fail(kInvalidValue, "%s: no device", name);
  const int blocks = ceil_div(a.sorted_len, a.bs);
  // Workgroups of 128 features that will have rows: the blocks that the local routes (one in ep_size)
  // fill, at least one for each expert that routes spread evenly would reach.
  const double local = static_cast<double>(a.N) * a.top_k / ep_size;
  const double reached = a.experts * (1.0 - __builtin_exp(local * __builtin_log1p(-1.0 / (a.experts + 1e-9))));
  const double live = reached > local / a.bs ? reached : local / a.bs;
  const double units = live * ceil_div(a.M, 128);
  // Tiles as wide as the experts' rows: 256 x 128 (and then a mapping that keeps an expert's tiles
  // on one XCD) from 72 rows an expert on, 128 x 64 from 32, or where a block is over 32.  MXFP8 in
  // 128 x 64 / 256 x 128, in us, at 48, 64, 80, 192 rows an expert on average: 4096 x 7168 over 48 experts
  // 197 / 219, 224 / 233, 262 / 203, 437 / 360; 7168 x 2048 over 48 104 / 122, 119 / 130, 142 / 135, 232 / 226;
  // 2816 x 2048 over 64 57 / 66, 69 / 81, 86 / 87, 148 / 140; 2048 x 1408 over 64 33 / 37, 43 / 51, 52 / 42, 86 /
  // 82 (16 experts of 4096 x 4096, few tiles a CU, go either way: 54 / 42 at 64, 54 / 71 at 80).  MXFP4 rows
  // rank alike.  In 128 x 32 / 128 x 64 with blocks of 32: 2816 x 2048 at 24 and 48 rows 50 / 53, 71 / 67,
  // 4096 x 7168 177 / 169, 229 / 179.
  const double rows = local / a.experts;
  if (a.K >= kTileMinK && rows >= 72.0) {
    launch_tile<Tile256x128<kXFormat>, true>(a, blocks, stream);
    return launch_status(name);
  }
  if (a.bs > 32 || (a.K >= kTileMinK && rows >= 32.0)) {
    if (a.K < kTileMinK) launch_stream<kXFormat, 1, 4, true>(a, blocks, stream);
    else launch_tile<Tile128x64<kXFormat>, true>(a, blocks, stream);
    return launch_status(name);
  }
  // Short blocks: tiles of 128 x 32, or, where too few of them have rows, the streaming kernel, whose
  // waves share K.  Rows of 2 KB of weights or multiples of it meet in few memory channels when
  // streamed; other long ones stream as well until there are several tiles a CU.  Streaming / tiled, MXFP8,
  // in us, 2816 features with 6, 20, 35, 61 experts reached (127, 443, 747, 1340 units): k 2560 8.3 / 7.4,
  // 17 / 15, 31 / 26, 66 / 53; k 4096 11.6 / 10.6, 33 / 27, 60 / 50, 101 / 77; k 5120 12.9 / 12.6, 34 / 34, 64 / 56,
  // 115 / 104; k 6144 15.3 / 14.2, 43 / 41, 71 / 64, 127 / 120; k 7168 15.9 / 15.1, 49 / 47, 73 / 71, 134 / 133; k 8192
  // 18.1 / 16.8, 56 / 56, 98 / 102, 172 / 160.  With 10 or 12 experts (a tile and a bit a CU) k 6144 to 8192
  // stream 20 to 35% faster, with 2 (63 units) any k does, 4.3 / 6.7 to 12 / 16.  MXFP4 rows, streamed with
  // eight steps in flight, gain 5 to 20% on the tiles from k 6144 on below 1340 units, and at k 8192 lose
  // it by the rule (747 units 91 / 105).
  const double enough = a.K <= 2560 ? 0.25 * cu : a.K < 6144 || a.K % 4096 == 0 ? 0.5 * cu : 5.0 * cu;
  const bool tiled = a.K >= kTileMinK && units >= enough;
  if (tiled) launch_tile<MxTile<kXFormat, 4, 1, 2, 2, 6>, true>(a, blocks, stream);
  else if (a.bs > 16) launch_stream<kXFormat, 1, 2, true>(a, blocks, stream);
  // Eight steps in flight where the workgroups follow each other, four where each CU has few (4096 x
  // 7168 over 48 experts, MXFP8, at 4, 8, 32, 64 tokens: 12 / 13.5, 16.7 / 18.5, 77 / 69, 131 / 116 us).
  else if (kXFormat == kMxE4M3 && a.M % 32 == 0) {
    if (units <= cu) launch_stream<kXFormat, 2, 1, true>(a, blocks, stream);
    else launch_stream<kXFormat, 2, 1, true, 8>(a, blocks, stream);
  } else if (units <= cu) launch_stream<kXFormat, 1, 1, true>(a, blocks, stream);
  else launch_stream<kXFormat, 1, 1, true, 8>(a, blocks, stream);
  return launch_status(name);
}

}  // namespace
}  // namespace pega

using namespace pega;

// No reference counterpart: Y = X . W^T of microscaled operands.
PEGA_API int pega_mx_gemm(const uint8_t* w_codes, const uint8_t* w_scales, const uint8_t* x_codes,
                          const uint8_t* x_scales, int x_format, uint16_t* Y, int M, int N, int K,
                          hipStream_t stream) {
  MxArgs a{w_codes, w_scales, x_codes, x_scales, Y, M, N, K, nullptr, nullptr, nullptr, nullptr, 0, 0, 1, 0, 1};
  const int rc = mx_gemm_checks("mx_gemm", a, x_format);
  if (rc != kSuccess) return rc;
  if (N > 32 * kMaxGridY) return fail(kNotSupported, "mx_gemm: too many rows (N=%d)", N);
  if (N == 0) return kSuccess;
  const int apart = mx_gemm_apart("mx_gemm", a, x_format);
  if (apart != kSuccess) return apart;
  return x_format == kMxE4M3 ? dense_launch<kMxE4M3>(a, stream, "mx_gemm")
                             : dense_launch<kMxE2M1>(a, stream, "mx_gemm");
}

// No reference counterpart: the grouped GEMM of pega_wna16_gemm on microscaled operands.
PEGA_API int pega_mx_grouped_gemm(const uint8_t* x_codes, const uint8_t* x_scales, int x_format,
                                  uint16_t* output, const uint8_t* w_codes, const uint8_t* w_scales,
                                  const int32_t* sorted_token_ids, const int32_t* expert_ids,
                                  const int32_t* num_tokens_post_padded, const float* topk_weights,
                                  int sorted_token_ids_len, int moe_block_size, int top_k,
                                  bool mul_topk_weights, int size_m, int size_n, int size_k,
                                  int local_experts, int ep_size, hipStream_t stream) {
  MxArgs a{w_codes, w_scales, x_codes, x_scales, output, size_n, size_m, size_k, sorted_token_ids,
           expert_ids, num_tokens_post_padded, topk_weights, sorted_token_ids_len, moe_block_size,
           top_k, mul_topk_weights ? 1 : 0, local_experts};
  const int rc = mx_gemm_checks("mx_grouped_gemm", a, x_format);
  if (rc != kSuccess) return rc;
  if (!sorted_token_ids || !expert_ids || !num_tokens_post_padded || (mul_topk_weights && !topk_weights))
    return fail(kInvalidValue, "mx_grouped_gemm: null pointer");
  if (!(moe_block_size == 8 || (moe_block_size >= 16 && moe_block_size <= 64 && moe_block_size % 16 == 0)))
    return fail(kInvalidValue, "mx_grouped_gemm: block size %d not in {8,16,32,48,64}", moe_block_size);
  if (top_k <= 0 || local_experts <= 0 || ep_size <= 0 || sorted_token_ids_len < 0 ||
      static_cast<long long>(size_m) * top_k >= (1LL << 31))
    return fail(kInvalidValue, "mx_grouped_gemm: bad shape top_k=%d experts=%d sorted=%d", top_k,
                local_experts, sorted_token_ids_len);
  if (sorted_token_ids_len > static_cast<long long>(kMaxGridY) * moe_block_size)
    return fail(kNotSupported, "mx_grouped_gemm: too many blocks (%d ids in blocks of %d)",
                sorted_token_ids_len, moe_block_size);
  // the gathered rows are addressed through one 32-bit range
  if (static_cast<long long>(size_m) * size_k >= static_cast<long long>(kOutOfRange))
    return fail(kNotSupported, "mx_grouped_gemm: activations over 2 GiB (%d x %d)", size_m, size_k);
  if (size_m == 0 || sorted_token_ids_len == 0) return kSuccess;
  const int apart = mx_gemm_apart("mx_grouped_gemm", a, x_format);
  if (apart != kSuccess) return apart;
  return x_format == kMxE4M3 ? grouped_launch<kMxE4M3>(a, ep_size, stream, "mx_grouped_gemm")
                             : grouped_launch<kMxE2M1>(a, ep_size, stream, "mx_grouped_gemm");
}

// Residual add + root-mean-square norm on MI355X (gfx950):
//
//   s = residual + x            residual_out = bf16(s)
//   y = s * weight / sqrt(mean(s^2) + eps)
//   normed = bf16(y)            codes, scales = MXFP8(y)   (either or both)
//
// One pass: a row's values stay in registers between the sum of squares and the outputs, so a
// row is read once and each output written once; the bytes bound it.
//
// The sums and the products are in 64 bits: a value's E4M3 code and its block's scale follow the
// formula however near y lies to a rounding border (in 32 bits about one value in 10^6 goes to the
// neighbouring code, and which ones depends on the order of the sum).  y reaches 32 bits rounded to
// odd (the last bit set if anything was cut off), after which one more rounding, to bf16 or to a
// code, is the rounding of y itself, among fp32's smallest numbers too.  Past fp32's range y is an
// infinity.  The norm is of s itself, not of bf16(s), so normed is not quite the norm of
// residual_out.  The 64-bit work hides behind the memory: 4096 rows of 7168 with every output take
// 56 us (265 MB, 4.7 TB/s; a copy of 1 GiB reaches 5.1), one row 4.9 us, of which the launch itself is
// 2.3.
#include "common.h"
#include "mx_format.h"
#include "pega_moe.h"

namespace pega {
namespace {

// y in fp32, rounded to odd: the low 29 mantissa bits cut off, and the last one kept set if any
// of them was (adding 2^29 - 1 to them carries into it then).  What is left converts exactly in
// fp32's normal range.
__device__ __forceinline__ float to_odd(double y) {
  const uint64_t b = __builtin_bit_cast(uint64_t, y);
  const uint32_t lo = static_cast<uint32_t>(b);
  const uint32_t odd = (lo & 0x1fffffffu) + 0x1fffffffu;
  const uint64_t cut = (b & 0xffffffff00000000ull) | ((lo | odd) & 0xe0000000u);
  return static_cast<float>(__builtin_bit_cast(double, cut));
}

// The same below that range (2^-126), where fp32 holds the multiples of 2^-149: bf16's smallest
// numbers (from 2^-133 on) and MXFP8's of the lowest scale (2^-136) would be rounded twice otherwise.
__device__ __forceinline__ float to_odd_small(double y) {
  const double steps = __builtin_fabs(y) * 0x1p149;  // exact, below 2^23
  const uint32_t whole = static_cast<uint32_t>(steps);
  const uint32_t odd = whole | (static_cast<double>(whole) != steps ? 1u : 0u);
  return __builtin_copysignf(__builtin_bit_cast(float, odd), static_cast<float>(y));
}
// (what rounds to 0 there is 0 in every output)
__device__ __forceinline__ bool is_subnormal(float v) { return __builtin_amdgcn_classf(v, 0x90); }

template <int kCtrl>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint64_t o = static_cast<uint64_t>(mx_dpp<kCtrl>(static_cast<uint32_t>(b >> 32))) << 32 |
                     mx_dpp<kCtrl>(static_cast<uint32_t>(b));
  return v + __builtin_bit_cast(double, o);
}

// The sum of 16 consecutive lanes, in each of them.
__device__ __forceinline__ double sum16(double v) {
  v = dpp_add<0xB1>(v);     // quad_perm [1,0,3,2]
  v = dpp_add<0x4E>(v);     // quad_perm [2,3,0,1]
  v = dpp_add<0x141>(v);    // row_half_mirror
  return dpp_add<0x140>(v); // row_mirror
}

__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(b)), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(b >> 32)), lane);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// A row is taken by blockDim.x threads, a whole number of waves, CH vectors of 8 columns a lane;
// a workgroup takes blockDim.y rows.  Every load of a row has returned before its first store
// (the sum needs them all), so an output may be the buffer of an input.
constexpr int kMaxWaves = 16;

template <int CH, bool kX32>
__global__ __launch_bounds__(CH == 1 ? 256 : CH == 2 ? 512 : 64 * kMaxWaves) void add_rmsnorm_kernel(
    const void* x, const uint16_t* residual, const uint16_t* __restrict__ weight, double eps,
    uint16_t* residual_out, uint16_t* normed, uint8_t* codes, uint8_t* scales, int rows,
    int hidden) {
  __shared__ double s_sum[kMaxWaves];
  const int lanes = blockDim.x, lane = threadIdx.x;
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int vecs = hidden >> 3;
  const bool in = row < rows;
  const long long base = static_cast<long long>(row) * hidden;

  uint4 xr[CH][kX32 ? 2 : 1], rr[CH], wr[CH];
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int v = lane + c * lanes;
    const bool ok = in && v < vecs;
    const long long at = base + 8LL * v;
    if constexpr (kX32) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(x) + at);
      xr[c][0] = ok ? p[0] : zero;
      xr[c][1] = ok ? p[1] : zero;
    } else {
      xr[c][0] = ok ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at) : zero;
    }
    // no residual: -0, which leaves every x as it is
    rr[c] = make_uint4(0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u);
    if (ok && residual) rr[c] = *reinterpret_cast<const uint4*>(residual + at);
    wr[c] = v < vecs ? *reinterpret_cast<const uint4*>(weight + 8 * v) : zero;
  }
  double s[CH][8], sum = 0.0;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t rw[4] = {rr[c].x, rr[c].y, rr[c].z, rr[c].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float xv;
      if constexpr (kX32) {
        const uint4 q = xr[c][i >> 2];
        const uint32_t w = (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
        xv = __builtin_bit_cast(float, w);
      } else {
        const uint4 q = xr[c][0];
        const uint32_t w = (i >> 1) == 0 ? q.x : (i >> 1) == 1 ? q.y : (i >> 1) == 2 ? q.z : q.w;
        xv = (i & 1) ? bf_hi(w) : bf_lo(w);
      }
      const float rv = (i & 1) ? bf_hi(rw[i >> 1]) : bf_lo(rw[i >> 1]);
      s[c][i] = static_cast<double>(xv) + static_cast<double>(rv);
      sum = __builtin_fma(s[c][i], s[c][i], sum);
    }
  }
  sum = sum16(sum);
  sum = (lane_f64(sum, 0) + lane_f64(sum, 16)) + (lane_f64(sum, 32) + lane_f64(sum, 48));
  if (lanes > 64) {
    if ((lane & 63) == 0) s_sum[lane >> 6] = sum;
    __syncthreads();
    const int w = lane & 15;
    sum = sum16(w < lanes >> 6 ? s_sum[w] : 0.0);
  }
  const double inv = 1.0 / __builtin_sqrt(sum / hidden + eps);

  const bool whole = (hidden & 127) == 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int v = lane + c * lanes;
    const bool ok = in && v < vecs;
    const long long at = base + 8LL * v;
    const uint32_t ww[4] = {wr[c].x, wr[c].y, wr[c].z, wr[c].w};
    if (residual_out && ok) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(to_odd(s[c][2 * i]), to_odd(s[c][2 * i + 1]));
      *reinterpret_cast<uint4*>(residual_out + at) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const double p0 = s[c][i] * inv * static_cast<double>(bf_lo(ww[i >> 1]));
      const double p1 = s[c][i + 1] * inv * static_cast<double>(bf_hi(ww[i >> 1]));
      y[i] = to_odd(p0);
      y[i + 1] = to_odd(p1);
      // hardly ever, in any lane: a jump
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(is_subnormal(y[i]) | is_subnormal(y[i + 1])) != 0, 0)) {
        y[i] = is_subnormal(y[i]) ? to_odd_small(p0) : y[i];
        y[i + 1] = is_subnormal(y[i + 1]) ? to_odd_small(p1) : y[i + 1];
      }
    }
    if (normed && ok)
      *reinterpret_cast<uint4*>(normed + at) =
          make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                     pack_bf16x2(y[6], y[7]));
    if (codes) {
      uint32_t w[2];
      const uint32_t scale = mx_encode8<kMxE4M3>(y, w);
      mx_store8<kMxE4M3>(codes + base, scales + (base >> 5), v, ok, whole, w, scale);
    }
  }
}

template <int CH>
void launch_norm(bool x32, const void* x, const uint16_t* residual, const uint16_t* weight,
                 double eps, uint16_t* residual_out, uint16_t* normed, uint8_t* codes,
                 uint8_t* scales, int rows, int hidden, hipStream_t stream) {
  const int waves = ceil_div(hidden / 8, 64 * CH), per = waves == 1 ? 4 : 1;
  const auto kernel = x32 ? add_rmsnorm_kernel<CH, true> : add_rmsnorm_kernel<CH, false>;
  const int most = (1 << 25) / waves;  // rows a launch: below 2^32 threads, a multiple of four where per is
  for (int r = 0; r < rows; r += most) {
    const int n = rows - r < most ? rows - r : most;
    const long long at = static_cast<long long>(r) * hidden;
    hipLaunchKernelGGL(kernel, dim3(ceil_div(n, per)), dim3(64 * waves, per), 0, stream,
                       static_cast<const uint8_t*>(x) + (x32 ? 4 : 2) * at, residual ? residual + at : nullptr,
                       weight, eps, residual_out ? residual_out + at : nullptr, normed ? normed + at : nullptr,
                       codes ? codes + at : nullptr, scales ? scales + at / kMxBlock : nullptr, n, hidden);
    if (rows - r <= most) break;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace pega

using namespace pega;

// No reference counterpart as one symbol: the add and the norm between two blocks.
PEGA_API int pega_add_rmsnorm(const void* x, bool x_is_f32, const uint16_t* residual,
                              const uint16_t* weight, double eps, uint16_t* residual_out,
                              uint16_t* normed, uint8_t* mxfp8_codes, uint8_t* mxfp8_scales,
                              int rows, int hidden_dim, hipStream_t stream) {
  if (rows < 0 || hidden_dim <= 0 || !(eps >= 0.0))
    return fail(kInvalidValue, "add_rmsnorm: bad arguments (rows=%d hidden=%d)", rows, hidden_dim);
  if (rows == 0) return kSuccess;  // empty tensors have no address
  if (!x || !weight) return fail(kInvalidValue, "add_rmsnorm: null pointer");
  if (!residual_out && !normed && !mxfp8_codes)
    return fail(kInvalidValue, "add_rmsnorm: no output");
  if (!mxfp8_codes != !mxfp8_scales)
    return fail(kInvalidValue, "add_rmsnorm: MXFP8 codes and scales go together");
  if (hidden_dim % 8 != 0 || hidden_dim > 32768 || (mxfp8_codes && hidden_dim % kMxBlock != 0))
    return fail(kNotSupported, "add_rmsnorm: hidden_dim %d (a multiple of 8, of 32 for MXFP8, at "
                "most 32768)", hidden_dim);
  if (!aligned16(x) || !aligned16(residual) || !aligned16(weight) || !aligned16(residual_out) ||
      !aligned16(normed) || !aligned16(mxfp8_codes) || (reinterpret_cast<uintptr_t>(mxfp8_scales) & 3u))
    return fail(kNotSupported, "add_rmsnorm: buffers must be 16-byte aligned (scales 4)");
  // An output may be the bf16 buffer of x or of residual, row for row; any other overlap would
  // let one row's stores meet another row's loads.
  const long long n = static_cast<long long>(rows) * hidden_dim;
  struct Span { const void* p; long long bytes; };
  const Span outs[4] = {{residual_out, 2 * n}, {normed, 2 * n}, {mxfp8_codes, n}, {mxfp8_scales, n / kMxBlock}};
  const Span ins[3] = {{x, (x_is_f32 ? 4 : 2) * n}, {residual, 2 * n}, {weight, 2LL * hidden_dim}};
  for (int o = 0; o < 4; ++o) {
    for (int i = 0; i < 3; ++i)
      if (overlap(outs[o].p, outs[o].bytes, ins[i].p, ins[i].bytes) &&
          !(o < 2 && i < 2 && outs[o].p == ins[i].p && ins[i].bytes == 2 * n))
        return fail(kInvalidValue, "add_rmsnorm: an output overlaps an input");
    for (int i = 0; i < o; ++i)
      if (overlap(outs[o].p, outs[o].bytes, outs[i].p, outs[i].bytes))
        return fail(kInvalidValue, "add_rmsnorm: two outputs overlap");
  }
  const int vecs = hidden_dim / 8;
#define PEGA_NORM(CH) \
  launch_norm<CH>(x_is_f32, x, residual, weight, eps, residual_out, normed, mxfp8_codes, \
                  mxfp8_scales, rows, hidden_dim, stream)
  // Few vectors a lane finish a row soonest, but a CU must hold eight waves a SIMD for the memory:
  // one vector up to four waves, two up to eight.  More than a few thousand waves keep the memory
  // busy anyway and then gain from fewer of them: 7168 columns take 5.0 us (two vectors a lane)
  // against 5.5 (four) at one row, 19 both at 1024, 61 against 57 at 4096.
  if (vecs <= 4 * 64) PEGA_NORM(1);
  else if (vecs <= 8 * 2 * 64 && (vecs <= 8 * 64 || rows <= 1024)) PEGA_NORM(2);
  else PEGA_NORM(4);
#undef PEGA_NORM
  return launch_status("add_rmsnorm");
}

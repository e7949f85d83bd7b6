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

// y in fp32 for one more rounding (to_odd, to_odd_small where one of the wave's pairs needs it).
__device__ __forceinline__ void to_odd2(double p0, double p1, float* y) {
  y[0] = to_odd(p0);
  y[1] = to_odd(p1);
  // hardly ever, in any lane: a jump
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(is_subnormal(y[0]) || is_subnormal(y[1])) != 0, 0)) {
    y[0] = is_subnormal(y[0]) ? to_odd_small(p0) : y[0];
    y[1] = is_subnormal(y[1]) ? to_odd_small(p1) : y[1];
  }
}

// The sum over a row's lanes, in each of them.  s_sum: a place a wave, used by this sum alone.
__device__ __forceinline__ double row_sum(double sum, double* s_sum, int lanes, int lane) {
  sum = sum16(sum);
  sum = (lane_f64(sum, 0) + lane_f64(sum, 16)) + (lane_f64(sum, 32) + lane_f64(sum, 48));
  if (lanes > 64) {
    if ((lane & 63) == 0) s_sum[lane >> 6] = sum;
    __syncthreads();
    const int w = lane & 15;
    sum = sum16(w < lanes >> 6 ? s_sum[w] : 0.0);
  }
  return sum;
}

__device__ __forceinline__ float bf_at(uint4 q, int i) {
  const uint32_t w = (i >> 1) == 0 ? q.x : (i >> 1) == 1 ? q.y : (i >> 1) == 2 ? q.z : q.w;
  return (i & 1) ? bf_hi(w) : bf_lo(w);
}

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
  const double inv = 1.0 / __builtin_sqrt(row_sum(sum, s_sum, lanes, lane) / hidden + eps);

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
    for (int i = 0; i < 8; i += 2)
      to_odd2(s[c][i] * inv * static_cast<double>(bf_lo(ww[i >> 1])),
              s[c][i + 1] * inv * static_cast<double>(bf_hi(ww[i >> 1])), y + i);
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

// The same between two blocks that are normed on both sides:
//
//   y = x * post_weight / sqrt(mean(x^2) + eps)      (x itself without a post_weight)
//   s = residual_scale * residual + gate * y         residual_out = bf16(s)
//   z = s * pre_weight / sqrt(mean(s^2) + eps)       normed = bf16(z), codes, scales = MXFP8(z)
//
// with a gate for each column, each row, each value, or none, and weights that are stored less one
// (`one` = 1) or as they are (0).  One pass as above with two sums; all loads of a row are in flight
// before the first sum, and the row stays in registers until its last output is stored, so that
// each value is read and written once.  Sums, norms and s are in 64 bits.
// One row is bound by its latency, of the loads and of two sums over the workgroup one after the
// other: 6.0 us for 7168 columns.  Many bf16 rows are bound by memory: 4096 x 7168 with a gate for
// each value, bf16 and MXFP8 outputs 66 us, 4.9 TB/s.
struct SandwichArgs {
  const void* x;
  const uint16_t *residual, *post, *pre, *gate;
  long long gate_row;  // elements from a row's gate to the next row's
  bool gate_cols;      // a gate for each column of a row, not one for the row
  double eps, scale, one;
  uint16_t *residual_out, *normed;
  uint8_t *codes, *scales;
  int rows, hidden;
};

// What a wave's lanes have written to LDS before, its lanes read behind it (a wave's own accesses go in order).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A lane's 8 columns of an fp32 row are two loads' worth.  Taken as they lie, each load of a wave would touch
// half of every line; so a wave loads its 128 pieces of 16 bytes in order, and its lanes exchange them
// (4096 rows of 7168 columns 104 us without, 69 with; 333 of 2048 6.2 and 5.3).
template <int CH, bool kX32>
__global__ __launch_bounds__(64 * kMaxWaves) void sandwich_rmsnorm_kernel(
    SandwichArgs p) {
  __shared__ double s_sum[2][kMaxWaves];
  const int lanes = blockDim.x, lane = threadIdx.x, in_wave = lane & 63;
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int vecs = p.hidden >> 3;
  const bool in = row < p.rows;
  const long long base = static_cast<long long>(row) * p.hidden;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint4 ones = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);
  const uint4 none = make_uint4(0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u);  // -0: adds nothing

  uint4 xr[CH][kX32 ? 2 : 1], rr[CH], pw[CH], gr[CH], nw[CH];
  uint4 gate_one = ones;
  if (p.gate && !p.gate_cols && in) {
    const uint32_t g = p.gate[row * p.gate_row] * 0x10001u;
    gate_one = make_uint4(g, g, g, g);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int v = lane + c * lanes;
    const bool ok = in && v < vecs;
    const long long at = base + 8LL * v;
    if constexpr (kX32) {  // pieces of 4 columns, each load's side by side
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p.x) + base);
      const int piece = 2 * (v - in_wave) + in_wave;
      xr[c][0] = in && piece < 2 * vecs ? q[piece] : zero;
      xr[c][1] = in && piece + 64 < 2 * vecs ? q[piece + 64] : zero;
    } else {
      xr[c][0] = ok ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + at) : zero;
    }
    rr[c] = none;
    if (ok && p.residual) rr[c] = *reinterpret_cast<const uint4*>(p.residual + at);
    gr[c] = gate_one;
    if (ok && p.gate_cols) gr[c] = *reinterpret_cast<const uint4*>(p.gate + row * p.gate_row + 8 * v);
    pw[c] = ones;
    if (v < vecs && p.post) pw[c] = *reinterpret_cast<const uint4*>(p.post + 8 * v);
    nw[c] = zero;
    if (v < vecs && p.pre) nw[c] = *reinterpret_cast<const uint4*>(p.pre + 8 * v);
  }
  if constexpr (kX32) {  // a lane's two pieces, by way of its wave's part of LDS
    extern __shared__ uint4 s_x[];
    uint4* part = s_x + 128 * ((threadIdx.y * blockDim.x + threadIdx.x) >> 6);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      // (even pieces in one half, odd ones in the other, so that the reads meet no bank twice)
      part[(in_wave >> 1) + 64 * (in_wave & 1)] = xr[c][0];
      part[(in_wave >> 1) + 64 * (in_wave & 1) + 32] = xr[c][1];
      wave_sync();
      xr[c][0] = part[in_wave];
      xr[c][1] = part[in_wave + 64];
      wave_sync();
    }
  }
  const auto x_at = [&](int c, int i) {
    if constexpr (kX32) {
      const uint4 q = xr[c][i >> 2];
      return __builtin_bit_cast(float, (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w);
    } else {
      return bf_at(xr[c][0], i);
    }
  };
  double inv = 1.0;
  const double post_one = p.post ? p.one : 0.0;
  if (p.post) {
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double v = static_cast<double>(x_at(c, i));
        sum = __builtin_fma(v, v, sum);
      }
    inv = 1.0 / __builtin_sqrt(row_sum(sum, s_sum[0], lanes, lane) / p.hidden + p.eps);
  }
  double s[CH][8], sum = 0.0;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double y = static_cast<double>(x_at(c, i));
      if (p.post) y = y * inv * (post_one + static_cast<double>(bf_at(pw[c], i)));
      const double r = p.scale * static_cast<double>(bf_at(rr[c], i));
      s[c][i] = p.gate ? __builtin_fma(static_cast<double>(bf_at(gr[c], i)), y, r) : y + r;
      if (lane + c * lanes >= vecs) s[c][i] = 0.0;  // a row's gate may be an infinity
      sum = __builtin_fma(s[c][i], s[c][i], sum);
    }
  if (p.residual_out) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int v = lane + c * lanes;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) to_odd2(s[c][i], s[c][i + 1], y + i);
      if (in && v < vecs)
        *reinterpret_cast<uint4*>(p.residual_out + base + 8LL * v) =
            make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                       pack_bf16x2(y[6], y[7]));
    }
  }
  if (!p.pre) return;
  inv = 1.0 / __builtin_sqrt(row_sum(sum, s_sum[1], lanes, lane) / p.hidden + p.eps);
  const bool whole = (p.hidden & 127) == 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int v = lane + c * lanes;
    const bool ok = in && v < vecs;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      to_odd2(s[c][i] * inv * (p.one + static_cast<double>(bf_at(nw[c], i))),
              s[c][i + 1] * inv * (p.one + static_cast<double>(bf_at(nw[c], i + 1))), y + i);
    if (p.normed && ok)
      *reinterpret_cast<uint4*>(p.normed + base + 8LL * v) =
          make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                     pack_bf16x2(y[6], y[7]));
    if (p.codes) {
      uint32_t w[2];
      const uint32_t scale = mx_encode8<kMxE4M3>(y, w);
      mx_store8<kMxE4M3>(p.codes + base, p.scales + (base >> 5), v, ok, whole, w, scale);
    }
  }
}

template <int CH>
void launch_sandwich(SandwichArgs p, bool x32, hipStream_t stream) {
  const int waves = ceil_div(p.hidden / 8, 64 * CH), per = waves == 1 ? 4 : 1;
  const auto kernel = x32 ? sandwich_rmsnorm_kernel<CH, true> : sandwich_rmsnorm_kernel<CH, false>;
  const int most = (1 << 25) / waves;  // rows a launch, as launch_norm's
  for (int rows = p.rows;; rows -= most) {
    p.rows = rows < most ? rows : most;
    hipLaunchKernelGGL(kernel, dim3(ceil_div(p.rows, per)), dim3(64 * waves, per), x32 ? 2048 * waves * per : 0, stream,
                       p);
    if (rows <= most) return;
    const long long at = static_cast<long long>(most) * p.hidden;
    p.x = static_cast<const uint8_t*>(p.x) + (x32 ? 4 : 2) * at;
    if (p.residual) p.residual += at;
    if (p.gate) p.gate += most * p.gate_row;
    if (p.residual_out) p.residual_out += at;
    if (p.normed) p.normed += at;
    if (p.codes) p.codes += at, p.scales += at / kMxBlock;
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

// No reference counterpart: what stands between two blocks normed on both sides.
PEGA_API int pega_sandwich_rmsnorm(const void* x, bool x_is_f32, const uint16_t* residual,
                                   double residual_scale, const uint16_t* post_weight,
                                   const uint16_t* gate, int gate_kind, const uint16_t* pre_weight,
                                   bool unit_offset, double eps, uint16_t* residual_out,
                                   uint16_t* normed, uint8_t* mxfp8_codes, uint8_t* mxfp8_scales,
                                   int rows, int hidden_dim, hipStream_t stream) {
  if (rows < 0 || hidden_dim <= 0 || !(eps >= 0.0) || gate_kind < 0 || gate_kind > 3)
    return fail(kInvalidValue, "sandwich_rmsnorm: bad arguments (rows=%d hidden=%d gate_kind=%d)", rows,
                hidden_dim, gate_kind);
  if (rows == 0) return kSuccess;  // empty tensors have no address
  const bool want_norm = normed || mxfp8_codes;
  if (!x || (gate_kind != 0 && !gate) || (want_norm && !pre_weight))
    return fail(kInvalidValue, "sandwich_rmsnorm: null pointer");
  if (!residual_out && !want_norm) return fail(kInvalidValue, "sandwich_rmsnorm: no output");
  if (!mxfp8_codes != !mxfp8_scales)
    return fail(kInvalidValue, "sandwich_rmsnorm: MXFP8 codes and scales go together");
  if (hidden_dim % 8 != 0 || hidden_dim > 32768 || (mxfp8_codes && hidden_dim % kMxBlock != 0))
    return fail(kNotSupported, "sandwich_rmsnorm: hidden_dim %d (a multiple of 8, of 32 for MXFP8, at "
                "most 32768)", hidden_dim);
  if (!aligned16(x) || !aligned16(residual) || !aligned16(post_weight) || !aligned16(pre_weight) ||
      (gate_kind == 2 ? reinterpret_cast<uintptr_t>(gate) & 1u : gate_kind != 0 && !aligned16(gate)) ||
      !aligned16(residual_out) || !aligned16(normed) || !aligned16(mxfp8_codes) ||
      (reinterpret_cast<uintptr_t>(mxfp8_scales) & 3u))
    return fail(kNotSupported, "sandwich_rmsnorm: buffers must be 16-byte aligned (scales 4, a gate per "
                "row 2)");
  // As in add_rmsnorm: an output may be the bf16 buffer of x or of residual, and overlaps nothing else.
  const long long n = static_cast<long long>(rows) * hidden_dim;
  const long long gates = gate_kind == 0 ? 0 : gate_kind == 1 ? hidden_dim : gate_kind == 2 ? rows : n;
  struct Span { const void* p; long long bytes; };
  const Span outs[4] = {{residual_out, 2 * n}, {normed, 2 * n}, {mxfp8_codes, n}, {mxfp8_scales, n / kMxBlock}};
  const Span ins[5] = {{x, (x_is_f32 ? 4 : 2) * n}, {residual, 2 * n}, {post_weight, 2LL * hidden_dim},
                       {pre_weight, 2LL * hidden_dim}, {gate, 2 * gates}};
  for (int o = 0; o < 4; ++o) {
    for (int i = 0; i < 5; ++i)
      if (overlap(outs[o].p, outs[o].bytes, ins[i].p, ins[i].bytes) &&
          !(o < 2 && i < 2 && outs[o].p == ins[i].p && ins[i].bytes == 2 * n))
        return fail(kInvalidValue, "sandwich_rmsnorm: an output overlaps an input");
    for (int i = 0; i < o; ++i)
      if (overlap(outs[o].p, outs[o].bytes, outs[i].p, outs[i].bytes))
        return fail(kInvalidValue, "sandwich_rmsnorm: two outputs overlap");
  }
  SandwichArgs p{x, residual, post_weight, want_norm ? pre_weight : nullptr, gate_kind ? gate : nullptr,
                 gate_kind == 2 ? 1 : gate_kind == 3 ? hidden_dim : 0, gate_kind == 1 || gate_kind == 3,
                 eps, residual ? residual_scale : 1.0, unit_offset ? 1.0 : 0.0, residual_out, normed,
                 mxfp8_codes, mxfp8_scales, rows, hidden_dim};
  const int vecs = hidden_dim / 8;
  // Vectors a lane, in us without MXFP8, a gate for each row (bf16 x unless fp32 is said).  More of
  // them take fewer waves to a row and more registers to a lane; with fp32 rows four spill 69, and are taken
  // above 16384 columns alone, where two would need more waves than a workgroup has (1024 rows of 32768 columns
  // 167 us, bf16 82).
  //   one or two:  4096 columns, 1 row 4.3 and 4.8; 4096 rows 37.0 and 33.6, fp32 39.6 and 38.7;
  //                7168 columns, 1024 rows 25.4 and 19.2, fp32 27.3 and 23.2; 2048 columns, 1 row 3.6 and 4.4
  //   two or four: 7168 columns, 1 row 6.0 and 7.3; 4096 fp32 rows 71 and 150; 8192 columns, 4096 rows
  //                56.5 and 54.4; 16384 columns, 1 row 9.7 and 10.0, 1024 rows 46 and 35, fp32 56 and 83
  if (vecs <= 256 || (vecs <= 640 && (x_is_f32 || rows <= 256))) launch_sandwich<1>(p, x_is_f32, stream);
  else if (vecs <= 512 || (vecs <= 1024 && rows <= 1024) || (vecs <= 2048 && x_is_f32))
    launch_sandwich<2>(p, x_is_f32, stream);
  else launch_sandwich<4>(p, x_is_f32, stream);
  return launch_status("sandwich_rmsnorm");
}

// Rows into a microscaled format and back (mx_format.h): the load-time quantisation of MXFP4
// weights, the activations' quantisation in front of an MX product, SwiGLU with the quantisation
// in its epilogue, and the values that codes and scales stand for.  Each is one pass over its
// bytes; eight columns a lane, 16-byte loads.  9728 x 2560, three sets in turn: to MXFP4 and back 10.7 us
// each (63 MB, 5.9 TB/s, partly out of the last-level cache), to MXFP8 and back 12.5; 16384 x 7168 to
// MXFP4 52 us (5.7 TB/s; a copy of 1 GiB reaches 5.1), to MXFP8 61 us.  The bytes bound these.  SwiGLU of
// 9728 x 2560 takes 32 us to MXFP8 (126 MB, 3.9 TB/s) and 31 to MXFP4 (113 MB), of four times the rows 116
// and 113 (4.3 and 4.0 TB/s): the vector instructions bound it, 386 for a wave's 512 values (the hardware
// exponential, a division and the checks that make it the exact bf16 SwiGLU), four cycles each.
#include "common.h"
#include "mx_format.h"
#include "pega_moe.h"

namespace pega {
namespace {

constexpr int kThreads = 256;

// Rows lie one after another, blocks never cross a row, and a row's scales are next to the one's
// before: but for SwiGLU's operands the rows are one long row of `vecs` vectors of 8, a lane each.
// (Four a lane, their loads ahead of their work, measured the same on long tensors, 16384 x 7168
// to MXFP8 in 63 against 62 us, and lost 0.3 us on short ones.)
// kSwiglu: x holds gate then up columns (row_vecs vectors each), and the values are SwiGLU's bf16
// (swiglu_one).
template <int kFormat, bool kSwiglu>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const uint16_t* __restrict__ x,
                                                               uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales,
                                                               uint32_t vecs, uint32_t row_vecs) {
  const uint32_t v8 = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t from = min(v8, vecs - 1);
  const uint4* p = reinterpret_cast<const uint4*>(x) + from;
  float v[8];
  if constexpr (kSwiglu) {
    p += static_cast<long long>(from / row_vecs) * row_vecs;  // the up columns of the rows before
    const uint4 g = p[0], u = p[row_vecs];
    const uint32_t gw[4] = {g.x, g.y, g.z, g.w}, uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = bf2f(swiglu_one(bf_lo(gw[k]), bf_lo(uw[k])));
      v[2 * k + 1] = bf2f(swiglu_one(bf_hi(gw[k]), bf_hi(uw[k])));
    }
  } else {
    const uint4 a = p[0];
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = bf_lo(aw[k]);
      v[2 * k + 1] = bf_hi(aw[k]);
    }
  }
  uint32_t w[2];
  const uint32_t scale = mx_encode8<kFormat>(v, w);
  mx_store8<kFormat>(codes, scales, v8, v8 < vecs, (v8 | 15u) < vecs, w, scale);
}

// The value of a code times its scale has at most four significant bits, so bf16 holds it exactly
// (down to bf16's own smallest numbers).
template <int kFormat>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales,
                                                                 uint16_t* __restrict__ out,
                                                                 uint32_t vecs) {
  const uint32_t v8 = blockIdx.x * kThreads + threadIdx.x;
  if (v8 >= vecs) return;
  const uint32_t sb = scales[v8 >> 2];
  // 2^s as a float: 2^-127 is below the normal range, 255 is NaN
  const float s = __builtin_bit_cast(float, sb == 0 ? 0x00400000u : sb == 255u ? 0x7fc00000u : sb << 23);
  float v[8];
  if constexpr (kFormat == kMxE4M3) {
    const uint2 q = reinterpret_cast<const uint2*>(codes)[v8];
    const uint32_t w[2] = {q.x, q.y};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[h]), false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[h]), true);
      v[4 * h] = lo[0];
      v[4 * h + 1] = lo[1];
      v[4 * h + 2] = hi[0];
      v[4 * h + 3] = hi[1];
    }
  } else {
    const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[v8];
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
    v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
  }
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(v[2 * j] * s, v[2 * j + 1] * s);
  reinterpret_cast<uint4*>(out)[v8] = make_uint4(o[0], o[1], o[2], o[3]);
}

// A kernel indexes a launch's vectors with 32 bits: longer tensors are worked on in runs of rows
// (multiples of four, which keep the scales' alignment).  launch(first value, its vectors, blocks).
template <typename Launch>
void in_runs(int rows, int cols, Launch launch) {
  const long long most = ((1LL << 33) / cols) & ~3LL;  // 2^30 vectors; cols is at most 2^30
  for (long long r = 0; r < rows; r += most) {
    const uint32_t vecs = static_cast<uint32_t>((rows - r < most ? rows - r : most) * (cols / 8));
    launch(r * cols, vecs, dim3((vecs + kThreads - 1) / kThreads));
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// `row_bytes`: of a row of rows_bf16.
int mx_checks(const char* name, const void* rows_bf16, long long row_bytes, const void* codes,
              const void* scales, int format, int rows, int cols) {
  if (rows < 0 || cols <= 0) return fail(kInvalidValue, "%s: bad arguments (rows=%d cols=%d)", name, rows, cols);
  // no rows: nothing to do, and empty tensors have no address
  if (rows > 0 && (!rows_bf16 || !codes || !scales)) return fail(kInvalidValue, "%s: null pointer", name);
  if (format != kMxE4M3 && format != kMxE2M1)
    return fail(kInvalidValue, "%s: format %d (0 E4M3, 1 E2M1)", name, format);
  if (cols % kMxBlock != 0 || cols > (1 << 30))
    return fail(kNotSupported, "%s: cols %d is not a multiple of %d up to 2^30", name, cols, kMxBlock);
  if (!aligned(rows_bf16, 16) || !aligned(codes, 16) || !aligned(scales, 4))
    return fail(kNotSupported, "%s: buffers must be 16-byte aligned (scales 4)", name);
  const long long n = static_cast<long long>(rows) * cols, nc = mx_code_bytes(format, n);
  if (overlap(rows_bf16, rows * row_bytes, codes, nc) ||
      overlap(rows_bf16, rows * row_bytes, scales, n / kMxBlock) ||
      overlap(codes, nc, scales, n / kMxBlock))
    return fail(kInvalidValue, "%s: buffers overlap", name);
  return kSuccess;
}

template <bool kSwiglu>
int quantize_launch(const char* name, const uint16_t* x, uint8_t* codes, uint8_t* scales,
                    int format, int rows, int cols, hipStream_t stream) {
  const int rc = mx_checks(name, x, (kSwiglu ? 4LL : 2LL) * cols, codes, scales, format, rows, cols);
  if (rc != kSuccess) return rc;
  if (rows == 0) return kSuccess;
  in_runs(rows, cols, [&](long long at, uint32_t vecs, dim3 grid) {
    const auto kernel = format == kMxE4M3 ? mx_quantize_kernel<kMxE4M3, kSwiglu>
                                          : mx_quantize_kernel<kMxE2M1, kSwiglu>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, x + at * (kSwiglu ? 2 : 1),
                       codes + mx_code_bytes(format, at), scales + at / kMxBlock, vecs,
                       static_cast<uint32_t>(cols / 8));
  });
  return launch_status(name);
}

}  // namespace
}  // namespace pega

using namespace pega;

// No reference counterpart (the reference's experts are INT4): rows of bf16 into an MX format.
PEGA_API int pega_mx_quantize(const uint16_t* x, uint8_t* codes, uint8_t* scales, int format,
                              int rows, int cols, hipStream_t stream) {
  return quantize_launch<false>("mx_quantize", x, codes, scales, format, rows, cols, stream);
}

// No reference counterpart: kimi_marlin_w13_swiglu_cuda then pega_mx_quantize in one pass.
PEGA_API int pega_mx_swiglu_quantize(const uint16_t* w13, uint8_t* codes, uint8_t* scales,
                                     int format, int rows, int intermediate_dim,
                                     hipStream_t stream) {
  return quantize_launch<true>("mx_swiglu_quantize", w13, codes, scales, format, rows,
                               intermediate_dim, stream);
}

// No reference counterpart: the values that codes and scales stand for, as bf16.
PEGA_API int pega_mx_dequantize(const uint8_t* codes, const uint8_t* scales, uint16_t* out,
                                int format, int rows, int cols, hipStream_t stream) {
  const int rc = mx_checks("mx_dequantize", out, 2LL * cols, codes, scales, format, rows, cols);
  if (rc != kSuccess) return rc;
  if (rows == 0) return kSuccess;
  in_runs(rows, cols, [&](long long at, uint32_t vecs, dim3 grid) {
    const auto kernel = format == kMxE4M3 ? mx_dequantize_kernel<kMxE4M3> : mx_dequantize_kernel<kMxE2M1>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, codes + mx_code_bytes(format, at),
                       scales + at / kMxBlock, out + at, vecs);
  });
  return launch_status("mx_dequantize");
}

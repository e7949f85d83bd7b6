// Rows into a microscaled format and back (mx_format.h): the load-time quantisation of MXFP4
// weights, the activations' quantisation in front of an MX product, SwiGLU with the quantisation
// in its epilogue, and the values that codes and scales stand for.  Each is one pass over its
// bytes, which bound it; eight columns a lane, 16-byte loads.
#include "common.h"
#include "mx_format.h"
#include "pega_moe.h"

namespace pega {
namespace {

constexpr int kThreads = 256;

// kSwiglu: x holds gate then up columns, and the values are SwiGLU's bf16 (swiglu_one).  A wave
// takes 64 vectors of one row at a time (a row's vectors in steps of 64, padded), so that the
// lanes of a block are lane quads whatever the width.
template <int kFormat, bool kSwiglu>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const uint16_t* __restrict__ x,
                                                               uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales,
                                                               int rows, int cols) {
  const int vecs = cols >> 3, spans = ceil_div(vecs, 64);
  const int lane = threadIdx.x & 63;
  const long long units = static_cast<long long>(rows) * spans;
  const bool whole = (cols & 127) == 0;
  for (long long u = static_cast<long long>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
       u < units; u += static_cast<long long>(gridDim.x) * (kThreads / 64)) {
    const long long row = u / spans;
    const int v8 = static_cast<int>(u - row * spans) * 64 + lane;
    const bool live = v8 < vecs;
    float v[8] = {};
    if (live) {
      const uint16_t* p = x + row * cols * (kSwiglu ? 2 : 1) + 8 * v8;
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
      if constexpr (kSwiglu) {
        const uint4 b = *reinterpret_cast<const uint4*>(p + cols);
        const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = bf2f(swiglu_one(bf_lo(aw[i]), bf_lo(bw[i])));
          v[2 * i + 1] = bf2f(swiglu_one(bf_hi(aw[i]), bf_hi(bw[i])));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = bf_lo(aw[i]);
          v[2 * i + 1] = bf_hi(aw[i]);
        }
      }
    }
    uint32_t w[2];
    const uint32_t scale = mx_encode8<kFormat>(v, w);
    const long long at = row * cols;
    mx_store8<kFormat>(codes + mx_code_bytes(kFormat, at), scales + (at >> 5), v8, live, whole, w,
                       scale);
  }
}

// The value of a code times its scale has at most four significant bits, so bf16 holds it exactly
// (down to bf16's own smallest numbers).
template <int kFormat>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales,
                                                                 uint16_t* __restrict__ out,
                                                                 long long vecs) {
  for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < vecs;
       i += static_cast<long long>(gridDim.x) * kThreads) {
    const uint32_t sb = scales[i >> 2];
    // 2^s as a float: 2^-127 is below the normal range, 255 is NaN
    const float s = __builtin_bit_cast(float, sb == 0 ? 0x00400000u : sb == 255u ? 0x7fc00000u : sb << 23);
    float v[8];
    if constexpr (kFormat == kMxE4M3) {
      const uint2 q = *reinterpret_cast<const uint2*>(codes + 8 * i);
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
      const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + 4 * i);
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
    *reinterpret_cast<uint4*>(out + 8 * i) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// `row_bytes`: of a row of rows_bf16.
int mx_checks(const char* name, const void* rows_bf16, long long row_bytes, const void* codes,
              const void* scales, int format, int rows, int cols) {
  if (!rows_bf16 || !codes || !scales || rows < 0 || cols <= 0)
    return fail(kInvalidValue, "%s: bad arguments (rows=%d cols=%d)", name, rows, cols);
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
  const long long units = static_cast<long long>(rows) * ceil_div(cols / 8, 64);
  const long long want = (units + kThreads / 64 - 1) / (kThreads / 64);
  const dim3 grid(static_cast<unsigned>(want < (1 << 20) ? want : (1 << 20)));
  if (format == kMxE4M3)
    hipLaunchKernelGGL((mx_quantize_kernel<kMxE4M3, kSwiglu>), grid, dim3(kThreads), 0, stream, x,
                       codes, scales, rows, cols);
  else
    hipLaunchKernelGGL((mx_quantize_kernel<kMxE2M1, kSwiglu>), grid, dim3(kThreads), 0, stream, x,
                       codes, scales, rows, cols);
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
  const long long vecs = static_cast<long long>(rows) * (cols / 8);
  const long long want = (vecs + kThreads - 1) / kThreads;
  const dim3 grid(static_cast<unsigned>(want < (1 << 20) ? want : (1 << 20)));
  if (format == kMxE4M3)
    hipLaunchKernelGGL((mx_dequantize_kernel<kMxE4M3>), grid, dim3(kThreads), 0, stream, codes,
                       scales, out, vecs);
  else
    hipLaunchKernelGGL((mx_dequantize_kernel<kMxE2M1>), grid, dim3(kThreads), 0, stream, codes,
                       scales, out, vecs);
  return launch_status("mx_dequantize");
}

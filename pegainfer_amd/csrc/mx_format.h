// Microscaled formats (OCP MX): 32 consecutive values of a row share one power-of-two scale, a
// byte s + 127 (E8M0, 255 = NaN); the values are E4M3 bytes or E2M1 nibbles, the even column of a
// byte low.  Rows are stored one after another, codes [rows][cols] bytes (E4M3) or [rows][cols / 2]
// (E2M1), scales [rows][cols / 32].
//
// The scale is the smallest 2^s, s >= -127, for which the block's largest magnitude still rounds
// to a value of the format: amax <= 464 * 2^s in E4M3 (448 is its largest value, 480 would be the
// next, and the tie at 464 goes to the even 448), amax < 7 * 2^s in E2M1 (6, then 8, the tie at 7
// going to 8).  With it no value is off by more than half a step of its own binade; the power of
// two below (the largest not above amax, over the format's) would cut E4M3 values off by up to an
// eighth.  A block that holds an infinity or a NaN has scale 255, so that every value of it reads
// as NaN, and codes 0.
#pragma once

#include "common.h"

namespace pega {

constexpr int kMxBlock = 32;
enum MxFormat : int { kMxE4M3 = 0, kMxE2M1 = 1 };

__host__ __device__ constexpr long long mx_code_bytes(int format, long long values) {
  return format == kMxE4M3 ? values : values / 2;
}

// Lane moves inside rows of 16 lanes, without an "old" operand.
template <int kCtrl>
__device__ __forceinline__ uint32_t mx_dpp(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_mov_dpp(static_cast<int>(v), kCtrl, 0xF, 0xF, true));
}

// Scale byte of a block whose largest magnitude has the float bits `amax` (sign cleared; bits of
// a NaN or an infinity are the largest, so an unsigned maximum finds them).
template <int kFormat>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  constexpr int kTop = kFormat == kMxE4M3 ? 8 : 2;  // exponent of the format's largest value
  const int up = kFormat == kMxE4M3 ? (amax & 0x7fffffu) > 0x680000u    // 464 = 1.8125 * 2^8
                                    : (amax & 0x7fffffu) >= 0x600000u;  // 7 = 1.75 * 2^2
  const int s = static_cast<int>(amax >> 23) - kTop + up;
  return amax >= 0x7f800000u ? 255u : static_cast<uint32_t>(s > 0 ? s : 0);
}

// Eight consecutive values v of a block that lanes 4 i .. 4 i + 3 hold: the block's scale byte in
// every lane, the codes in out[0] (and out[1] for E4M3).  v * 2^-s is exact (where it falls among
// fp32's smallest numbers, the code is 0 either way), and the conversion rounds to nearest, ties
// to even.
template <int kFormat>
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], uint32_t (&out)[2]) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
    amax = amax > b ? amax : b;
  }
  uint32_t o = mx_dpp<0xB1>(amax);  // quad_perm [1,0,3,2]
  amax = amax > o ? amax : o;
  o = mx_dpp<0x4E>(amax);  // quad_perm [2,3,0,1]
  amax = amax > o ? amax : o;
  const uint32_t scale = mx_scale_byte<kFormat>(amax);
  const bool bad = scale == 255u;
  const float inv = __builtin_bit_cast(float, (254u - (bad ? 0u : scale)) << 23);  // 2^-s
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = v[i] * inv;
  if constexpr (kFormat == kMxE4M3) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * h], u[4 * h + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * h + 2], u[4 * h + 3], w, true);
      out[h] = bad ? 0u : static_cast<uint32_t>(w);
    }
  } else {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, u[0], u[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, u[2], u[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, u[4], u[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, u[6], u[7], 1.0f, 3);
    out[0] = bad ? 0u : w;
    out[1] = 0u;
  }
  return scale;
}

// Stores those codes and the scale byte at vector `v8` (8 columns each) of a row's codes and
// scales.  `whole`: the row is a multiple of 128 columns, so that the four blocks of a 16-lane
// row have one aligned word of scales, which its first lane stores (their bytes come over lane
// moves); otherwise each block's first lane stores its byte.  The 16 lanes hold consecutive
// vectors from a multiple of 16 on.
template <int kFormat>
__device__ __forceinline__ void mx_store8(uint8_t* codes, uint8_t* scales, int v8, bool live,
                                          bool whole, const uint32_t (&w)[2], uint32_t scale) {
  uint32_t four = scale | (mx_dpp<0x104>(scale) << 8);  // row_shl:4
  four |= mx_dpp<0x108>(scale) << 16;                   // row_shl:8
  four |= mx_dpp<0x10C>(scale) << 24;                   // row_shl:12
  if (!live) return;
  if constexpr (kFormat == kMxE4M3)
    *reinterpret_cast<uint2*>(codes + 8 * static_cast<long long>(v8)) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(codes + 4 * static_cast<long long>(v8)) = w[0];
  if (whole) {
    if ((v8 & 15) == 0) *reinterpret_cast<uint32_t*>(scales + (v8 >> 2)) = four;
  } else if ((v8 & 3) == 0) {
    scales[v8 >> 2] = static_cast<uint8_t>(scale);
  }
}

}  // namespace pega

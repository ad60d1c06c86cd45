// 8-bit activations: a row's elements in blocks of 32 neighbours share one
// scale byte b, the exponent field of a power of two (scale = 2^(b - 127)).
// With E the exponent of the block's largest magnitude:
//   int8:  b = max(E + 127 - 6, 1),   code = rne(x / scale) in [-127, 127]
//   e4m3:  b = max(E + 127 - 7, 10),  code = x / scale rounded to e4m3
// (E = 127: b = 248 and codes of at most 120 in e4m3, so that none stands for
// more than FP32 holds.)
// code * scale has at most 7 significant bits and an exponent inside BF16's
// normal range, so it is exact in BF16: reading a code back rounds nothing,
// and its product with a BF16 value is exact in FP32.  A block that holds an
// infinity or a NaN gets b = 255 and codes of zero, which read back as
// 0 * inf = NaN in all of its elements.
#pragma once

#include "common.h"

namespace smx {

constexpr int kAct8Block = 32;

// The scale byte of a block from the exponent field of its largest magnitude.
template <int FMT>
__device__ __forceinline__ int act8_scale_byte(int field) {
  if (field == 255) return 255;
  if constexpr (FMT == SMX_ACT8_INT8) return max(field - 6, 1);
  return max(field - 7, 10) + (field == 254 ? 1 : 0);
}

__device__ __forceinline__ float act8_scale(int b) { return __uint_as_float(static_cast<uint32_t>(b) << 23); }

// Four codes (one dword) to four values.
template <int FMT>
__device__ __forceinline__ void act8_unpack4(uint32_t w, float scale, float *v) {
  if constexpr (FMT == SMX_ACT8_INT8) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = static_cast<float>(static_cast<int8_t>(w >> (8 * k))) * scale;
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    v[0] = lo[0] * scale;
    v[1] = lo[1] * scale;
    v[2] = hi[0] * scale;
    v[3] = hi[1] * scale;
  }
}

// Four values to four codes; inv = 1 / scale.  int8: adding 1.5 * 2^23 leaves
// the value rounded to nearest even in the low byte, after the clamp.
template <int FMT>
__device__ __forceinline__ uint32_t act8_pack4(const float *v, float inv) {
  if constexpr (FMT == SMX_ACT8_INT8) {
    constexpr float kMagic = 12582912.f;
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      u[k] = __float_as_uint(__builtin_amdgcn_fmed3f(__builtin_fmaf(v[k], inv, kMagic), kMagic - 127.f, kMagic + 127.f));
    const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u);
    return __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu) | a;
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true));
  }
}

}  // namespace smx

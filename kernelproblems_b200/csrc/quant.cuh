// quant.cuh — 8-bit floating formats with one scale for a row or for a group
// of its values: scale rule, rounding, and the maxima that NaN passes through.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace frag {

// |f| as an unsigned word: ordered like the magnitude, with NaN above
// infinity, so an integer maximum keeps a NaN where fmaxf would drop it.
__device__ __forceinline__ uint32_t mag_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

template <bool E5M2>
__device__ __forceinline__ constexpr float fp8_max() { return E5M2 ? 57344.0f : 448.0f; }

// The scale of values whose largest magnitude is `most` (mag_bits), and the
// factor that q is made with, 1 / scale.  All zero: 1.  A scale is at least
// 2^-126, so that the factor stays finite.  E8M0: the power of two at or
// above (no value is then clipped), 255 for inf and NaN.
template <bool E5M2, bool E8M0>
__device__ __forceinline__ float quant_scale(uint32_t most, float& inv, uint8_t& byte) {
  float s = __uint_as_float(most) * (1.0f / fp8_max<E5M2>());
  // (not fmaxf: it would turn NaN into the bound)
  if (s < 1.17549435e-38f) s = 1.17549435e-38f;
  if (most == 0) s = 1.0f;
  if (E8M0) {
    const uint32_t e = min((__float_as_uint(s) + 0x7fffffu) >> 23, 255u);
    byte = static_cast<uint8_t>(e);
    s = e == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(e << 23);
    inv = e == 255u ? s : __uint_as_float((254u - e) << 23);
  } else {
    inv = 1.0f / s;
  }
  return s;
}

template <bool E5M2>
__device__ __forceinline__ uint16_t to_fp8x2(float lo, float hi) {
  return static_cast<uint16_t>(
      __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3));
}
template <bool E5M2>
__device__ __forceinline__ uint8_t to_fp8(float v) {
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3));
}

// Block-wide maximum of unsigned words, broadcast; one barrier, `slots` and
// `parity` as for block_sum.
__device__ __forceinline__ uint32_t block_umax(uint32_t v, uint32_t (*slots)[32], int parity) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nw = (blockDim.x + 31) >> 5;
  v = __reduce_max_sync(0xffffffffu, v);
  if (lane == 0) slots[parity][warp] = v;
  __syncthreads();
  uint32_t t = 0;
  for (int i = 0; i < nw; ++i) t = max(t, slots[parity][i]);
  return t;
}

struct QuantOut {
  uint8_t* q;
  void* scale;    // float or, with e8m0, bytes
  int64_t groups;  // scales of a row
};

template <bool E8M0>
__device__ __forceinline__ void store_scale(const QuantOut& o, int64_t i, float s, uint8_t byte) {
  if (E8M0) static_cast<uint8_t*>(o.scale)[i] = byte;
  else static_cast<float*>(o.scale)[i] = s;
}

}  // namespace frag

// quant.cuh — 8-bit floating formats with one scale for a row or for a group
// of its values: scale rule, rounding, and the maxima that NaN passes through.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace frag {

// Maximum that keeps a NaN (fmaxf would drop it), of magnitudes.
__device__ __forceinline__ float max_mag(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(fabsf(b)));
  return m;
}
// The same of a magnitude and two values, in one instruction.
__device__ __forceinline__ float max_mag2(float a, float2 b) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b.x), "f"(b.y));
  return m;
}
// Magnitudes in the order of their bits, with NaN (0x7fffffff) above infinity:
// an integer maximum over a warp.
__device__ __forceinline__ float warp_max_mag(float m) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
}

template <bool E5M2>
__device__ __forceinline__ constexpr float fp8_max() { return E5M2 ? 57344.0f : 448.0f; }

// The scale of values whose largest magnitude is `most`, and the factor that q
// is made with, 1 / scale (the hardware's reciprocal, 1 ulp: q moves only where
// y / scale is that near a tie).  All zero: 1.  A scale is at least 2^-126, so
// that the factor stays finite.  E8M0: the power of two at or above (no value
// is then clipped), 255 for inf and NaN.
template <bool E5M2, bool E8M0>
__device__ __forceinline__ float quant_scale(float most, float& inv, uint8_t& byte) {
  float s = most * (1.0f / fp8_max<E5M2>());
  // (not fmaxf: it would turn NaN into the bound)
  if (s < 1.17549435e-38f) s = most == 0.f ? 1.0f : 1.17549435e-38f;
  if (E8M0) {
    const uint32_t e = min((__float_as_uint(s) + 0x7fffffu) >> 23, 255u);
    byte = static_cast<uint8_t>(e);
    s = e == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(e << 23);
    inv = e == 255u ? s : __uint_as_float((254u - e) << 23);
  } else {
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
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

// Block-wide sum in a fixed order and maximum of magnitudes, broadcast; one
// barrier each, `slots` and `parity` as for block_sum.  The warps' results are
// combined by every warp's lanes: these rows hold 16 values a thread, and a
// loop over the warps was a third of the kernel's instructions.
__device__ __forceinline__ float block_sum_lanes(float v, float (*slots)[32], int parity) {
  const int lane = threadIdx.x & 31, nw = (blockDim.x + 31) >> 5;
  v = warp_sum(v);
  if (lane == 0) slots[parity][threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < nw ? slots[parity][lane] : 0.f);
}
__device__ __forceinline__ float block_max_mag(float m, float (*slots)[32], int parity) {
  const int lane = threadIdx.x & 31, nw = (blockDim.x + 31) >> 5;
  m = warp_max_mag(m);
  if (lane == 0) slots[parity][threadIdx.x >> 5] = m;
  __syncthreads();
  return warp_max_mag(lane < nw ? slots[parity][lane] : 0.f);
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

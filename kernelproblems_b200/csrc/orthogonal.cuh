// orthogonal.cuh — what the two forms of the Newton-Schulz chain share: its
// number formats, the caller's tensors, and swizzled shared memory.
#pragma once

#include <cuda_fp16.h>

#include "tc.cuh"

namespace frag {

constexpr float kXScale = 256.0f;   // X is kept times 2^8
constexpr float kAScale = 1024.0f;  // A and B times 2^10

// GRAM A = X X', POLY B = b A + c A A, STEP X <- a X + B X; the last step's
// STEP writes the result (LAST) or the weights (UPDATE) instead of X.
enum Mode { GRAM = 0, POLY = 1, STEP = 2, LAST = 3, UPDATE = 4 };

struct Elem {  // a tensor of bf16 or fp32 elements with strides
  void* p;
  int f32;
  int64_t sb, sr, sc;
};
__device__ __forceinline__ float load_elem(const Elem& e, int64_t i) {
  return e.f32 ? static_cast<const float*>(e.p)[i] : bf16_to_f(static_cast<const uint16_t*>(e.p)[i]);
}
__device__ __forceinline__ void store_elem(const Elem& e, int64_t i, float v) {
  if (e.f32) static_cast<float*>(e.p)[i] = v;
  else static_cast<uint16_t*>(e.p)[i] = f_to_bf16(v);
}

constexpr int kMaxSteps = 32;

__device__ __forceinline__ uint4 pack_h8(const float* f) {
  uint4 v;
  __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  return v;
}
__device__ __forceinline__ uint4 ld_shared(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void st_shared(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float ld_shared_f(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void st_shared_h(uint32_t a, __half v) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(a), "h"(__half_as_ushort(v)) : "memory");
}
// 16-byte unit u of row r of a chunk (128-byte rows under the 128-byte swizzle).
__device__ __forceinline__ uint32_t unit(uint32_t base, int r, int u) { return base + r * 128 + ((u ^ (r & 7)) << 4); }

// The matrices to be orthogonalised: a gradient, or with momentum
//   m' = mu m + (1 - mu) g,  u = mu m' + (1 - mu) g (nesterov) or m'
struct PrepP {
  Elem g, mom, mom_out;
  int has_mom, nesterov;
  float mu;
  int64_t rows, cols, ldx;  // of one matrix
  float eps;
  __half* hi;
  __half* lo;
  float* partials;  // [E, blocks]
  unsigned* counters;
  int count;  // of them, cleared for the chain of products
};

// The last step's result and what it updates: out = X, or keep par - rate X.
struct ResultP {
  int last;  // LAST or UPDATE
  Elem out, par;
  float keep, rate;
};

// Everything in one launch for matrices with a side of at most 128 that fit in
// a cluster's shared memory; -1 (nothing launched) when they do not.
int orthogonalise_small(const PrepP& prep, int64_t E, int steps, const float* co, const ResultP& res, cudaStream_t s);

}  // namespace frag

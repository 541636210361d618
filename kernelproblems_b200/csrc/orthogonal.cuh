// orthogonal.cuh — what the two forms of the Newton-Schulz chain share: its
// number formats, the caller's tensors, and swizzled shared memory.
#pragma once

#include <cuda_fp16.h>

#include "tc.cuh"

namespace frag {

constexpr float kXScale = 256.0f;   // X is kept times 2^8
constexpr float kAScale = 1024.0f;  // A and B times 2^10
// lo, where it is no operand of a product, times another 2^11: as large as hi
// at most, and clear of fp16's subnormals wherever hi is.
constexpr float kLoScale = 2048.0f;

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

// V neighbouring elements of a row (V = 8: one 16- or two 16-byte accesses).
template <int V>
__device__ __forceinline__ void load_elems(const Elem& e, int64_t i, float (&f)[V]) {
  if (V == 8 && e.f32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(e.p) + i));
    const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(e.p) + i) + 1);
    f[0] = a.x, f[1 % V] = a.y, f[2 % V] = a.z, f[3 % V] = a.w, f[4 % V] = b.x, f[5 % V] = b.y, f[6 % V] = b.z, f[7 % V] = b.w;
  } else if (V == 8) {
    const uint4 u = ld_cached(static_cast<const uint16_t*>(e.p) + i);
#pragma unroll
    for (int k = 0; k < V / 2; ++k) f[2 * k] = bf16lo(u4_word(u, k)), f[(2 * k + 1) % V] = bf16hi(u4_word(u, k));
  } else {
    f[0] = load_elem(e, i);
  }
}
template <int V>
__device__ __forceinline__ void store_elems(const Elem& e, int64_t i, const float (&f)[V]) {
  if (V == 8 && e.f32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(e.p) + i);
    o[0] = make_float4(f[0], f[1 % V], f[2 % V], f[3 % V]);
    o[1] = make_float4(f[4 % V], f[5 % V], f[6 % V], f[7 % V]);
  } else if (V == 8) {
    uint4 u;
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int k = 0; k < V / 2; ++k) w[k] = pack_bf16x2(f[2 * k], f[(2 * k + 1) % V]);
    st_global(static_cast<uint16_t*>(e.p) + i, u);
  } else {
    store_elem(e, i, f[0]);
  }
}

// The matrix to be orthogonalised at (r, c): the gradient or the momentum's
// look-ahead; m' in `m`.
template <int V>
__device__ __forceinline__ void prep_value(const PrepP& p, int64_t e, int64_t r, int64_t c, float (&u)[V],
                                           float (&m)[V]) {
  load_elems<V>(p.g, e * p.g.sb + r * p.g.sr + c * p.g.sc, u);
  if (!p.has_mom) return;
  load_elems<V>(p.mom, e * p.mom.sb + r * p.mom.sr + c * p.mom.sc, m);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const float g = (1.0f - p.mu) * u[k];
    m[k] = p.mu * m[k] + g;
    u[k] = p.nesterov ? p.mu * m[k] + g : m[k];
  }
}

// Rows of whole 8-element chunks, aligned for 16-byte accesses.
inline bool chunked(const Elem& e, int64_t E, int64_t rows, int64_t cols) {
  return cols % 8 == 0 && e.sc == 1 && (rows == 1 || e.sr % 8 == 0) && (E == 1 || e.sb % 8 == 0) && aligned16(e.p);
}

// The last step's result and what it updates: out = X, or keep par - rate X.
struct ResultP {
  int last;  // LAST or UPDATE
  Elem out, par;
  float keep, rate;
};

// Everything in one launch, without a workspace, for matrices with a side of at
// most 128 that fit in a cluster's shared memory: whether m x n are such.
bool small_takes(int64_t m, int64_t n);
int orthogonalise_small(const PrepP& prep, int64_t E, int steps, const float* co, const ResultP& res, cudaStream_t s);

}  // namespace frag

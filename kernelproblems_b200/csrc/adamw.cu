// adamw.cu — one AdamW step over many tensors in one launch, with the moments
// in 32 bits or in 8.
//
//   g' = scale g,  m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2
//   p' = (1 - lr wd) p - lr / c1 m' / (sqrt(v') / sqrt(c2) + eps),  c = 1 - b^t
//
// 8 bits: m and r = sqrt(v) as E4M3 numbers times a scale for each 128 values,
// max / 448.  The root is held because its range is half of v's in exponents:
// E4M3 spans 2^18, so v 2^36.  What is not zero of r stays at least the smallest
// E4M3 number: a root that became 0 beside a first moment that did not would
// make the next step m / eps.  The step itself uses the unrounded moments.
//
// Bound: HBM.  28 bytes a value in 32 bits (30 with a bf16 copy), 10.1 for a bf16
// tensor with states in 8.  Everything is read and written once, nothing is kept on
// chip, so the kernel only has to keep enough loads in flight: eight
// neighbouring values a thread, 16-byte accesses, all of a chunk's loads before its
// arithmetic.
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "quant.cuh"
#include "tensor_list.cuh"

namespace frag {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 128;                  // values of a scale
constexpr int64_t kChunk = 2 * 8 * kThreads;  // values

struct Entry {
  void* p;
  const void* g;
  uint16_t* copy;
  int64_t numel;
  int64_t state;  // first value in the flat states, a multiple of kGroup
  float lr_scale, decay;
};

template <int CAP>
struct List {
  Entry t[CAP];
  uint32_t first[CAP + 1];
  uint8_t kind[CAP];  // bit 0: fp32 p, 1: fp32 g, 2: 16-byte aligned
  int count;
};

struct Step {
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  const float* grad_scale;  // or nullptr
  const float* lr_dev;      // or nullptr: lr
  const int64_t* step_dev;  // or nullptr: c1, root
  double lr, beta1, beta2;
  double log1, log2;  // of the betas
  double c1, root;    // 1 - beta1^step, 1 / sqrt(1 - beta2^step)
  float eps;
};

// What all values of a tensor share.
struct Factors {
  float b1, a1, b2, a2;  // beta, 1 - beta
  float keep;            // 1 - lr wd
  float rate;            // lr / c1
  float root;            // 1 / sqrt(c2)
  float eps;
  float g;               // gradient's scale
};

// The products and sums of the moments are rounded one by one: fused, they would
// differ in the last bit from the same formula elsewhere, and the 8 bits
// that follow would then round differently at ties.
__device__ __forceinline__ void update(float p, float g, float& m, float& v, float& r, float& out,
                                       const Factors& f) {
  g = __fmul_rn(g, f.g);
  m = __fadd_rn(__fmul_rn(f.b1, m), __fmul_rn(f.a1, g));
  v = __fadd_rn(__fmul_rn(f.b2, v), __fmul_rn(__fmul_rn(f.a2, g), g));
  r = __fsqrt_rn(v);
  // (the quotient's 2 ulp are 2^-22 of the step)
  out = fmaf(p, f.keep, -__fdividef(f.rate * m, fmaf(r, f.root, f.eps)));
}

__device__ __forceinline__ float e4m3_to_f(uint8_t b) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(b, __NV_E4M3);
  return __half2float(__half(h));
}
__device__ __forceinline__ float2 e4m3x2_to_f2(uint16_t b) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(b, __NV_E4M3);
  return __half22float2(__half2(h));
}

// A group's scale, and 1 / scale.  All zero: 1.
__device__ __forceinline__ float state_scale(float most, float& inv) {
  float s = most * (1.0f / 448.0f);
  if (s < 1.17549435e-38f) s = most == 0.f ? 1.0f : 1.17549435e-38f;
  inv = __frcp_rn(s);
  return s;
}

// A root's multiple of the scale: what is not zero stays so.
__device__ __forceinline__ float at_least_smallest(float r, float q) { return r > 0.f ? fmaxf(q, 0x1p-9f) : q; }

template <class T>
__device__ __forceinline__ float value(const T* p) {
  return sizeof(T) == 2 ? bf16_to_f(*reinterpret_cast<const uint16_t*>(p)) : *reinterpret_cast<const float*>(p);
}
template <class T>
__device__ __forceinline__ void set_value(T* p, float f) {
  if (sizeof(T) == 2) *reinterpret_cast<uint16_t*>(p) = f_to_bf16(f);
  else *reinterpret_cast<float*>(p) = f;
}

// Eight neighbouring values from a 16-byte boundary, n of them (any n >= 8: all).
// RO: nothing writes them in this launch.
template <bool RO, class T>
__device__ __forceinline__ void load8(const T* p, int64_t n, float (&f)[8]) {
  if (n >= 8) {
    if (sizeof(T) == 2) {
      unpack8(RO ? ld_stream(p) : ld_plain(p), f);
    } else {
      float4 a, b;
      if (RO) {
        a = ld_stream_f4(p);
        b = ld_stream_f4(p + 4);
      } else {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
      }
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? value(p + i) : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int64_t n, const float (&f)[8]) {
  if (n >= 8) {
    if (sizeof(T) == 2) {
      st_global(p, pack8(f));
    } else {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) set_value(p + i, f[i]);
  }
}

// States of a tensor: whole groups.
__device__ __forceinline__ int64_t held_by(const Entry& e) { return (e.numel + kGroup - 1) / kGroup * kGroup; }

// A chunk of a tensor whose pointers are 16-byte aligned: thread t has eight
// neighbouring values, a group is 16 neighbouring lanes.  The states behind a
// tensor's end belong to its last group and stay zero (their p and g read as
// zero), so they are moved whole.
template <bool EIGHT, class P, class G>
__device__ __forceinline__ void chunk_aligned(const Entry& e, const Step& s, const Factors& f, int64_t from) {
#pragma unroll
  for (int k = 0; k < kChunk / (8 * kThreads); ++k) {
    const int64_t at = from + (k * kThreads + threadIdx.x) * 8;
    const int64_t left = e.numel - at;
    if (left + (threadIdx.x & 31) * 8 <= 0) return;  // the whole warp is behind the end
    const int64_t st = e.state + at;
    P* p = static_cast<P*>(e.p) + at;
    float pv[8], gv[8], m[8], v[8], r[8];
    const bool in_group = at < held_by(e);
    load8<false>(p, left, pv);
    load8<true>(static_cast<const G*>(e.g) + at, left, gv);
    float ms = 0.f, vs = 0.f;
    if (EIGHT) {
      uint2 mq = make_uint2(0, 0), vq = make_uint2(0, 0);
      if (in_group) {
        mq = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(s.m) + st);
        vq = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(s.v) + st);
        ms = s.m_scale[st / kGroup];
        vs = s.v_scale[st / kGroup];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = e4m3x2_to_f2(static_cast<uint16_t>((i < 2 ? mq.x : mq.y) >> (16 * (i & 1))));
        const float2 b = e4m3x2_to_f2(static_cast<uint16_t>((i < 2 ? vq.x : vq.y) >> (16 * (i & 1))));
        m[2 * i] = __fmul_rn(a.x, ms);
        m[2 * i + 1] = __fmul_rn(a.y, ms);
        const float x = __fmul_rn(b.x, vs), y = __fmul_rn(b.y, vs);
        v[2 * i] = __fmul_rn(x, x);
        v[2 * i + 1] = __fmul_rn(y, y);
      }
    } else {
      load8<false>(static_cast<const float*>(s.m) + st, in_group ? 8 : 0, m);
      load8<false>(static_cast<const float*>(s.v) + st, in_group ? 8 : 0, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) update(pv[i], gv[i], m[i], v[i], r[i], pv[i], f);
    store8(p, left, pv);
    if (e.copy) store8(e.copy + at, left, pv);
    if (EIGHT) {
      float mm = 0.f, rm = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mm = max_mag(mm, m[i]);
        rm = max_mag(rm, r[i]);
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        mm = max_mag(mm, __shfl_xor_sync(0xffffffffu, mm, o));
        rm = max_mag(rm, __shfl_xor_sync(0xffffffffu, rm, o));
      }
      float mi, ri;
      ms = state_scale(mm, mi);
      vs = state_scale(rm, ri);
      if (in_group) {
        uint32_t a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = to_fp8x2<false>(__fmul_rn(m[2 * i], mi), __fmul_rn(m[2 * i + 1], mi));
          b[i] = to_fp8x2<false>(at_least_smallest(r[2 * i], __fmul_rn(r[2 * i], ri)),
                                 at_least_smallest(r[2 * i + 1], __fmul_rn(r[2 * i + 1], ri)));
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(s.m) + st) = make_uint2(a[0] | a[1] << 16, a[2] | a[3] << 16);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(s.v) + st) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
        if ((threadIdx.x & 15) == 0) {
          s.m_scale[st / kGroup] = ms;
          s.v_scale[st / kGroup] = vs;
        }
      }
    } else if (in_group) {
      store8(static_cast<float*>(s.m) + st, 8, m);
      store8(static_cast<float*>(s.v) + st, 8, v);
    }
  }
}

// The same where some pointer is not aligned: lane l of a warp has every 32nd
// of 256 values, single accesses that a warp makes to neighbouring addresses; a
// group is four of its rows.
template <bool EIGHT, class P, class G>
__device__ __forceinline__ void chunk_any(const Entry& e, const Step& s, const Factors& f, int64_t from) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
  for (int k = 0; k < kChunk / (8 * kThreads); ++k) {
    const int64_t at = from + (k * (kThreads / 32) + warp) * 256 + lane;
    if (at - lane >= e.numel) return;
    const int64_t st = e.state + at;
    P* p = static_cast<P*>(e.p) + at;
    const G* g = static_cast<const G*>(e.g) + at;
    const int64_t held = held_by(e);
    float pv[8], gv[8], m[8], v[8], r[8];
    float ms[2] = {0.f, 0.f}, vs[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = at + 32 * i < e.numel, st_in = at + 32 * i < held;
      pv[i] = in ? value(p + 32 * i) : 0.f;
      gv[i] = in ? value(g + 32 * i) : 0.f;
      if (EIGHT) {
        if (i % 4 == 0 && st_in) {
          ms[i / 4] = s.m_scale[(st + 32 * i) / kGroup];
          vs[i / 4] = s.v_scale[(st + 32 * i) / kGroup];
        }
        m[i] = st_in ? e4m3_to_f(static_cast<const uint8_t*>(s.m)[st + 32 * i]) : 0.f;
        v[i] = st_in ? e4m3_to_f(static_cast<const uint8_t*>(s.v)[st + 32 * i]) : 0.f;
      } else {
        m[i] = st_in ? static_cast<const float*>(s.m)[st + 32 * i] : 0.f;
        v[i] = st_in ? static_cast<const float*>(s.v)[st + 32 * i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (EIGHT) {
        m[i] = __fmul_rn(m[i], ms[i / 4]);
        v[i] = __fmul_rn(v[i], vs[i / 4]);
        v[i] = __fmul_rn(v[i], v[i]);
      }
      update(pv[i], gv[i], m[i], v[i], r[i], pv[i], f);
      if (at + 32 * i < e.numel) {
        set_value(p + 32 * i, pv[i]);
        if (e.copy) set_value(e.copy + at + 32 * i, pv[i]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mi = 0.f, ri = 0.f;
      if (EIGHT) {
        float mm = 0.f, rm = 0.f;
#pragma unroll
        for (int i = 4 * h; i < 4 * h + 4; ++i) {
          mm = max_mag(mm, m[i]);
          rm = max_mag(rm, r[i]);
        }
        ms[h] = state_scale(warp_max_mag(mm), mi);
        vs[h] = state_scale(warp_max_mag(rm), ri);
        if (lane == 0 && at + 128 * h < held) {
          s.m_scale[(st + 128 * h) / kGroup] = ms[h];
          s.v_scale[(st + 128 * h) / kGroup] = vs[h];
        }
      }
#pragma unroll
      for (int i = 4 * h; i < 4 * h + 4; ++i) {
        if (at + 32 * i >= held) continue;
        if (EIGHT) {
          static_cast<uint8_t*>(s.m)[st + 32 * i] = to_fp8<false>(__fmul_rn(m[i], mi));
          static_cast<uint8_t*>(s.v)[st + 32 * i] = to_fp8<false>(at_least_smallest(r[i], __fmul_rn(r[i], ri)));
        } else {
          static_cast<float*>(s.m)[st + 32 * i] = m[i];
          static_cast<float*>(s.v)[st + 32 * i] = v[i];
        }
      }
    }
  }
}

template <bool EIGHT, class P, class G>
__device__ __forceinline__ void chunk(bool aligned, const Entry& e, const Step& s, const Factors& f, int64_t from) {
  if (aligned) chunk_aligned<EIGHT, P, G>(e, s, f, from);
  else chunk_any<EIGHT, P, G>(e, s, f, from);
}

template <int CAP, bool EIGHT>
__global__ void __launch_bounds__(kThreads) adamw(const __grid_constant__ List<CAP> L, const __grid_constant__ Step s) {
  const int i = find_tensor(L.first, L.count, blockIdx.x);
  const Entry& e = L.t[i];
  const double lr = s.lr_dev ? static_cast<double>(*s.lr_dev) : s.lr;
  const float scale = s.grad_scale ? *s.grad_scale : 1.0f;
  double c1 = s.c1, root = s.root;
  if (s.step_dev) {
    __shared__ double c[2];
    const int64_t step = *s.step_dev;
    if (step < 1) return;
    if (threadIdx.x == 0) {
      c[0] = -expm1(static_cast<double>(step) * s.log1);
      c[1] = 1.0 / sqrt(-expm1(static_cast<double>(step) * s.log2));
    }
    __syncthreads();
    c1 = c[0];
    root = c[1];
  }
  if (!isfinite(scale) || !isfinite(lr)) return;
  Factors f;
  f.b1 = static_cast<float>(s.beta1);
  f.a1 = static_cast<float>(1.0 - s.beta1);
  f.b2 = static_cast<float>(s.beta2);
  f.a2 = static_cast<float>(1.0 - s.beta2);
  f.keep = static_cast<float>(1.0 - lr * static_cast<double>(e.lr_scale) * static_cast<double>(e.decay));
  f.rate = static_cast<float>(lr * static_cast<double>(e.lr_scale) / c1);
  f.root = static_cast<float>(root);
  f.eps = s.eps;
  f.g = scale;
  const int64_t from = static_cast<int64_t>(blockIdx.x - L.first[i]) * kChunk;
  const bool aligned = L.kind[i] & 4;
  switch (L.kind[i] & 3) {
    case 0: chunk<EIGHT, uint16_t, uint16_t>(aligned, e, s, f, from); break;
    case 1: chunk<EIGHT, float, uint16_t>(aligned, e, s, f, from); break;
    case 2: chunk<EIGHT, uint16_t, float>(aligned, e, s, f, from); break;
    default: chunk<EIGHT, float, float>(aligned, e, s, f, from);
  }
}

template <int CAP, bool EIGHT>
int launch(const frag_adamw_tensor* t, const void* const* grads, const int32_t* grad_dtypes, int count,
           const Step& step, cudaStream_t s) {
  List<CAP> L;
  int64_t c = 0;
  int n = 0;
  for (int i = 0; i < count; ++i) {
    if (!grads[i] || t[i].numel == 0) continue;
    const bool aligned = aligned16(t[i].param) && aligned16(grads[i]) && (!t[i].copy || aligned16(t[i].copy));
    L.t[n] = {t[i].param, grads[i], static_cast<uint16_t*>(t[i].copy), t[i].numel, t[i].state_offset,
              t[i].lr_scale, t[i].weight_decay};
    L.kind[n] = (t[i].param_dtype == FRAG_DT_F32 ? 1 : 0) | (grad_dtypes[i] == FRAG_DT_F32 ? 2 : 0) | (aligned ? 4 : 0);
    L.first[n++] = static_cast<uint32_t>(c);
    c += ceil_div(t[i].numel, kChunk);
    if (c > 0x7fffffffLL) return FRAG_ERR_SHAPE;
  }
  L.first[n] = static_cast<uint32_t>(c);
  L.count = n;
  if (c == 0) return FRAG_OK;
  adamw<CAP, EIGHT><<<dim3(static_cast<unsigned>(c)), kThreads, 0, s>>>(L, step);
  return check_launch();
}

template <bool EIGHT>
int launch_lists(const frag_adamw_tensor* t, const void* const* grads, const int32_t* grad_dtypes, int64_t count,
                 const Step& step, cudaStream_t s) {
  for (int64_t i = 0; i < count; i += kListLarge) {
    const int n = static_cast<int>(std::min<int64_t>(kListLarge, count - i));
    const int st = n <= kListSmall ? launch<kListSmall, EIGHT>(t + i, grads + i, grad_dtypes + i, n, step, s)
                                   : launch<kListLarge, EIGHT>(t + i, grads + i, grad_dtypes + i, n, step, s);
    if (st != FRAG_OK) return st;
  }
  return FRAG_OK;
}

}  // namespace
}  // namespace frag

using namespace frag;

extern "C" {

int frag_adamw_update(const frag_adamw_tensor* tensors, const void* const* grads, const int32_t* grad_dtypes,
                      int64_t count, void* exp_avg, void* exp_avg_sq, float* exp_avg_scale, float* exp_avg_sq_scale,
                      double lr, const float* lr_device, double beta1, double beta2, double eps, int64_t step,
                      const int64_t* step_device, const float* grad_scale, frag_stream_t stream) {
  if (count < 0 || (count > 0 && (!tensors || !grads || !grad_dtypes))) return FRAG_ERR_INVALID_ARG;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return FRAG_ERR_INVALID_ARG;
  if (!std::isfinite(eps) || eps < 0.0) return FRAG_ERR_INVALID_ARG;
  if (!lr_device && !std::isfinite(lr)) return FRAG_ERR_INVALID_ARG;
  if (!step_device && step < 1) return FRAG_ERR_INVALID_ARG;
  const bool eight = exp_avg_scale != nullptr;
  if (eight != (exp_avg_sq_scale != nullptr)) return FRAG_ERR_INVALID_ARG;
  int64_t values = 0;
  for (int64_t i = 0; i < count; ++i) {
    const frag_adamw_tensor& t = tensors[i];
    if (t.numel < 0 || t.state_offset < 0 || (t.numel > 0 && !t.param)) return FRAG_ERR_INVALID_ARG;
    if ((t.param_dtype != FRAG_DT_BF16 && t.param_dtype != FRAG_DT_F32) ||
        (grad_dtypes[i] != FRAG_DT_BF16 && grad_dtypes[i] != FRAG_DT_F32))
      return FRAG_ERR_INVALID_ARG;
    if (!std::isfinite(t.lr_scale) || !std::isfinite(t.weight_decay)) return FRAG_ERR_INVALID_ARG;
    if (t.state_offset % kGroup) return FRAG_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(t.param) % (t.param_dtype == FRAG_DT_F32 ? 4 : 2) ||
        reinterpret_cast<uintptr_t>(grads[i]) % (grad_dtypes[i] == FRAG_DT_F32 ? 4 : 2) ||
        reinterpret_cast<uintptr_t>(t.copy) % 2)
      return FRAG_ERR_ALIGN;
    if (t.numel > (1LL << 40)) return FRAG_ERR_SHAPE;
    values += t.numel;
  }
  if (values == 0) return FRAG_OK;
  if (!exp_avg || !exp_avg_sq) return FRAG_ERR_INVALID_ARG;
  if (!aligned16(exp_avg) || !aligned16(exp_avg_sq)) return FRAG_ERR_ALIGN;
  Step p = {exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, grad_scale, lr_device, step_device, lr, beta1, beta2,
            std::log(beta1), std::log(beta2), 1.0, 1.0, static_cast<float>(eps)};
  if (!step_device) {
    p.c1 = -std::expm1(static_cast<double>(step) * p.log1);
    p.root = 1.0 / std::sqrt(-std::expm1(static_cast<double>(step) * p.log2));
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return eight ? launch_lists<true>(tensors, grads, grad_dtypes, count, p, s)
               : launch_lists<false>(tensors, grads, grad_dtypes, count, p, s);
}

}  // extern "C"

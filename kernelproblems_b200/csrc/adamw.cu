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
// make the next step m / eps.  The step itself uses the unrounded moments.  Rounding to
// nearest holds a code until a step moves it by half of E4M3's (3 to 6 percent), so what
// decays more slowly than its group stays behind: from beta2 of about 0.98 and beta1
// of 0.95 on (the entry point's documentation has figures).
//
// Bound: HBM.  28 bytes a value in 32 bits (30 with a bf16 copy), 10.1 for a bf16
// tensor with states in 8.  Everything is read and written once, nothing is kept on
// chip, so the kernel only has to keep enough loads in flight.  218 million values
// in 9 tensors: fp32 throughout 888 us (6.9 TB/s, above a copy's 6.5 as more is read
// than written), with a bf16 copy 960; fp32 parameters, bf16 gradients and copies,
// states in 8 bits 523; bf16 with states in 8 bits 395 (5.6 TB/s), where four fifths
// of the issue slots are busy (416 in a run of 4000 calls, of any input).  Off 16-byte boundaries 884, 627 and 519: shifts and
// the warps' ends; loads and stores of single values took 900, 746 and 634.
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "quant.cuh"
#include "tensor_list.cuh"

namespace frag {
namespace {

// A block takes one chunk, a thread eight values of it: twelve blocks an SM (40
// registers) have 12288 values in flight, 72 KB of bf16 parameters, gradients and 8-bit
// states.  218 million bf16 values with states in 8 bits: 395 us; with ten blocks 510.  (Before the roots'
// rounding 372; blocks of 256 threads 379, of 512 463; two chunks a thread 588 at four
// blocks of 256 an SM, 446 one.)  States in 32 bits: nine blocks, where twelve spill
// off 16-byte boundaries (1003 us against 884, at them 887 both).
constexpr int kThreads = 128;
constexpr int resident(bool eight) { return eight ? 12 : 9; }
constexpr int kGroup = 128;                // values of a scale
constexpr int64_t kChunk = 8 * kThreads;  // values

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
  double log1, log2;        // of the betas
  float lr;
  float b1, a1, b2, a2;     // beta, 1 - beta
  float c1, root;           // 1 / (1 - beta1^step), 1 / sqrt(1 - beta2^step)
  float eps;
};

// What all values of a tensor share.
struct Factors {
  float keep;  // 1 - lr wd
  float rate;  // lr / (1 - beta1^step)
  float root;  // 1 / sqrt(1 - beta2^step)
  float g;     // the gradient's scale
};

__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// A product that no sum is contracted with (which happens to __fmul2_rn's).
__device__ __forceinline__ float2 product(float2 a, float2 b) { return __ffma2_rn(a, b, twice(0.f)); }
// m' and v', each operation rounded by itself, as elementary 32-bit operations have
// them, and roots rounded to nearest below: states in 8 bits are then those of the
// formula in 32 bits to the last bit.  (Contracted, one of 400000 codes is its
// neighbour, a sixteenth off, and where |m| / r is large that shows in the next step.)
__device__ __forceinline__ float2 first_moment(float2 m, float2 g, const Step& s) {
  return __fadd2_rn(product(m, twice(s.b1)), product(g, twice(s.a1)));
}
__device__ __forceinline__ float2 second_moment(float2 v, float2 g, const Step& s) {
  return __fadd2_rn(product(v, twice(s.b2)), product(product(g, twice(s.a2)), g));
}
__device__ __forceinline__ float root_of(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float least_of(float a, float b, float c) {
  float m;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// Square roots rounded to nearest, by a step of Newton's iteration whose residual is
// exact in an FMA (P. Markstein, Computation of elementary functions on the IBM RISC
// System/6000 processor, 1990): s = v y of an approximate y near 1 / sqrt(v), then
// s + (v - s^2) y / 2.  An approximate y does not make that exact by argument, so it
// was compared with the library's root on a B200: none of the 1761607681 numbers from
// 2^-90 to 2^120 differs.  A thread with values outside (what underflows, infinity,
// single zeros; not all zeros, as of rows that no gradient came by) takes the
// library's for all.  218 million bf16 values: 395 us, with the library's for all
// 406, with an approximation's last bit 375; a decoder layer's gradients 434 and 469.
__device__ __forceinline__ void roots(const float2 (&v)[4], float2 (&r)[4]) {
  float least = v[0].x, most = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    least = least_of(least, v[i].x, v[i].y);
    most = max_mag2(most, v[i]);
  }
  if ((least >= 0x1p-90f && most <= 0x1p+120f) || most == 0.f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 y;
      const float2 a = __fadd2_rn(v[i], twice(0x1p-120f));  // (v itself, but of zeros)
      asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(a.x));
      asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(a.y));
      const float2 s = __fmul2_rn(v[i], y);
      r[i] = __ffma2_rn(__ffma2_rn(make_float2(-s.x, -s.y), s, v[i]), __fmul2_rn(y, twice(0.5f)), s);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = make_float2(__fsqrt_rn(v[i].x), __fsqrt_rn(v[i].y));
  }
}
__device__ __forceinline__ float inverse(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// p' from m' and r = sqrt(v').  Root, reciprocal and product are off by some 2^-22
// of the step, which is small beside p.
__device__ __forceinline__ float2 parameter(float2 p, float2 m, float2 r, const Factors& f, const Step& s) {
  const float2 d = __ffma2_rn(r, twice(f.root), twice(s.eps));
  const float2 u = __fmul2_rn(__fmul2_rn(m, twice(-f.rate)), make_float2(inverse(d.x), inverse(d.y)));
  return __ffma2_rn(p, twice(f.keep), u);
}

__device__ __forceinline__ float2 e4m3x2_to_f2(uint32_t b) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(b), __NV_E4M3);
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
__device__ __forceinline__ float& part(float2& v, int i) { return i ? v.y : v.x; }

// The first W of W + 4 words from `bytes` on (even, below 16; the same for a warp).
template <int W>
__device__ __forceinline__ void shift_words(uint32_t (&w)[W + 4], int bytes) {
  const int bits = 8 * (bytes & 2);
  auto from = [&](int q) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = __funnelshift_r(w[i + q], w[i + q + 1], bits);
  };
  switch (bytes >> 2) {
    case 0: from(0); break;
    case 1: from(1); break;
    case 2: from(2); break;
    default: from(3);
  }
}

// Eight neighbouring values as they lie in memory.  ANY: from any address, all else
// from a 16-byte boundary.
template <class T, bool ANY>
struct Eight {
  static constexpr int E = 16 / sizeof(T), K = 8 / E, W = 4 * K;  // values of a 16-byte chunk, chunks, words
  uint4 raw[K], last;  // ANY: `last`, the chunk behind
  int shift;           // ANY: bytes that raw begins before the values

  static __device__ __forceinline__ int bytes_off(const T* p) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15u);
  }

  // Asks for n of them (8 or more: all); settle() then makes them the values.  RO:
  // nothing writes them in this launch.  ANY: the chunks that they lie in, whole,
  // where those are the tensor's own (what neighbours write meanwhile is shifted
  // out); `first`: the tensor's first values.
  template <bool RO>
  __device__ __forceinline__ void load(const T* p, int n, bool first) {
    auto chunk = [](const T* a) {
      return RO ? ld_stream(reinterpret_cast<const uint4*>(a)) : ld_plain(reinterpret_cast<const uint4*>(a));
    };
    shift = ANY ? bytes_off(p) : 0;
    const int off = shift / static_cast<int>(sizeof(T));
    if (!shift ? n >= 8 : !first && n >= 8 + E - off) {
#pragma unroll
      for (int k = 0; k < K; ++k) raw[k] = chunk(p - off + k * E);
      if (ANY && shift) last = chunk(p - off + 8);
    } else {
      float2 f[4];
#pragma unroll
      for (int i = 0; i < 8; ++i) part(f[i / 2], i & 1) = i < n ? value(p + i) : 0.f;
      set(f);
      shift = 0;
    }
  }
  __device__ __forceinline__ void settle() {
    if constexpr (ANY) {
      if (!shift) return;
      uint32_t w[W + 4];
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = u4_word(raw[i / 4], i & 3);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[W + i] = u4_word(last, i);
      shift_words<W>(w, shift);
#pragma unroll
      for (int k = 0; k < K; ++k) raw[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 2) return bf16x2_to_f2(u4_word(raw[0], i));
    else return make_float2(__uint_as_float(u4_word(raw[i / 2], 2 * (i & 1))),
                            __uint_as_float(u4_word(raw[i / 2], 2 * (i & 1) + 1)));
  }
  __device__ __forceinline__ void set(const float2 (&f)[4]) {
    if constexpr (sizeof(T) == 2) {
      raw[0] = make_uint4(f2_to_bf16x2(f[0]), f2_to_bf16x2(f[1]), f2_to_bf16x2(f[2]), f2_to_bf16x2(f[3]));
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        raw[q] = make_uint4(__float_as_uint(f[2 * q].x), __float_as_uint(f[2 * q].y), __float_as_uint(f[2 * q + 1].x),
                            __float_as_uint(f[2 * q + 1].y));
    }
  }
  // n of them; by whole warps, whose lanes' values lie one behind the other.  ANY: a
  // chunk is written whole by the lane that has its last value, with the lane before's
  // part of it; value by value where it reaches out of the warp's values.
  __device__ __forceinline__ void store(T* p, int n) const {
    const int bytes = ANY ? bytes_off(p) : 0;
    if (!ANY || !bytes) {
      if (n >= 8) {
#pragma unroll
        for (int k = 0; k < K; ++k) st_global(reinterpret_cast<uint4*>(p) + k, raw[k]);
      } else {
        store_some(p, n, 0xff);
      }
      return;
    }
    const int off = bytes / static_cast<int>(sizeof(T)), lane = threadIdx.x & 31;
    uint32_t w[W + 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __shfl_up_sync(0xffffffffu, u4_word(raw[K - 1], i), 1);
#pragma unroll
    for (int i = 0; i < W; ++i) w[4 + i] = u4_word(raw[i / 4], i & 3);
    shift_words<W>(w, 16 - bytes);
    uint32_t single = 0;  // the values of chunks that are not written whole
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      // chunk k: values k E - off to (k + 1) E - off - 1; the last is the next lane's first
      const bool whole = n >= (k + 1) * E - off && (k > 0 || lane > 0) && (k < K || lane < 31);
      const int i = 4 * k % W;
      if (whole && k < K) st_global(reinterpret_cast<uint4*>(p - off) + k, make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]));
      if (!whole) single |= ((1u << E) - 1) << (k * E) >> off;
    }
    store_some(p, n, single);
  }

 private:
  // Those of the first n (or 8) whose bit is set, one by one.
  __device__ __forceinline__ void store_some(T* p, int n, uint32_t which) const {
    which &= n >= 8 ? 0xffu : (1u << max(n, 0)) - 1;
    if (!which) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(which >> i & 1)) continue;
      const uint32_t word = u4_word(raw[i / E], i % E * static_cast<int>(sizeof(T)) / 4);
      if constexpr (sizeof(T) == 2) p[i] = static_cast<uint16_t>(i & 1 ? word >> 16 : word);
      else p[i] = __uint_as_float(word);
    }
  }
};

// The scales of a group, 16 neighbouring lanes, by its lanes' largest first moments
// and roots: 1 / scale of both, and the scale that the lane is for.  After one exchange
// lanes without bit 3 go on with the moments and the others with the roots, so that
// both take one shuffle a level and one division.
__device__ __forceinline__ float group_scales(float m, float r, float& m_inv, float& r_inv) {
  const bool second = threadIdx.x & 8;
  float v = max_mag(second ? r : m, __shfl_xor_sync(0xffffffffu, second ? m : r, 8));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v = max_mag(v, __shfl_xor_sync(0xffffffffu, v, o));
  float inv;
  const float scale = state_scale(v, inv), other = __shfl_xor_sync(0xffffffffu, inv, 8);
  m_inv = second ? other : inv;
  r_inv = second ? inv : other;
  return scale;
}

// A chunk of a tensor: thread t has eight neighbouring values, a group is 16
// neighbouring lanes.  ANY: parameters, gradients or copies off 16-byte boundaries
// (states never are).  The states behind a tensor's end belong to its last group and
// stay zero (their p and g read as zero), so they are moved whole.  `n`: the chunk's
// values.
template <bool EIGHT, bool ANY, class P, class G>
__device__ __forceinline__ void chunk(const Entry& e, const Step& s, const Factors& f, int64_t from, int n) {
  P* p0 = static_cast<P*>(e.p) + from;
  const G* g0 = static_cast<const G*>(e.g) + from;
  const int64_t st = e.state + from;
  const int held = (n + kGroup - 1) / kGroup * kGroup;
  const int at = threadIdx.x * 8;
  if (at - (threadIdx.x & 31) * 8 >= n) return;  // the whole warp
  const bool in = at < held;
  Eight<P, ANY> p;
  Eight<G, ANY> g;
  p.template load<false>(p0 + at, n - at, from + at == 0);
  g.template load<true>(g0 + at, n - at, from + at == 0);
  float2 pv[4];
  if constexpr (EIGHT) {
    uint8_t *m0 = static_cast<uint8_t*>(s.m) + st, *v0 = static_cast<uint8_t*>(s.v) + st;
    float *ms = s.m_scale + st / kGroup, *vs = s.v_scale + st / kGroup;
    uint2 mq = make_uint2(0, 0), vq = make_uint2(0, 0);
    float mb = 0.f, vb = 0.f;
    if (in) {
      mq = *reinterpret_cast<const uint2*>(m0 + at);
      vq = *reinterpret_cast<const uint2*>(v0 + at);
      mb = ms[at / kGroup];
      vb = vs[at / kGroup];
    }
    p.settle();
    g.settle();
    float2 m[4], v[4], r[4];
    float mm = 0.f, rm = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 gi = __fmul2_rn(g.pair(i), twice(f.g));
      const float2 mo = e4m3x2_to_f2((i < 2 ? mq.x : mq.y) >> (16 * (i & 1)) & 0xffff);
      const float2 ro = product(e4m3x2_to_f2((i < 2 ? vq.x : vq.y) >> (16 * (i & 1)) & 0xffff), twice(vb));
      m[i] = first_moment(product(mo, twice(mb)), gi, s);
      v[i] = second_moment(product(ro, ro), gi, s);
      mm = max_mag2(mm, m[i]);
    }
    roots(v, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pv[i] = parameter(p.pair(i), m[i], r[i], f, s);
      rm = max_mag2(rm, r[i]);
    }
    float mi, ri;
    const float scale = group_scales(mm, rm, mi, ri);
    if (in) {
      uint32_t a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = __fmul2_rn(m[i], twice(mi)), y = __fmul2_rn(r[i], twice(ri));
        a[i] = to_fp8x2<false>(x.x, x.y);
        b[i] = to_fp8x2<false>(at_least_smallest(r[i].x, y.x), at_least_smallest(r[i].y, y.y));
      }
      *reinterpret_cast<uint2*>(m0 + at) = make_uint2(a[0] | a[1] << 16, a[2] | a[3] << 16);
      *reinterpret_cast<uint2*>(v0 + at) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
      if ((threadIdx.x & 7) == 0) (threadIdx.x & 8 ? vs : ms)[at / kGroup] = scale;
    }
  } else {
    float *m0 = static_cast<float*>(s.m) + st + at, *v0 = static_cast<float*>(s.v) + st + at;
    Eight<float, false> m, v;
    m.template load<false>(m0, in ? 8 : 0, false);
    v.template load<false>(v0, in ? 8 : 0, false);
    p.settle();
    g.settle();
    float2 mn[4], vn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 gi = __fmul2_rn(g.pair(i), twice(f.g));
      mn[i] = first_moment(m.pair(i), gi, s);
      vn[i] = second_moment(v.pair(i), gi, s);
      pv[i] = parameter(p.pair(i), mn[i], make_float2(root_of(vn[i].x), root_of(vn[i].y)), f, s);
    }
    if (in) {
      m.set(mn);
      m.store(m0, 8);
      v.set(vn);
      v.store(v0, 8);
    }
  }
  p.set(pv);
  p.store(p0 + at, n - at);
  if (e.copy) {
    Eight<uint16_t, ANY> c;
    c.set(pv);
    c.store(e.copy + from + at, n - at);
  }
}

template <int CAP, bool EIGHT>
__global__ void __launch_bounds__(kThreads, resident(EIGHT)) adamw(const __grid_constant__ List<CAP> L,
                                                                   const __grid_constant__ Step s) {
  const int i = find_tensor(L.first, L.count, blockIdx.x);
  const Entry& e = L.t[i];
  const float lr = (s.lr_dev ? *s.lr_dev : s.lr) * e.lr_scale;
  Factors f;
  f.g = s.grad_scale ? *s.grad_scale : 1.0f;
  float c1 = s.c1;
  f.root = s.root;
  // (In 64 bits, as the host has them, in every block ahead of its loads: 218 million bf16
  // values with states in 8 bits 445 us for 395, fp32 888 both.)
  if (s.step_dev) {
    __shared__ float c[2];
    const int64_t step = *s.step_dev;
    if (step < 1) return;
    if (threadIdx.x == 0) {
      c[0] = static_cast<float>(-1.0 / expm1(static_cast<double>(step) * s.log1));
      c[1] = static_cast<float>(1.0 / sqrt(-expm1(static_cast<double>(step) * s.log2)));
    }
    __syncthreads();
    c1 = c[0];
    f.root = c[1];
  }
  if (!isfinite(f.g) || !isfinite(lr)) return;
  f.keep = fmaf(-lr, e.decay, 1.0f);
  f.rate = lr * c1;
  const int64_t from = static_cast<int64_t>(blockIdx.x - L.first[i]) * kChunk;
  const int n = static_cast<int>(min(e.numel - from, kChunk));
  switch (L.kind[i]) {
    case 0: chunk<EIGHT, true, uint16_t, uint16_t>(e, s, f, from, n); break;
    case 1: chunk<EIGHT, true, float, uint16_t>(e, s, f, from, n); break;
    case 2: chunk<EIGHT, true, uint16_t, float>(e, s, f, from, n); break;
    case 3: chunk<EIGHT, true, float, float>(e, s, f, from, n); break;
    case 4: chunk<EIGHT, false, uint16_t, uint16_t>(e, s, f, from, n); break;
    case 5: chunk<EIGHT, false, float, uint16_t>(e, s, f, from, n); break;
    case 6: chunk<EIGHT, false, uint16_t, float>(e, s, f, from, n); break;
    default: chunk<EIGHT, false, float, float>(e, s, f, from, n);
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
  // (a normal number in 32 bits: the reciprocal takes what lies below for 0)
  if (!std::isfinite(eps) || eps < 0x1p-126) return FRAG_ERR_INVALID_ARG;
  // (in 32 bits, as the kernel takes it: there a rate that is not finite changes nothing)
  if (!lr_device && !std::isfinite(static_cast<float>(lr))) return FRAG_ERR_INVALID_ARG;
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
    if (!lr_device && !std::isfinite(static_cast<float>(lr) * t.lr_scale)) return FRAG_ERR_INVALID_ARG;
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
  Step p = {};
  p.m = exp_avg;
  p.v = exp_avg_sq;
  p.m_scale = exp_avg_scale;
  p.v_scale = exp_avg_sq_scale;
  p.grad_scale = grad_scale;
  p.lr_dev = lr_device;
  p.step_dev = step_device;
  p.log1 = std::log(beta1);
  p.log2 = std::log(beta2);
  p.lr = static_cast<float>(lr);
  p.b1 = static_cast<float>(beta1);
  p.a1 = static_cast<float>(1.0 - beta1);
  p.b2 = static_cast<float>(beta2);
  p.a2 = static_cast<float>(1.0 - beta2);
  p.eps = static_cast<float>(eps);
  if (!step_device) {
    p.c1 = static_cast<float>(-1.0 / std::expm1(static_cast<double>(step) * p.log1));
    p.root = static_cast<float>(1.0 / std::sqrt(-std::expm1(static_cast<double>(step) * p.log2)));
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return eight ? launch_lists<true>(tensors, grads, grad_dtypes, count, p, s)
               : launch_lists<false>(tensors, grads, grad_dtypes, count, p, s);
}

}  // extern "C"

// rmsnorm_quant.cu — (residual add +) RMSNorm with its output in 8 bits and
// scales, and the gradient of the same in bf16 and in 8 bits.
//
// Forward, row by row:
//   h = bf16(res + x), rstd = 1/sqrt(mean(h^2) + eps), y = h rstd w,
//   scale = max|y| / fmax over the row or each group of it, q = fp8(y / scale)
// h is rounded because it is the residual stream that the backward reads; y
// is not rounded before it becomes 8 bits, so q and scale carry one rounding.
//
// Gradient: xhat = x rstd, g = dy w,
//   dx = dres + (g - xhat mean(xhat g)) rstd,  dw = sum over rows of dy xhat
// rounded once to bf16 and once, from the same 32 bits, to 8.
//
// Bound: HBM with the residual (32768 rows of 8192, group 128: 284 us, 6.6 TB/s,
// the measured copy's rate; scales for whole rows 278), instruction issue
// without (three bytes a value: 16384 rows of 4096 41 us for a floor of 31, 52
// with a scale for each 128) and in the gradient (8192 rows of 4096 with the
// residual 58 us for a floor of 46, 3.5 of them the dweight's second pass).
// Further from it: rows above 8192 values (4096 rows of 16384 with the residual
// 92 us for 72, the gradient 153 for 92), rows that are not aligned (8192 rows of
// 4097 92 us for 36, the gradient 190 for 46) and rows above 16384 values (4096
// rows of 20000 373 us for 88, the gradient 523 for 113).
#include <algorithm>
#include <atomic>

#include "quant.cuh"

namespace frag {
namespace {

// Which kernel takes rows of N values: chunks of eight in registers (a warp or
// a block a row), single values in registers where rows are not aligned, or
// the row read again from L2 where it does not fit in registers.
enum RowKind { ROW_WARP, ROW_BLOCK, ROW_ODD_WARP, ROW_ODD, ROW_ANY };
struct RowShape {
  RowKind kind;
  int K, threads;  // chunks (or four single values) a thread, threads of a block
};
// Rows of up to so many values are a warp's; the gradient keeps twice the
// values of the forward in registers.
constexpr int kWarpRowFwd = 1024, kWarpRowBwd = 512;
RowShape row_shape(int64_t N, bool aligned, int warp_row) {
  if (N > 16384) return {ROW_ANY, 0, 256};
  if (!aligned || N % 8 != 0) {
    if (N <= warp_row) return {ROW_ODD_WARP, N <= 256 ? 2 : N <= 512 ? 4 : 8, 256};
    const int K = N <= 8192 ? 4 : 8;
    return {ROW_ODD, K, static_cast<int>(ceil_div(N, 128 * K) * 32)};
  }
  if (N <= warp_row) return {ROW_WARP, N <= 256 ? 1 : N <= 512 ? 2 : 4, 256};
  // Two chunks a thread up to 512 threads, four beyond (16384 rows of 4096 with
  // the residual: two 72 us, four 76, one 86).
  const int K = N <= 8192 ? 2 : 4;
  return {ROW_BLOCK, K, static_cast<int>(ceil_div(N, 256 * K) * 32)};
}

struct QuantFwdP {
  const uint16_t* x;
  const uint16_t* res;
  const uint16_t* w;
  uint16_t* h;
  float* rstd;
  int64_t xs, rs;  // row strides
  QuantOut o;
  int64_t N;
  int group;  // 0: the row
  float eps;
};

// Quantise the row's values value(n), n < N, from a whole block: a scale for
// the row, or a warp for each group in turn.
template <bool E5M2, bool E8M0, class F>
__device__ __forceinline__ void quant_row(const QuantOut& o, int64_t row, int64_t N, int group, F value,
                                          float (*slots)[32]) {
  uint8_t* q = o.q + row * N;
  if (group == 0) {
    float most = 0.f;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) most = max_mag(most, value(n));
    most = block_max_mag(most, slots, 0);
    float inv;
    uint8_t byte = 0;
    const float s = quant_scale<E5M2, E8M0>(most, inv, byte);
    if (threadIdx.x == 0) store_scale<E8M0>(o, row, s, byte);
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) q[n] = to_fp8<E5M2>(value(n) * inv);
    return;
  }
  const int lane = threadIdx.x & 31;
  for (int64_t g = threadIdx.x >> 5; g < o.groups; g += blockDim.x >> 5) {
    const int64_t n0 = g * group, n1 = min(N, n0 + group);
    float v[4];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = n0 + lane + 32 * i;
      v[i] = n < n1 ? value(n) : 0.f;
      most = max_mag(most, v[i]);
    }
    most = warp_max_mag(most);
    float inv;
    uint8_t byte = 0;
    const float s = quant_scale<E5M2, E8M0>(most, inv, byte);
    if (lane == 0) store_scale<E8M0>(o, row * o.groups + g, s, byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = n0 + lane + 32 * i;
      if (n < n1) q[n] = to_fp8<E5M2>(v[i] * inv);
    }
  }
}

// Quantise the K chunks of eight values that each of a row's T threads holds;
// `most` is each chunk's largest magnitude.
template <int K, bool WARP, bool E5M2, bool E8M0>
__device__ __forceinline__ void quant_chunks(const QuantOut& o, int64_t row, int64_t N, int group, int t, int T,
                                             int chunks, const float2 (&y)[K][4], const float (&most)[K],
                                             float (*slots)[32], int parity) {
  float inv = 0.f, s;
  uint8_t byte = 0;
  if (group == 0) {
    float m = most[0];
#pragma unroll
    for (int k = 1; k < K; ++k) m = max_mag(m, most[k]);
    m = WARP ? warp_max_mag(m) : block_max_mag(m, slots, parity);
    s = quant_scale<E5M2, E8M0>(m, inv, byte);
    if (t == 0) store_scale<E8M0>(o, row, s, byte);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = t + k * T;
    if (group) {
      float m = most[k];
      m = max_mag(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max_mag(m, __shfl_xor_sync(0xffffffffu, m, 2));
      if (group >= 64) m = max_mag(m, __shfl_xor_sync(0xffffffffu, m, 4));
      if (group >= 128) m = max_mag(m, __shfl_xor_sync(0xffffffffu, m, 8));
      s = quant_scale<E5M2, E8M0>(m, inv, byte);
      const int lanes = group >> 3;
      if ((c & (lanes - 1)) == 0 && c < chunks) store_scale<E8M0>(o, row * o.groups + c / lanes, s, byte);
    }
    if (c < chunks) {
      const float2 f = make_float2(inv, inv);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = __fmul2_rn(y[k][i], f);
        w[i] = to_fp8x2<E5M2>(v.x, v.y);
      }
      const uint2 q = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
      *reinterpret_cast<uint2*>(o.q + row * N + static_cast<int64_t>(c) * 8) = q;
    }
  }
}

// Quantise values that lie 32 apart, 4 K of them a thread (zeros past the
// row): value i of round k is number first + k step + 32 i.
template <int K, bool WARP, bool E5M2, bool E8M0>
__device__ __forceinline__ void quant_lanes(const QuantOut& o, int64_t row, int N, int group, int first, int step,
                                            const float (&y)[K][4], float (*slots)[32], int parity) {
  uint8_t* q = o.q + row * N;
  const int lane = threadIdx.x & 31;
  float inv = 0.f, s;
  uint8_t byte = 0;
  if (group == 0) {
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = max_mag(m, y[k][i]);
    m = WARP ? warp_max_mag(m) : block_max_mag(m, slots, parity);
    s = quant_scale<E5M2, E8M0>(m, inv, byte);
    if (WARP ? lane == 0 : threadIdx.x == 0) store_scale<E8M0>(o, row, s, byte);
  }
  const int per = group >> 5;  // 1, 2 or 4 lane rows a group
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float m[4];
    if (group) {
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = warp_max_mag(fabsf(y[k][i]));
      if (per >= 2) {
        m[0] = m[1] = max_mag(m[0], m[1]);
        m[2] = m[3] = max_mag(m[2], m[3]);
      }
      if (per == 4) m[0] = m[1] = m[2] = m[3] = max_mag(m[0], m[2]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = first + k * step + 32 * i;
      if (group) {
        s = quant_scale<E5M2, E8M0>(m[i], inv, byte);
        if (lane == 0 && (i & (per - 1)) == 0 && n < N) store_scale<E8M0>(o, row * o.groups + n / group, s, byte);
      }
      if (n < N) q[n] = to_fp8<E5M2>(y[k][i] * inv);
    }
  }
}

// Any width, any alignment: one CTA per row, the row read once for each pass
// (the later passes from L2).
template <bool E5M2, bool E8M0>
__global__ void __launch_bounds__(256) quant_fwd_any(const QuantFwdP p) {
  __shared__ float slots[2][32];
  __shared__ float mslots[2][32];
  const int64_t row = blockIdx.x;
  const uint16_t* x = p.x + row * p.xs;
  const uint16_t* res = p.res ? p.res + row * p.rs : nullptr;
  auto h = [&](int64_t n) {
    const float v = bf16_to_f(x[n]);
    return res ? round_bf16(bf16_to_f(res[n]) + v) : v;
  };
  float ss = 0.f;
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) {
    const float v = h(n);
    if (p.h) p.h[row * p.N + n] = f_to_bf16(v);
    ss = fmaf(v, v, ss);
  }
  const float r = rsqrtf(block_sum_lanes(ss, slots, 0) / static_cast<float>(p.N) + p.eps);
  if (p.rstd && threadIdx.x == 0) p.rstd[row] = r;
  quant_row<E5M2, E8M0>(p.o, row, p.N, p.group, [&](int64_t n) { return (h(n) * r) * bf16_to_f(p.w[n]); },
                        mslots);
}

// Rows of 16-byte chunks, the row in registers: thread t of the row's threads
// owns the chunks t, t + T, ... (K of them); T is the block, or with WARP a
// warp of it (rows of up to 1024 values, no barrier).  A group of 32, 64 or 128
// values is 4, 8 or 16 neighbouring lanes.  A block (or warp) stays for R rows,
// with the weights in registers and the next row's loads in flight while this
// one is reduced (without AHEAD, where registers run out, not).
template <int K, bool WARP, bool AHEAD, bool HAS_RES, bool E5M2, bool E8M0>
__global__ void __launch_bounds__(512) quant_fwd_vec(const QuantFwdP p, int64_t M, int R) {
  __shared__ float slots[2][32];
  __shared__ float mslots[2][32];
  const int T = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int per = WARP ? blockDim.x >> 5 : 1;
  int64_t row = static_cast<int64_t>(blockIdx.x) * per * R + (WARP ? threadIdx.x >> 5 : 0);
  const int64_t end = min(M, static_cast<int64_t>(blockIdx.x + 1) * per * R);
  const int chunks = static_cast<int>(p.N >> 3);
  uint4 xv[K], rv[K], wv[K];
  auto load = [&](int64_t n) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = t + k * T;
      if (n < end && c < chunks) {
        xv[k] = HAS_RES ? ld_plain(p.x + n * p.xs + c * 8) : ld_stream(p.x + n * p.xs + c * 8);
        if (HAS_RES) rv[k] = ld_plain(p.res + n * p.rs + c * 8);
      }
    }
  };
#pragma unroll
  for (int k = 0; k < K; ++k) xv[k] = rv[k] = make_uint4(0, 0, 0, 0);
  load(row);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = t + k * T;
    wv[k] = c < chunks ? ld_cached(p.w + c * 8) : make_uint4(0, 0, 0, 0);
  }
  for (int parity = 0; row < end; row += per, parity ^= 1) {
    uint4 hv[K];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = t + k * T;
      hv[k] = HAS_RES ? add_bf16x8(rv[k], xv[k]) : xv[k];
      if (HAS_RES && p.h && c < chunks) st_global(p.h + row * p.N + c * 8, hv[k]);
      float2 sq = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = bf16x2_to_f2(u4_word(hv[k], i));
        sq = __ffma2_rn(v, v, sq);
      }
      ss += sq.x + sq.y;
    }
    if (AHEAD) load(row + per);
    ss = WARP ? warp_sum(ss) : block_sum_lanes(ss, slots, parity);
    const float r = rsqrtf(ss / static_cast<float>(p.N) + p.eps);
    if (p.rstd && t == 0) p.rstd[row] = r;
    float2 y[K][4];
    float most[K];
    const float2 r2 = make_float2(r, r);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      most[k] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[k][i] = __fmul2_rn(__fmul2_rn(bf16x2_to_f2(u4_word(hv[k], i)), r2), bf16x2_to_f2(u4_word(wv[k], i)));
        most[k] = max_mag2(most[k], y[k][i]);
      }
      if (t + k * T >= chunks) most[k] = 0.f;  // (past the row there are zeros, but 0 * inf is NaN)
    }
    quant_chunks<K, WARP, E5M2, E8M0>(p.o, row, p.N, p.group, t, T, chunks, y, most, mslots, parity);
    if (!AHEAD) load(row + per);
  }
}

// Rows without that alignment, up to 16384 values in registers: warp w of the
// row's W owns 128 neighbouring values at a time, lane l every 32nd of them, so
// a group of 32, 64 or 128 lies within a warp.  WARP: a warp a row (W = 1).
template <int K, bool WARP, bool HAS_RES, bool E5M2, bool E8M0>
__global__ void __launch_bounds__(512) quant_fwd_odd(const QuantFwdP p, int64_t M) {
  __shared__ float slots[2][32];
  __shared__ float mslots[2][32];
  const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= M) return;
  const bool lead = WARP ? (threadIdx.x & 31) == 0 : threadIdx.x == 0;
  const int N = static_cast<int>(p.N);
  const uint16_t* x = p.x + row * p.xs;
  const uint16_t* res = HAS_RES ? p.res + row * p.rs : nullptr;
  const int first = (WARP ? 0 : (threadIdx.x >> 5) * 128) + (threadIdx.x & 31), step = WARP ? 128 : blockDim.x * 4;
  float y[K][4];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = first + k * step + 32 * i;
      y[k][i] = n < N ? bf16_to_f(x[n]) : 0.f;
    }
  if (HAS_RES) {
    float rf[K][4];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = first + k * step + 32 * i;
        rf[k][i] = n < N ? bf16_to_f(res[n]) : 0.f;
      }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = first + k * step + 32 * i;
        const uint16_t h = f_to_bf16(rf[k][i] + y[k][i]);
        if (p.h && n < N) p.h[row * p.N + n] = h;
        y[k][i] = bf16_to_f(h);
      }
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) ss = fmaf(y[k][i], y[k][i], ss);
  ss = WARP ? warp_sum(ss) : block_sum_lanes(ss, slots, 0);
  const float r = rsqrtf(ss / static_cast<float>(N) + p.eps);
  if (p.rstd && lead) p.rstd[row] = r;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = first + k * step + 32 * i;
      y[k][i] = n < N ? (y[k][i] * r) * bf16_to_f(p.w[n]) : 0.f;
    }
  quant_lanes<K, WARP, E5M2, E8M0>(p.o, row, N, p.group, first, step, y, mslots, 0);
}

struct QuantBwdP {
  const uint16_t* dy;
  const uint16_t* x;
  const float* rstd;
  const uint16_t* w;
  const uint16_t* dres;
  uint16_t* dx;
  float* partials;  // [G, N]
  int64_t ys, xs, rs;
  QuantOut o;
  int64_t N;
  int group;
};

// The sums of dweight that each of a block's warps holds for its own rows,
// added in warp order into the block's partials: value(n) of warp w at
// acc[w * N + n] of shared memory.
__device__ __forceinline__ void store_partials(const QuantBwdP& p, const float* acc) {
  __syncthreads();
  for (int n = threadIdx.x; n < p.N; n += blockDim.x) {
    float t = 0.f;
    for (int w = 0; w < blockDim.x >> 5; ++w) t += acc[w * p.N + n];
    p.partials[static_cast<int64_t>(blockIdx.x) * p.N + n] = t;
  }
}

// dx of one value, in 32 bits.
__device__ __forceinline__ float grad_of(float g, float xhat, float mean, float r) { return (g - xhat * mean) * r; }

// The gradient's arithmetic on a chunk of eight, in pairs (one instruction for
// two columns): the chunk's part of sum(x g), g = dy w ...
__device__ __forceinline__ float chunk_dot(const uint4& y, const uint4& x, const uint4& w) {
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    s = __ffma2_rn(bf16x2_to_f2(u4_word(x, i)), __fmul2_rn(bf16x2_to_f2(u4_word(y, i)), bf16x2_to_f2(u4_word(w, i))), s);
  return s.x + s.y;
}
// ... and d = dres + (g - xhat mean) r, dweight += dy xhat, the largest |d|.
template <bool HAS_RES>
__device__ __forceinline__ float chunk_grad(const uint4& y, const uint4& x, const uint4& w, const uint4& res, float mean,
                                            float r, float2 (&acc)[4], float2 (&d)[4]) {
  const float2 r2 = make_float2(r, r), m2 = make_float2(-mean, -mean);
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 dy = bf16x2_to_f2(u4_word(y, i));
    const float2 xhat = __fmul2_rn(bf16x2_to_f2(u4_word(x, i)), r2);
    acc[i] = __ffma2_rn(dy, xhat, acc[i]);
    const float2 t = __ffma2_rn(xhat, m2, __fmul2_rn(dy, bf16x2_to_f2(u4_word(w, i))));
    d[i] = HAS_RES ? __ffma2_rn(t, r2, bf16x2_to_f2(u4_word(res, i))) : __fmul2_rn(t, r2);
    most = max_mag2(most, d[i]);
  }
  return most;
}
__device__ __forceinline__ uint4 pack_pairs(const float2 (&d)[4]) {
  return make_uint4(f2_to_bf16x2(d[0]), f2_to_bf16x2(d[1]), f2_to_bf16x2(d[2]), f2_to_bf16x2(d[3]));
}

// Rows of up to 512 values in 16-byte chunks, a warp a row: a block's warps
// take rows_per_block rows in turn.
template <int K, bool HAS_RES, bool E5M2, bool E8M0>
__global__ void __launch_bounds__(256) quant_bwd_warp(const QuantBwdP p, int64_t M, int64_t rows_per_block) {
  extern __shared__ float sacc[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = static_cast<int>(p.N >> 3);
  uint4 wv[K];
  float2 acc[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = lane + 32 * k;
    wv[k] = c < chunks ? ld_cached(p.w + c * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[k][i] = make_float2(0.f, 0.f);
  }
  const int64_t r1 = min(M, (static_cast<int64_t>(blockIdx.x) + 1) * rows_per_block);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * rows_per_block + warp; row < r1; row += blockDim.x >> 5) {
    uint4 yv[K], xv[K], rv[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = lane + 32 * k;
      yv[k] = xv[k] = rv[k] = make_uint4(0, 0, 0, 0);
      if (c < chunks) {
        yv[k] = ld_stream(p.dy + row * p.ys + c * 8);
        xv[k] = ld_stream(p.x + row * p.xs + c * 8);
        if (HAS_RES) rv[k] = ld_stream(p.dres + row * p.rs + c * 8);
      }
    }
    const float r = __ldg(p.rstd + row);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) sum += chunk_dot(yv[k], xv[k], wv[k]);
    const float mean = r * warp_sum(sum) / static_cast<float>(p.N);
    float2 d[K][4];
    float most[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = lane + 32 * k;
      most[k] = chunk_grad<HAS_RES>(yv[k], xv[k], wv[k], rv[k], mean, r, acc[k], d[k]);
      if (c >= chunks) most[k] = 0.f;
      if (p.dx && c < chunks) st_global(p.dx + row * p.N + c * 8, pack_pairs(d[k]));
    }
    quant_chunks<K, true, E5M2, E8M0>(p.o, row, p.N, p.group, lane, 32, chunks, d, most, nullptr, 0);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = lane + 32 * k;
    if (c < chunks) {
      float4* o = reinterpret_cast<float4*>(sacc + warp * p.N + c * 8);
      o[0] = make_float4(acc[k][0].x, acc[k][0].y, acc[k][1].x, acc[k][1].y);
      o[1] = make_float4(acc[k][2].x, acc[k][2].y, acc[k][3].x, acc[k][3].y);
    }
  }
  if (p.partials) store_partials(p, sacc);
}

// Longer rows in 16-byte chunks, a block a row: thread 0 streams the rows of
// the block (dy, x, dres) into a ring of S stages by bulk copies, S rows ahead
// of the arithmetic; dweight sums stay in registers, thread-owned columns.
// Four chunks a thread do not fit in the 128 registers of 512 threads: 276 bytes
// are spilled with the residual and 200 without (three chunks: 64 and 16).
template <int K, bool HAS_RES, bool E5M2, bool E8M0>
__global__ void __launch_bounds__(K == 3 ? 256 : 512, K == 3 ? 2 : 1)
quant_bwd_ring(const QuantBwdP p, int64_t M, int64_t rows_per_block, int S, int* err) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float slots[2][32];
  __shared__ float mslots[2][32];
  __shared__ int s_abort;
  constexpr int NIN = HAS_RES ? 3 : 2;
  const int N = static_cast<int>(p.N), chunks = N >> 3, row_bytes = N * 2, stage_bytes = NIN * row_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + static_cast<size_t>(S) * stage_bytes);
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * rows_per_block;
  const int rows = static_cast<int>(min(M - r0, rows_per_block));
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < S; ++i) mbar_init(&bars[i], 1);
    mbar_init_fence();
  }
  __syncthreads();
  int issued = 0;
  auto issue = [&](int i) {
    if (i >= rows) return;
    unsigned char* st = smem + static_cast<size_t>(i % S) * stage_bytes;
    mbar_arrive_expect_tx(&bars[i % S], stage_bytes);
    const uint64_t pol = l2_policy_evict_first();
    bulk_g2s_hint(st, p.dy + (r0 + i) * p.ys, row_bytes, &bars[i % S], pol);
    bulk_g2s_hint(st + row_bytes, p.x + (r0 + i) * p.xs, row_bytes, &bars[i % S], pol);
    if (HAS_RES) bulk_g2s_hint(st + 2 * row_bytes, p.dres + (r0 + i) * p.rs, row_bytes, &bars[i % S], pol);
    issued = i + 1;
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < S; ++i) issue(i);
  uint4 wv[K];
  float2 acc[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = threadIdx.x + k * blockDim.x;
    wv[k] = c < chunks ? ld_cached(p.w + c * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[k][i] = make_float2(0.f, 0.f);
  }
  int i = 0;
  for (; i < rows; ++i) {
    const int64_t row = r0 + i;
    const float r = __ldg(p.rstd + row);
    const unsigned char* st = smem + static_cast<size_t>(i % S) * stage_bytes;
    if (!mbar_wait(&bars[i % S], (i / S) & 1, err)) s_abort = 1;
    uint4 yv[K], xv[K], rv[K];
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = threadIdx.x + k * blockDim.x;
      yv[k] = xv[k] = rv[k] = make_uint4(0, 0, 0, 0);
      if (c < chunks) {
        yv[k] = *reinterpret_cast<const uint4*>(st + c * 16);
        xv[k] = *reinterpret_cast<const uint4*>(st + row_bytes + c * 16);
        if (HAS_RES) rv[k] = *reinterpret_cast<const uint4*>(st + 2 * row_bytes + c * 16);
      }
      sum += chunk_dot(yv[k], xv[k], wv[k]);
    }
    const float mean = r * block_sum_lanes(sum, slots, i & 1) / static_cast<float>(N);
    if (s_abort) break;
    if (threadIdx.x == 0) issue(i + S);  // every thread has read stage i % S
    float2 d[K][4];
    float most[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = threadIdx.x + k * blockDim.x;
      most[k] = chunk_grad<HAS_RES>(yv[k], xv[k], wv[k], rv[k], mean, r, acc[k], d[k]);
      if (c >= chunks) most[k] = 0.f;
      if (p.dx && c < chunks) st_stream(p.dx + row * N + c * 8, pack_pairs(d[k]));
    }
    quant_chunks<K, false, E5M2, E8M0>(p.o, row, N, p.group, threadIdx.x, blockDim.x, chunks, d, most, mslots, i & 1);
  }
  if (threadIdx.x == 0 && s_abort)
    for (int j = i; j < issued; ++j) mbar_wait(&bars[j % S], (j / S) & 1, nullptr);
  if (!p.partials) return;
  float* part = p.partials + static_cast<int64_t>(blockIdx.x) * N;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = threadIdx.x + k * blockDim.x;
    if (c < chunks) {
      *reinterpret_cast<float4*>(part + c * 8) = make_float4(acc[k][0].x, acc[k][0].y, acc[k][1].x, acc[k][1].y);
      *reinterpret_cast<float4*>(part + c * 8 + 4) = make_float4(acc[k][2].x, acc[k][2].y, acc[k][3].x, acc[k][3].y);
    }
  }
}

// Rows without that alignment, up to 16384 values, single values in registers
// (the layout of quant_fwd_odd); WARP: a warp a row.  Eight rounds of values in a
// block's threads (above 8192) spill 208 to 216 bytes with the residual, 64 to 72
// without.
template <int K, bool WARP, bool HAS_RES, bool E5M2, bool E8M0>
__global__ void __launch_bounds__(512) quant_bwd_odd(const QuantBwdP p, int64_t M, int64_t rows_per_block) {
  extern __shared__ float sacc[];  // WARP
  __shared__ float slots[2][32];
  __shared__ float mslots[2][32];
  const int N = static_cast<int>(p.N), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = (WARP ? 0 : warp * 128) + lane, step = WARP ? 128 : blockDim.x * 4;
  float acc[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[k][i] = 0.f;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * rows_per_block, r1 = min(M, r0 + rows_per_block);
  int parity = 0;
  for (int64_t row = r0 + (WARP ? warp : 0); row < r1; row += WARP ? blockDim.x >> 5 : 1, parity ^= 1) {
    const uint16_t* dy = p.dy + row * p.ys;
    const uint16_t* x = p.x + row * p.xs;
    const uint16_t* dres = HAS_RES ? p.dres + row * p.rs : nullptr;
    const float r = __ldg(p.rstd + row);
    float g[K][4], xh[K][4], d[K][4];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = first + k * step + 32 * i;
        g[k][i] = n < N ? bf16_to_f(dy[n]) : 0.f;
        xh[k][i] = n < N ? bf16_to_f(x[n]) : 0.f;
        d[k][i] = HAS_RES && n < N ? bf16_to_f(dres[n]) : 0.f;
      }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = first + k * step + 32 * i;
        xh[k][i] *= r;
        acc[k][i] = fmaf(g[k][i], xh[k][i], acc[k][i]);
        g[k][i] *= n < N ? bf16_to_f(__ldg(p.w + n)) : 0.f;
        sum = fmaf(xh[k][i], g[k][i], sum);
      }
    const float mean = (WARP ? warp_sum(sum) : block_sum_lanes(sum, slots, parity)) / static_cast<float>(N);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = first + k * step + 32 * i;
        d[k][i] = n < N ? d[k][i] + grad_of(g[k][i], xh[k][i], mean, r) : 0.f;
        if (p.dx && n < N) p.dx[row * N + n] = f_to_bf16(d[k][i]);
      }
    quant_lanes<K, WARP, E5M2, E8M0>(p.o, row, N, p.group, first, step, d, mslots, parity);
  }
  if (!p.partials) return;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = first + k * step + 32 * i;
      if (n < N) (WARP ? sacc + warp * N : p.partials + static_cast<int64_t>(blockIdx.x) * N)[n] = acc[k][i];
    }
  if (WARP) store_partials(p, sacc);
}

template <bool E5M2, bool E8M0>
__global__ void __launch_bounds__(256) quant_bwd_any(const QuantBwdP p) {
  __shared__ float slots[2][32];
  __shared__ float mslots[2][32];
  const int64_t row = blockIdx.x;
  const uint16_t* dy = p.dy + row * p.ys;
  const uint16_t* x = p.x + row * p.xs;
  const uint16_t* dres = p.dres ? p.dres + row * p.rs : nullptr;
  const float r = p.rstd[row];
  float sum = 0.f;
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x)
    sum = fmaf(bf16_to_f(x[n]) * r, bf16_to_f(dy[n]) * bf16_to_f(p.w[n]), sum);
  const float mean = block_sum_lanes(sum, slots, 0) / static_cast<float>(p.N);
  auto dx = [&](int64_t n) {
    const float xhat = bf16_to_f(x[n]) * r;
    const float d = (bf16_to_f(dy[n]) * bf16_to_f(p.w[n]) - xhat * mean) * r;
    return dres ? bf16_to_f(dres[n]) + d : d;
  };
  if (p.dx)
    for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) p.dx[row * p.N + n] = f_to_bf16(dx(n));
  quant_row<E5M2, E8M0>(p.o, row, p.N, p.group, dx, mslots);
}

// dweight partials of a row block, one thread per column.
__global__ void __launch_bounds__(256) quant_bwd_any_dw(const QuantBwdP p, int64_t M, int64_t rows_per_block) {
  const int64_t col = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (col >= p.N) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows_per_block;
  const int64_t r1 = min(M, r0 + rows_per_block);
  float acc = 0.f;
  for (int64_t row = r0; row < r1; ++row)
    acc = fmaf(bf16_to_f(p.dy[row * p.ys + col]), bf16_to_f(p.x[row * p.xs + col]) * p.rstd[row], acc);
  p.partials[static_cast<int64_t>(blockIdx.y) * p.N + col] = acc;
}

// Row blocks of the dweight partials: the same for every call of M rows of N.
struct QuantBwdPlan {
  int64_t G, rows_per_block;
};
// Chunks of a thread and threads of a row's block, and blocks of an SM: two
// chunks, but three just above 4096, where two would leave one block of little
// more than 256 threads an SM (22686 rows of 4176, group 128: 172 us against
// 222; from 6160 on two are faster, 8192 rows of 8192 111 against 155 for four).
int ring_chunks(int64_t N) { return N <= 4096 ? 2 : N <= 6144 ? 3 : N <= 8192 ? 2 : 4; }
int ring_threads(int64_t N) { return static_cast<int>(ceil_div(N, 256 * ring_chunks(N)) * 32); }
int ring_blocks(int threads) { return std::max(1, std::min(4, 512 / threads)); }

QuantBwdPlan quant_bwd_plan(int64_t M, int64_t N) {
  int sms = sm_count();
  if (sms <= 0) sms = 148;
  // a warp a row: two blocks of eight an SM; a block a row: 512 threads an SM
  const int64_t blocks = N <= kWarpRowBwd ? std::min<int64_t>(ceil_div(M, 8), 2 * sms)
                                          : std::min<int64_t>(M, ring_blocks(ring_threads(N)) * sms);
  const int64_t rows = ceil_div(M, std::max<int64_t>(1, blocks));
  return {ceil_div(M, rows), rows};
}

template <int K, bool HAS_RES, bool E5M2, bool E8M0>
int launch_bwd_ring(const QuantBwdP& p, int64_t M, const QuantBwdPlan& pl, cudaStream_t s) {
  const int stage_bytes = (HAS_RES ? 3 : 2) * static_cast<int>(p.N) * 2;
  const int threads = ring_threads(p.N), cps = ring_blocks(threads);
  const int S = std::min(8, (220 * 1024 / cps - 1024) / (stage_bytes + 8));
  const int smem = S * (stage_bytes + 8);
  auto kern = quant_bwd_ring<K, HAS_RES, E5M2, E8M0>;
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kern), smem)) return FRAG_ERR_CUDA;
  kern<<<static_cast<unsigned>(pl.G), threads, smem, s>>>(p, M, pl.rows_per_block, S, device_error_word());
  return check_launch();
}

template <bool HAS_RES, bool E5M2, bool E8M0>
int launch_bwd(const QuantBwdP& p, int64_t M, const QuantBwdPlan& pl, const RowShape& r, cudaStream_t s) {
  const unsigned G = static_cast<unsigned>(pl.G);
  const int wsmem = static_cast<int>(8 * p.N * sizeof(float));  // the warps' dweight sums (up to 16 KB)
  switch (r.kind) {
    case ROW_WARP:
      if (r.K == 1) quant_bwd_warp<1, HAS_RES, E5M2, E8M0><<<G, 256, wsmem, s>>>(p, M, pl.rows_per_block);
      else quant_bwd_warp<2, HAS_RES, E5M2, E8M0><<<G, 256, wsmem, s>>>(p, M, pl.rows_per_block);
      return check_launch();
    case ROW_BLOCK:
      switch (ring_chunks(p.N)) {
        case 2: return launch_bwd_ring<2, HAS_RES, E5M2, E8M0>(p, M, pl, s);
        case 3: return launch_bwd_ring<3, HAS_RES, E5M2, E8M0>(p, M, pl, s);
        default: return launch_bwd_ring<4, HAS_RES, E5M2, E8M0>(p, M, pl, s);
      }
    case ROW_ODD_WARP:
      if (r.K == 2) quant_bwd_odd<2, true, HAS_RES, E5M2, E8M0><<<G, 256, wsmem, s>>>(p, M, pl.rows_per_block);
      else quant_bwd_odd<4, true, HAS_RES, E5M2, E8M0><<<G, 256, wsmem, s>>>(p, M, pl.rows_per_block);
      return check_launch();
    case ROW_ODD:
      if (r.K == 4) quant_bwd_odd<4, false, HAS_RES, E5M2, E8M0><<<G, r.threads, 0, s>>>(p, M, pl.rows_per_block);
      else quant_bwd_odd<8, false, HAS_RES, E5M2, E8M0><<<G, r.threads, 0, s>>>(p, M, pl.rows_per_block);
      return check_launch();
    default: break;
  }
  quant_bwd_any<E5M2, E8M0><<<static_cast<unsigned>(M), 256, 0, s>>>(p);
  int st = check_launch();
  if (st != FRAG_OK || !p.partials) return st;
  quant_bwd_any_dw<<<dim3(static_cast<unsigned>(ceil_div(p.N, 256)), G), 256, 0, s>>>(p, M, pl.rows_per_block);
  return check_launch();
}

// `units` rows (or eights of rows) over blocks that stay for R of them.  With
// the residual, R = 4 as far as that leaves two blocks for every place on the
// device: 32768 rows of 8192, group 128, 284 us against 357 for one and 326
// for as many blocks as are resident; 16384 rows of 4096 75, 89 and 88.
// Without, as many blocks as are resident: 16384 rows of 4096 40, 61 for one.
template <auto kern>  // (a parameter of its own for each kernel: their types are the same)
int launch_stay(int64_t units, bool has_res, int threads, const QuantFwdP& p, int64_t M, cudaStream_t s) {
  // this kernel's resident blocks by warps of a block; the same on every device of this architecture
  static std::atomic<int> per_sm[33];
  int n = per_sm[threads / 32].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0) == cudaSuccess && n > 0) {
      per_sm[threads / 32].store(n, std::memory_order_relaxed);
    } else {
      cudaGetLastError();
      n = 1;
    }
  }
  const int64_t places = static_cast<int64_t>(n) * std::max(1, sm_count());
  const int64_t R = has_res ? std::max<int64_t>(1, std::min<int64_t>(4, units / (2 * places))) : ceil_div(units, places);
  kern<<<static_cast<unsigned>(ceil_div(units, R)), threads, 0, s>>>(p, M, static_cast<int>(R));
  return check_launch();
}

template <bool HAS_RES, bool E5M2, bool E8M0>
int launch_fwd(const QuantFwdP& p, int64_t M, const RowShape& r, cudaStream_t s) {
  const unsigned rows = static_cast<unsigned>(M), warps = static_cast<unsigned>(ceil_div(M, r.threads / 32));
  switch (r.kind) {
    case ROW_WARP:
      if (r.K == 1) return launch_stay<quant_fwd_vec<1, true, true, HAS_RES, E5M2, E8M0>>(warps, HAS_RES, r.threads, p, M, s);
      if (r.K == 2) return launch_stay<quant_fwd_vec<2, true, true, HAS_RES, E5M2, E8M0>>(warps, HAS_RES, r.threads, p, M, s);
      return launch_stay<quant_fwd_vec<4, true, !HAS_RES, HAS_RES, E5M2, E8M0>>(warps, HAS_RES, r.threads, p, M, s);
    case ROW_BLOCK:
      if (r.K == 2) return launch_stay<quant_fwd_vec<2, false, true, HAS_RES, E5M2, E8M0>>(rows, HAS_RES, r.threads, p, M, s);
      return launch_stay<quant_fwd_vec<4, false, !HAS_RES, HAS_RES, E5M2, E8M0>>(rows, HAS_RES, r.threads, p, M, s);
    case ROW_ODD_WARP:
      if (r.K == 2) quant_fwd_odd<2, true, HAS_RES, E5M2, E8M0><<<warps, r.threads, 0, s>>>(p, M);
      else if (r.K == 4) quant_fwd_odd<4, true, HAS_RES, E5M2, E8M0><<<warps, r.threads, 0, s>>>(p, M);
      else quant_fwd_odd<8, true, HAS_RES, E5M2, E8M0><<<warps, r.threads, 0, s>>>(p, M);
      break;
    case ROW_ODD:
      if (r.K == 4) quant_fwd_odd<4, false, HAS_RES, E5M2, E8M0><<<rows, r.threads, 0, s>>>(p, M);
      else quant_fwd_odd<8, false, HAS_RES, E5M2, E8M0><<<rows, r.threads, 0, s>>>(p, M);
      break;
    default: quant_fwd_any<E5M2, E8M0><<<rows, 256, 0, s>>>(p);
  }
  return check_launch();
}

template <class F>
int by_format(int format, int e8m0, F f) {
  if (format == FRAG_FP8_E4M3) return e8m0 ? f(std::false_type(), std::true_type()) : f(std::false_type(), std::false_type());
  return e8m0 ? f(std::true_type(), std::true_type()) : f(std::true_type(), std::false_type());
}

int check_quant(int64_t M, int64_t N, int format, int64_t group) {
  if (M < 0 || N < 0) return FRAG_ERR_INVALID_ARG;
  if (format != FRAG_FP8_E4M3 && format != FRAG_FP8_E5M2) return FRAG_ERR_INVALID_ARG;
  if (group != 0 && group != 32 && group != 64 && group != 128) return FRAG_ERR_SHAPE;
  if ((N == 0 && M > 0) || M > 0x7fffffffLL || N > 0x7fffffffLL) return FRAG_ERR_SHAPE;
  return FRAG_OK;
}

}  // namespace
}  // namespace frag

using namespace frag;

extern "C" {

int frag_rmsnorm_quant_fwd(const void* x, int64_t x_stride, const void* res, int64_t res_stride, const void* w,
                           void* q, void* scale, void* h, float* rstd, int64_t M, int64_t N, float eps,
                           int format, int64_t group, int scale_e8m0, frag_stream_t stream) {
  const int bad = check_quant(M, N, format, group);
  if (bad != FRAG_OK) return bad;
  if (M == 0) return FRAG_OK;
  if (!x || !w || !q || !scale || (h && !res)) return FRAG_ERR_INVALID_ARG;
  QuantFwdP p;
  p.x = static_cast<const uint16_t*>(x);
  p.res = static_cast<const uint16_t*>(res);
  p.w = static_cast<const uint16_t*>(w);
  p.h = static_cast<uint16_t*>(h);
  p.rstd = rstd;
  p.xs = x_stride;
  p.rs = res_stride;
  p.o = QuantOut{static_cast<uint8_t*>(q), scale, group ? ceil_div(N, group) : 1};
  p.N = N;
  p.group = static_cast<int>(group);
  p.eps = eps;
  const RowShape shape = row_shape(N, aligned16(x) && aligned16(w) && (!res || aligned16(res)) &&
                                          (!h || aligned16(h)) && aligned16(q) && (M == 1 || x_stride % 8 == 0) &&
                                          (M == 1 || !res || res_stride % 8 == 0),
                                   kWarpRowFwd);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return by_format(format, scale_e8m0, [&](auto e5m2, auto e8m0) {
    return res ? launch_fwd<true, decltype(e5m2)::value, decltype(e8m0)::value>(p, M, shape, s)
               : launch_fwd<false, decltype(e5m2)::value, decltype(e8m0)::value>(p, M, shape, s);
  });
}

size_t frag_rmsnorm_quant_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 0;
  return align_up(static_cast<size_t>(quant_bwd_plan(M, N).G) * N * sizeof(float), 256);
}

int frag_rmsnorm_quant_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* rstd,
                           const void* w, const void* dres, int64_t dres_stride, void* dx, void* q, void* scale,
                           float* dw, int64_t M, int64_t N, int format, int64_t group, int scale_e8m0,
                           void* workspace, size_t workspace_bytes, frag_stream_t stream) {
  const int bad = check_quant(M, N, format, group);
  if (bad != FRAG_OK) return bad;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (M == 0) return dw ? cuda_status(cudaMemsetAsync(dw, 0, N * sizeof(float), s)) : FRAG_OK;
  if (!dy || !x || !rstd || !w || !q || !scale) return FRAG_ERR_INVALID_ARG;
  const QuantBwdPlan pl = quant_bwd_plan(M, N);
  if (!workspace || workspace_bytes < frag_rmsnorm_quant_bwd_workspace_bytes(M, N)) return FRAG_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FRAG_ERR_ALIGN;
  QuantBwdP p;
  p.dy = static_cast<const uint16_t*>(dy);
  p.x = static_cast<const uint16_t*>(x);
  p.rstd = rstd;
  p.w = static_cast<const uint16_t*>(w);
  p.dres = static_cast<const uint16_t*>(dres);
  p.dx = static_cast<uint16_t*>(dx);
  p.partials = dw ? static_cast<float*>(workspace) : nullptr;
  p.ys = dy_stride;
  p.xs = x_stride;
  p.rs = dres_stride;
  p.o = QuantOut{static_cast<uint8_t*>(q), scale, group ? ceil_div(N, group) : 1};
  p.N = N;
  p.group = static_cast<int>(group);
  const RowShape shape =
      row_shape(N, aligned16(dy) && aligned16(x) && aligned16(w) && (!dres || aligned16(dres)) &&
                       (!dx || aligned16(dx)) && aligned16(q) && (M == 1 || (dy_stride % 8 == 0 && x_stride % 8 == 0)) &&
                       (M == 1 || !dres || dres_stride % 8 == 0),
                kWarpRowBwd);
  const int st = by_format(format, scale_e8m0, [&](auto e5m2, auto e8m0) {
    return dres ? launch_bwd<true, decltype(e5m2)::value, decltype(e8m0)::value>(p, M, pl, shape, s)
                : launch_bwd<false, decltype(e5m2)::value, decltype(e8m0)::value>(p, M, pl, shape, s);
  });
  if (st != FRAG_OK || !dw) return st;
  return dw_reduce_after(p.partials, pl.G, N, dw, shape.kind == ROW_BLOCK, s);
}

}  // extern "C"

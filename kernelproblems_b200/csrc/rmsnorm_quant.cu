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
#include <algorithm>

#include "quant.cuh"

namespace frag {
namespace {

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
                                          uint32_t (*slots)[32]) {
  uint8_t* q = o.q + row * N;
  if (group == 0) {
    uint32_t most = 0;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) most = max(most, mag_bits(value(n)));
    most = block_umax(most, slots, 0);
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
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = n0 + lane + 32 * i;
      v[i] = n < n1 ? value(n) : 0.f;
      most = max(most, mag_bits(v[i]));
    }
    most = __reduce_max_sync(0xffffffffu, most);
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

// Any width, any alignment: one CTA per row, the row read once for each pass
// (the later passes from L2).
template <bool E5M2, bool E8M0>
__global__ void __launch_bounds__(256) quant_fwd_any(const QuantFwdP p) {
  __shared__ float slots[2][32];
  __shared__ uint32_t mslots[2][32];
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
  const float r = rsqrtf(block_sum(ss, slots, 0) / static_cast<float>(p.N) + p.eps);
  if (p.rstd && threadIdx.x == 0) p.rstd[row] = r;
  quant_row<E5M2, E8M0>(p.o, row, p.N, p.group, [&](int64_t n) { return (h(n) * r) * bf16_to_f(p.w[n]); },
                        mslots);
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

template <bool E5M2, bool E8M0>
__global__ void __launch_bounds__(256) quant_bwd_any(const QuantBwdP p) {
  __shared__ float slots[2][32];
  __shared__ uint32_t mslots[2][32];
  const int64_t row = blockIdx.x;
  const uint16_t* dy = p.dy + row * p.ys;
  const uint16_t* x = p.x + row * p.xs;
  const uint16_t* dres = p.dres ? p.dres + row * p.rs : nullptr;
  const float r = p.rstd[row];
  float sum = 0.f;
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x)
    sum = fmaf(bf16_to_f(x[n]) * r, bf16_to_f(dy[n]) * bf16_to_f(p.w[n]), sum);
  const float mean = block_sum(sum, slots, 0) / static_cast<float>(p.N);
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

// Row blocks of the dweight partials: the same for every call of M rows.
struct QuantBwdPlan {
  int64_t G, rows_per_block;
};
QuantBwdPlan quant_bwd_plan(int64_t M) {
  int sms = sm_count();
  if (sms <= 0) sms = 148;
  const int64_t target = std::max<int64_t>(1, std::min<int64_t>(M, 2 * sms));
  const int64_t rows = ceil_div(M, target);
  return {ceil_div(M, rows), rows};
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
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return by_format(format, scale_e8m0, [&](auto e5m2, auto e8m0) {
    quant_fwd_any<decltype(e5m2)::value, decltype(e8m0)::value><<<static_cast<unsigned>(M), 256, 0, s>>>(p);
    return check_launch();
  });
}

size_t frag_rmsnorm_quant_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 0;
  return align_up(static_cast<size_t>(quant_bwd_plan(M).G) * N * sizeof(float), 256);
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
  const QuantBwdPlan pl = quant_bwd_plan(M);
  if (!workspace || workspace_bytes < frag_rmsnorm_quant_bwd_workspace_bytes(M, N)) return FRAG_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FRAG_ERR_ALIGN;
  QuantBwdP p;
  p.dy = static_cast<const uint16_t*>(dy);
  p.x = static_cast<const uint16_t*>(x);
  p.rstd = rstd;
  p.w = static_cast<const uint16_t*>(w);
  p.dres = static_cast<const uint16_t*>(dres);
  p.dx = static_cast<uint16_t*>(dx);
  p.partials = static_cast<float*>(workspace);
  p.ys = dy_stride;
  p.xs = x_stride;
  p.rs = dres_stride;
  p.o = QuantOut{static_cast<uint8_t*>(q), scale, group ? ceil_div(N, group) : 1};
  p.N = N;
  p.group = static_cast<int>(group);
  int st = by_format(format, scale_e8m0, [&](auto e5m2, auto e8m0) {
    quant_bwd_any<decltype(e5m2)::value, decltype(e8m0)::value><<<static_cast<unsigned>(M), 256, 0, s>>>(p);
    return check_launch();
  });
  if (st != FRAG_OK || !dw) return st;
  const dim3 grid(static_cast<unsigned>(ceil_div(N, 256)), static_cast<unsigned>(pl.G));
  quant_bwd_any_dw<<<grid, 256, 0, s>>>(p, M, pl.rows_per_block);
  st = check_launch();
  return st != FRAG_OK ? st : frag_dw_reduce(p.partials, pl.G, N, dw, nullptr, stream);
}

}  // extern "C"

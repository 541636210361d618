// layernorm.cu — (residual add +) layer norm, and its gradient with the sums
// over the rows for weight and bias.
//
// Forward, row by row:
//   h = T(res + x), mean = sum(h) / N, rstd = 1/sqrt(sum((h - mean)^2) / N + eps),
//   y = (h - mean) rstd w + b
// Gradient: xhat = (x - mean) rstd, g = dy w,
//   dx = dres + (g - mean(g) - xhat mean(xhat g)) rstd,
//   dw = sum over rows of dy xhat, db = sum over rows of dy
// Squares are taken about the mean, never as mean(h^2) - mean^2: with a mean of
// a hundred deviations that difference would lose four of the seven digits.
#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace frag {
namespace {

template <class T>
__device__ __forceinline__ float get(const T* p) {
  return sizeof(T) == 2 ? bf16_to_f(*reinterpret_cast<const uint16_t*>(p)) : *reinterpret_cast<const float*>(p);
}
template <class T>
__device__ __forceinline__ void put(T* p, float f) {
  if (sizeof(T) == 2) *reinterpret_cast<uint16_t*>(p) = f_to_bf16(f);
  else *reinterpret_cast<float*>(p) = f;
}
template <class T>
__device__ __forceinline__ float rounded(float f) { return sizeof(T) == 2 ? round_bf16(f) : f; }

// A weight or bias, of either type; `none` where there is none.
struct Vector {
  const void* p;
  int f32;
};
__device__ __forceinline__ float at(const Vector& v, int64_t n, float none) {
  if (!v.p) return none;
  return v.f32 ? static_cast<const float*>(v.p)[n] : bf16_to_f(static_cast<const uint16_t*>(v.p)[n]);
}

template <class T>
struct FwdP {
  const T* x;
  const T* res;
  T* y;
  T* h;
  Vector w, b;
  float* mean;
  float* rstd;
  int64_t xs, rs;  // row strides
  int64_t N;
  float eps;
};

template <class T>
struct BwdP {
  const T* dy;
  const T* x;
  const T* dres;
  T* dx;
  Vector w;
  const float* mean;
  const float* rstd;
  float* partials;  // [G, vectors, N]: dw, db, as far as wanted
  int64_t ys, xs, rs;
  int64_t N;
  int want_dw, want_db;
};

// Any width, any alignment: a block a row, the row read once for each pass
// (the later passes from L2).
template <class T>
__global__ void __launch_bounds__(256) fwd_any(const FwdP<T> p) {
  __shared__ float slots[2][32];
  const int64_t row = blockIdx.x;
  const T* x = p.x + row * p.xs;
  const T* res = p.res ? p.res + row * p.rs : nullptr;
  auto h = [&](int64_t n) { return res ? rounded<T>(get(res + n) + get(x + n)) : get(x + n); };
  float s = 0.f;
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) {
    const float v = h(n);
    if (p.h) put(p.h + row * p.N + n, v);
    s += v;
  }
  const float mean = block_sum(s, slots, 0) / static_cast<float>(p.N);
  s = 0.f;
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) {
    const float v = h(n) - mean;
    s = fmaf(v, v, s);
  }
  const float r = rsqrtf(block_sum(s, slots, 1) / static_cast<float>(p.N) + p.eps);
  if (threadIdx.x == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = r;
  }
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x)
    put(p.y + row * p.N + n, fmaf((h(n) - mean) * r, at(p.w, n, 1.f), at(p.b, n, 0.f)));
}

template <class T>
__global__ void __launch_bounds__(256) bwd_any_dx(const BwdP<T> p) {
  __shared__ float2 slots[2][32];
  const int64_t row = blockIdx.x;
  const T* dy = p.dy + row * p.ys;
  const T* x = p.x + row * p.xs;
  const float mean = p.mean[row], r = p.rstd[row];
  float2 s = make_float2(0.f, 0.f);
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) {
    const float g = get(dy + n) * at(p.w, n, 1.f);
    s.x += g;
    s.y = fmaf((get(x + n) - mean) * r, g, s.y);
  }
  s = block_sum2(s, slots, 0);
  const float invN = 1.0f / static_cast<float>(p.N);
  const float mg = s.x * invN, mx = s.y * invN;
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) {
    const float g = get(dy + n) * at(p.w, n, 1.f), xhat = (get(x + n) - mean) * r;
    const float d = (g - mg - xhat * mx) * r;
    put(p.dx + row * p.N + n, p.dres ? get(p.dres + row * p.rs + n) + d : d);
  }
}

// Columns of a block of rows, a thread each.
template <class T>
__global__ void __launch_bounds__(256) bwd_any_columns(const BwdP<T> p, int64_t M, int64_t R) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (n >= p.N) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * R, r1 = min(M, r0 + R);
  float dw = 0.f, db = 0.f;
  for (int64_t row = r0; row < r1; ++row) {
    const float g = get(p.dy + row * p.ys + n);
    dw = fmaf(g, (get(p.x + row * p.xs + n) - p.mean[row]) * p.rstd[row], dw);
    db += g;
  }
  float* to = p.partials + static_cast<int64_t>(blockIdx.y) * (p.want_dw + p.want_db) * p.N;
  if (p.want_dw) to[n] = dw;
  if (p.want_db) to[(p.want_dw ? p.N : 0) + n] = db;
}

// The G rows of [G, columns] partials added in a fixed order: 32 columns a
// block, warp w adds the rows w, w + 32, ..., then the warps' sums in order.  The
// first N columns go to `first`, the others to `second`.
__global__ void __launch_bounds__(1024) add_partials(const float* __restrict__ partials, int64_t G, int64_t columns,
                                                      int64_t N, float* first, float* second) {
  __shared__ float red[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float a = 0.f;
  if (col < columns) {
    for (int64_t g0 = warp; g0 < G; g0 += 32 * 16) {
      float v[16];  // one round trip for up to 512 rows
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = g0 + 32 * j < G ? partials[(g0 + 32 * j) * columns + col] : 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) a += v[j];
    }
  }
  red[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && col < columns) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) s += red[w][lane];
    if (col < N) first[col] = s;
    else second[col - N] = s;
  }
}

int launch_add_partials(const float* partials, int64_t G, int64_t N, float* dw, float* db, cudaStream_t s) {
  const int64_t columns = ((dw ? 1 : 0) + (db ? 1 : 0)) * N;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ceil_div(columns, 32)));
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, add_partials, partials, G, columns, N, dw ? dw : db, db));
}

// Blocks of rows that the columns' sums are split over, at most.
int64_t row_blocks() {
  const int sms = sm_count();
  return static_cast<int64_t>(sms > 0 ? sms : 148) * 4;
}

template <class T>
int forward(const FwdP<T>& p, int64_t M, cudaStream_t s) {
  fwd_any<T><<<dim3(static_cast<unsigned>(M)), 256, 0, s>>>(p);
  return check_launch();
}

template <class T>
int backward(const BwdP<T>& p, int64_t M, float* dw, float* db, cudaStream_t s) {
  bwd_any_dx<T><<<dim3(static_cast<unsigned>(M)), 256, 0, s>>>(p);
  if (int st = check_launch(); st != FRAG_OK || (!dw && !db)) return st;
  const int64_t R = ceil_div(M, std::min(M, row_blocks())), G = ceil_div(M, R);
  const dim3 grid(static_cast<unsigned>(ceil_div(p.N, 256)), static_cast<unsigned>(G));
  bwd_any_columns<T><<<grid, 256, 0, s>>>(p, M, R);
  if (int st = check_launch(); st != FRAG_OK) return st;
  return launch_add_partials(p.partials, G, p.N, dw, db, s);
}

bool known(int dtype) { return dtype == FRAG_DT_BF16 || dtype == FRAG_DT_F32; }
bool whole(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == FRAG_DT_F32 ? 4 : 2) == 0; }

}  // namespace
}  // namespace frag

using namespace frag;

extern "C" {

int frag_layernorm_fwd(const void* x, int64_t x_stride, const void* res, int64_t res_stride, const void* w,
                       const void* b, void* y, void* h, float* mean, float* rstd, int64_t M, int64_t N, float eps,
                       int dtype, int wdtype, frag_stream_t stream) {
  if (M < 0 || N < 0 || !known(dtype) || !known(wdtype)) return FRAG_ERR_INVALID_ARG;
  if (M == 0) return FRAG_OK;
  if (N == 0 || M > 0x7fffffffLL || N > (1LL << 31)) return FRAG_ERR_SHAPE;
  if (!x || !y || (h && !res)) return FRAG_ERR_INVALID_ARG;
  if (!whole(x, dtype) || !whole(res, dtype) || !whole(y, dtype) || !whole(h, dtype) || !whole(w, wdtype) ||
      !whole(b, wdtype))
    return FRAG_ERR_ALIGN;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Vector wv = {w, wdtype == FRAG_DT_F32}, bv = {b, wdtype == FRAG_DT_F32};
  if (dtype == FRAG_DT_F32)
    return forward<float>({static_cast<const float*>(x), static_cast<const float*>(res), static_cast<float*>(y),
                           static_cast<float*>(h), wv, bv, mean, rstd, x_stride, res_stride, N, eps},
                          M, s);
  return forward<uint16_t>({static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(res),
                            static_cast<uint16_t*>(y), static_cast<uint16_t*>(h), wv, bv, mean, rstd, x_stride,
                            res_stride, N, eps},
                           M, s);
}

size_t frag_layernorm_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 0;
  return align_up(static_cast<size_t>(std::min(M, row_blocks())) * 2 * N * sizeof(float), 256);
}

int frag_layernorm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                       const float* rstd, const void* w, const void* dres, int64_t dres_stride, void* dx, float* dw,
                       float* db, int64_t M, int64_t N, int dtype, int wdtype, void* workspace,
                       size_t workspace_bytes, frag_stream_t stream) {
  if (M < 0 || N < 0 || !known(dtype) || !known(wdtype)) return FRAG_ERR_INVALID_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (M == 0) {
    cudaError_t e = cudaSuccess;
    if (dw && N) e = cudaMemsetAsync(dw, 0, N * sizeof(float), s);
    if (db && N && e == cudaSuccess) e = cudaMemsetAsync(db, 0, N * sizeof(float), s);
    return cuda_status(e);
  }
  if (N == 0 || M > 0x7fffffffLL || N > (1LL << 31)) return FRAG_ERR_SHAPE;
  if (!dy || !x || !mean || !rstd || !dx) return FRAG_ERR_INVALID_ARG;
  if (!whole(dy, dtype) || !whole(x, dtype) || !whole(dres, dtype) || !whole(dx, dtype) || !whole(w, wdtype))
    return FRAG_ERR_ALIGN;
  if (dw || db) {
    if (!workspace || workspace_bytes < frag_layernorm_bwd_workspace_bytes(M, N)) return FRAG_ERR_WORKSPACE;
    if (!aligned16(workspace)) return FRAG_ERR_ALIGN;
  }
  const Vector wv = {w, wdtype == FRAG_DT_F32};
  float* ws = static_cast<float*>(workspace);
  if (dtype == FRAG_DT_F32)
    return backward<float>({static_cast<const float*>(dy), static_cast<const float*>(x),
                            static_cast<const float*>(dres), static_cast<float*>(dx), wv, mean, rstd, ws, dy_stride,
                            x_stride, dres_stride, N, dw != nullptr, db != nullptr},
                           M, dw, db, s);
  return backward<uint16_t>({static_cast<const uint16_t*>(dy), static_cast<const uint16_t*>(x),
                             static_cast<const uint16_t*>(dres), static_cast<uint16_t*>(dx), wv, mean, rstd, ws,
                             dy_stride, x_stride, dres_stride, N, dw != nullptr, db != nullptr},
                            M, dw, db, s);
}

}  // extern "C"

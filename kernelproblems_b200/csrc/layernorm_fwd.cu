// layernorm_fwd.cu — (residual add +) layer norm.
#include "layernorm.cuh"

namespace frag {
namespace {

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

// A chunk of h.
template <class T, bool RES>
__device__ __forceinline__ void input_chunk(const uint4& x, const uint4& res, float2* v) {
  if (RES && sizeof(T) == 2) {
    unpack<T>(add_bf16x8(res, x), v);
  } else {
    unpack<T>(x, v);
    if (RES) {
      float2 r[kP<T>];
      unpack<T>(res, r);
#pragma unroll
      for (int q = 0; q < kP<T>; ++q) v[q] = __fadd2_rn(r[q], v[q]);
    }
  }
}

// Sum of the squared distances from `mean` of the values inside the row.
template <class T, int V, Mode MODE>
__device__ __forceinline__ float row_squares(const Places<T, MODE>& at, int N, const float2 (&v)[V / 2], float mean) {
  float2 s = twice(0.f);
  const float2 m = twice(-mean);
#pragma unroll
  for (int k = 0; k < V / kE<T>; ++k) {
    if (!at[k].some(N)) continue;
    float2 d[kP<T>];
#pragma unroll
    for (int q = 0; q < kP<T>; ++q) d[q] = __fadd2_rn(v[k * kP<T> + q], m);
    own_values<T, MODE>(at[k], N, 0.f, d);
#pragma unroll
    for (int q = 0; q < kP<T>; ++q) s = __ffma2_rn(d[q], d[q], s);
  }
  return s.x + s.y;
}

// A chunk of y.
template <class T, Mode MODE>
__device__ __forceinline__ void write_chunk(T* row, const Place<T, MODE>& at, int N, const float2* v, float mean,
                                            float r, const float2* w, const float2* b) {
  float2 y[kP<T>];
#pragma unroll
  for (int q = 0; q < kP<T>; ++q)
    y[q] = __ffma2_rn(__fmul2_rn(__fadd2_rn(v[q], twice(-mean)), twice(r)), w[q], b[q]);
  store_chunk<T, MODE>(row, at, N, y);
}

// Rows of up to 512 values: L lanes a row, V values a lane, no barrier.  Groups
// of lanes stay within a class, with the weights in registers; each thread keeps
// its own chunks of the next rows in flight, kAhead of them, into its own places in
// shared memory, so nothing has to be waited for but its own copies.

template <class T, int V, int L, Mode MODE, bool RES>
__global__ void __launch_bounds__(256, lane_blocks(V, MODE, 4)) fwd_lanes(const FwdP<T> p, const Rows rows) {
  constexpr int E = kE<T>, P = kP<T>, K = V / E, ROW = (RES ? 2 : 1) * K;
  extern __shared__ __align__(16) uint4 held[];  // [kAhead][ROW][256]
  const int N = static_cast<int>(p.N);
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (256 / L);  // a multiple of the classes
  int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int off = MODE == EDGE ? static_cast<int>((rows.off + row % rows.classes * N) % E) : 0;
  const int t = threadIdx.x % L;
  const Places<T, MODE> at = {t, L, off};
  auto ask = [&](int64_t r, int s) {
    uint4* to = held + s * (ROW * 256) + threadIdx.x;
    if (r < rows.M) {
      ask_row<T, K, MODE>({p.x, p.xs}, r, rows.M, at, N, to);
      if (RES) ask_row<T, K, MODE>({p.res, p.rs}, r, rows.M, at, N, to + K * 256);
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < kAhead - 1; ++s) ask(row + s * groups, s);
  float2 w[V / 2], b[V / 2];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_vector<T, MODE>(p.w, at[k], N, 1.f, w + k * P);
    load_vector<T, MODE>(p.b, at[k], N, 0.f, b + k * P);
  }
  const float invN = 1.0f / static_cast<float>(N);
  int s = 0;
  // (the lanes of a warp stay together: shuffles are the whole warp's)
  for (int64_t lead = row - (threadIdx.x & 31) / L; lead < rows.M; lead += groups, row += groups) {
    ask(row + (kAhead - 1) * groups, (s + kAhead - 1) % kAhead);
    copies_wait<kAhead - 1>();
    const uint4* from = held + s * (ROW * 256) + threadIdx.x;
    s = (s + 1) % kAhead;
    const bool in = row < rows.M;
    float2 v[V / 2], sum = twice(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) {
#pragma unroll
        for (int q = 0; q < P; ++q) v[k * P + q] = twice(0.f);
        continue;
      }
      const uint4 none = make_uint4(0, 0, 0, 0);
      input_chunk<T, RES>(from[k * 256], RES ? from[(K + k) * 256] : none, v + k * P);
      own_values<T, MODE>(at[k], N, 0.f, v + k * P);
#pragma unroll
      for (int q = 0; q < P; ++q) sum = __fadd2_rn(sum, v[k * P + q]);
      if (RES && p.h && in) store_chunk<T, MODE>(p.h + row * p.N, at[k], N, v + k * P);
    }
    const float mean = lanes_sum<L>(sum.x + sum.y) * invN;
    const float r = rsqrtf(fmaf(lanes_sum<L>(row_squares<T, V, MODE>(at, N, v, mean)), invN, p.eps));
    if (!in) continue;
    if (t == 0 && p.mean) p.mean[row] = mean;
    if (t == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
    for (int k = 0; k < K; ++k)
      write_chunk<T, MODE>(p.y + row * p.N, at[k], N, v + k * P, mean, r, w + k * P, b + k * P);
  }
}

// How many of a row's values each warp holds.
template <class T, int V>
__device__ __forceinline__ float warp_holds(int w, int off, int N) {
  int n = 0;
#pragma unroll
  for (int k = 0; k < V / kE<T>; ++k) {
    const int from = (k * static_cast<int>(blockDim.x) + w * 32) * kE<T>;
    n += max(0, min(from + 32 * kE<T>, off + N) - max(from, off));
  }
  return static_cast<float>(n);
}

// Wider rows: a block a row at a time, V = 16 values a thread, the next rows in
// the ring.  A row's mean and 1 / deviation behind one barrier: each warp takes
// its own mean and squares about it, and the warps' (count, sum, squares) are
// joined,
//   squares = sum over warps of squares_w + n_w (mean_w - mean)^2
// where two sums over the block, one after the other, would need two.  The weights
// stay in registers (at most 80, so that three blocks of 256 threads share an SM);
// WIDE, with more than 768 threads a block and 64 registers, they come from L1.
template <class T, int V, Mode MODE, bool RES, bool WIDE>
__device__ __forceinline__ void fwd_ring_body(const FwdP<T>& p, const Rows& rows, const RingShape& shape, int* err) {
  constexpr int P = kP<T>, K = V / kE<T>, INPUTS = RES ? 2 : 1;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float2 slots[2][32];
  __shared__ int s_abort;
  const int N = static_cast<int>(p.N), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  Ring<T, INPUTS, MODE> ring;
  ring.in[0] = {p.x, p.xs};
  if (RES) ring.in[INPUTS - 1] = {p.res, p.rs};
  deal(ring, rows, shape, smem, N);
  const Places<T, MODE> at = {static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x), ring.off};
  if (threadIdx.x == 0) {
    s_abort = 0;
    ring.begin();
  }
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 0; i < ring.S; ++i) ring.issue(i);
  float2 w[WIDE ? 1 : V / 2], b[WIDE ? 1 : V / 2];
  if constexpr (!WIDE) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      load_vector<T, MODE>(p.w, at[k], N, 1.f, w + k * P);
      load_vector<T, MODE>(p.b, at[k], N, 0.f, b + k * P);
    }
  }
  const float invN = 1.0f / static_cast<float>(N);
  const float mine = warp_holds<T, V>(warp, ring.off, N), of_lane = lane < nw ? warp_holds<T, V>(lane, ring.off, N) : 0.f;
  const float inv_mine = mine > 0.f ? 1.0f / mine : 0.f, inv_lane = of_lane > 0.f ? 1.0f / of_lane : 0.f;
  int i = 0;
  for (; i < ring.count; ++i) {
    const int64_t row = ring.row(i);
    if (!ring.wait(i, err)) s_abort = 1;
    float2 v[V / 2], sum = twice(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = threadIdx.x + k * blockDim.x;
      if (!at[k].some(N)) {
#pragma unroll
        for (int q = 0; q < P; ++q) v[k * P + q] = twice(0.f);
        continue;
      }
      const uint4 none = make_uint4(0, 0, 0, 0);
      input_chunk<T, RES>(ring.chunk(i, 0, c), RES ? ring.chunk(i, INPUTS - 1, c) : none, v + k * P);
      own_values<T, MODE>(at[k], N, 0.f, v + k * P);
#pragma unroll
      for (int q = 0; q < P; ++q) sum = __fadd2_rn(sum, v[k * P + q]);
      if (RES && p.h) store_chunk<T, MODE>(p.h + row * p.N, at[k], N, v + k * P);
    }
    const float ws = warp_sum(sum.x + sum.y);
    const float wq = warp_sum(row_squares<T, V, MODE>(at, N, v, ws * inv_mine));
    if (lane == 0) slots[i & 1][warp] = make_float2(ws, wq);
    __syncthreads();
    if (s_abort) break;
    if (threadIdx.x == 0) ring.issue(i + ring.S);  // every thread has its values of stage i % S
    const float2 o = lane < nw ? slots[i & 1][lane] : twice(0.f);
    const float mean = warp_sum(o.x) * invN;
    const float d = fmaf(o.x, inv_lane, -mean);
    const float r = rsqrtf(fmaf(warp_sum(fmaf(of_lane * d, d, o.y)), invN, p.eps));
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = r;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if constexpr (WIDE) {
        float2 wk[P], bk[P];
        load_vector<T, MODE>(p.w, at[k], N, 1.f, wk);
        load_vector<T, MODE>(p.b, at[k], N, 0.f, bk);
        write_chunk<T, MODE>(p.y + row * p.N, at[k], N, v + k * P, mean, r, wk, bk);
      } else {
        write_chunk<T, MODE>(p.y + row * p.N, at[k], N, v + k * P, mean, r, w + k * P, b + k * P);
      }
    }
  }
  if (threadIdx.x == 0 && s_abort) ring.drain(i);
}

template <class T, Mode MODE, bool RES>
__global__ void __maxnreg__(FWD_REGS) fwd_ring(const FwdP<T> p, const Rows rows, const RingShape shape, int* err) {
  fwd_ring_body<T, FWD_V, MODE, RES, false>(p, rows, shape, err);
}
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
    put(p.y + row * p.N + n, fmaf((h(n) - mean) * r, vector_at(p.w, n, 1.f), vector_at(p.b, n, 0.f)));
}

template <class T, int V, int L, Mode MODE, bool RES>
int launch_fwd_lanes(const FwdP<T>& p, const Rows& rows, cudaStream_t s) {
  const int per = 256 / L;  // a multiple of 8, as the classes are a divisor of 8
  const int smem = kAhead * (RES ? 2 : 1) * V * 256 * static_cast<int>(sizeof(T));
  auto kernel = fwd_lanes<T, V, L, MODE, RES>;
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return FRAG_ERR_CUDA;
  const int64_t resident = static_cast<int64_t>(sm_count()) * std::min(lane_blocks(V, MODE, 4), kSmem / (smem + 1024));
  kernel<<<dim3(static_cast<unsigned>(std::min(ceil_div(rows.M, per), resident))), 256, smem, s>>>(p, rows);
  return check_launch();
}

template <class T, int V, Mode MODE, bool RES>
int launch_fwd_ring(const FwdP<T>& p, Rows rows, int64_t held, cudaStream_t s) {
  auto kernel = fwd_ring<T, MODE, RES>;
  const int threads = static_cast<int>(ceil_div(held, 32 * V) * 32);
  RingShape shape;
  int smem = 0;
  const int64_t blocks = plan_ring(rows, shape, &smem, RES ? 2 : 1, static_cast<int>(ceil_div(held, kE<T>)) * 16,
                                   ring_blocks(threads, FWD_REGS));
  if (!blocks) return FRAG_ERR_SHAPE;
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return FRAG_ERR_CUDA;
  kernel<<<dim3(static_cast<unsigned>(blocks)), threads, smem, s>>>(p, rows, shape, device_error_word());
  return check_launch();
}

template <class T, Mode MODE, bool RES>
int launch_fwd(const FwdP<T>& p, const Rows& rows, int64_t held, cudaStream_t s) {
  if (held <= 64) return launch_fwd_lanes<T, 8, 8, MODE, RES>(p, rows, s);
  if (held <= 128) return launch_fwd_lanes<T, 8, 16, MODE, RES>(p, rows, s);
  if (held <= 256) return launch_fwd_lanes<T, 8, 32, MODE, RES>(p, rows, s);
  if (held <= kLanes) return launch_fwd_lanes<T, 16, 32, MODE, RES>(p, rows, s);
  return launch_fwd_ring<T, FWD_V, MODE, RES>(p, rows, held, s);
}

template <class T>
int forward(const FwdP<T>& p, int64_t M, cudaStream_t s) {
  Layout lay(p.N, sizeof(T));
  lay.add(p.x, p.xs);
  lay.add(p.res, p.rs);
  lay.add(p.y, p.N);
  lay.add(p.h, p.N);
  const bool edge = lay.off || lay.residue;
  const int64_t held = p.N + (edge ? kE<T> - 1 : 0);  // values of a row's chunks, at most
  if (!lay.alike || held > kHeld) {
    fwd_any<T><<<dim3(static_cast<unsigned>(M)), 256, 0, s>>>(p);
    return check_launch();
  }
  const Rows rows = {M, lay.off, lay.classes(), 1};
  const bool full = p.N == 64 || p.N == 128 || p.N == 256 || p.N == 512 || (p.N > 512 && p.N % (32 * FWD_V) == 0);
  return by_mode(edge, full, [&](auto mode) {
    constexpr Mode MODE = decltype(mode)::value;
    return p.res ? launch_fwd<T, MODE, true>(p, rows, held, s) : launch_fwd<T, MODE, false>(p, rows, held, s);
  });
}

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
  const Vector wv = {w, wdtype == FRAG_DT_F32, aligned16(w)}, bv = {b, wdtype == FRAG_DT_F32, aligned16(b)};
  if (dtype == FRAG_DT_F32)
    return forward<float>({static_cast<const float*>(x), static_cast<const float*>(res), static_cast<float*>(y),
                           static_cast<float*>(h), wv, bv, mean, rstd, x_stride, res_stride, N, eps},
                          M, s);
  return forward<uint16_t>({static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(res),
                            static_cast<uint16_t*>(y), static_cast<uint16_t*>(h), wv, bv, mean, rstd, x_stride,
                            res_stride, N, eps},
                           M, s);
}

}  // extern "C"

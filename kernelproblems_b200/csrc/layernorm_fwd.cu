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
  float2 s = twice(0.f), s2 = s;
  const float2 m = twice(-mean);
#pragma unroll
  for (int k = 0; k < V / kE<T>; ++k) {
    if (!at[k].some(N)) continue;
    float2 d[kP<T>];
#pragma unroll
    for (int q = 0; q < kP<T>; ++q) d[q] = __fadd2_rn(v[k * kP<T> + q], m);
    own_values<T, MODE>(at[k], N, 0.f, d);
#pragma unroll
    for (int q = 0; q < kP<T>; q += 2) {
      s = __ffma2_rn(d[q], d[q], s);
      s2 = __ffma2_rn(d[q + 1], d[q + 1], s2);
    }
  }
  s = __fadd2_rn(s, s2);
  return s.x + s.y;
}

// 1 / N as a number and what that leaves out, so that a quotient is rounded once: sum / N
// is not off by a place where it is a number of 32 bits, as in a row of equal values.
// (Of an infinity the quotient is NaN, as the row's outputs are; as_stored is what its mean
// is.)  Bf16 rows without a residual pay for it: 32768 of 8192 174 us, by the product with
// 1 / N alone 168.
struct Count {
  float inverse, rest;
  __device__ __forceinline__ explicit Count(int N) {
    inverse = 1.0f / static_cast<float>(N);
    rest = fmaf(-inverse, static_cast<float>(N), 1.0f) * inverse;
  }
  __device__ __forceinline__ float mean(float sum) const { return fmaf(sum, inverse, sum * rest); }
  __device__ __forceinline__ float as_stored(float mean, float sum) const {
    return isfinite(mean) ? mean : sum * inverse;
  }
};

// A mean that is many deviations is off by some of them if its sum is rounded: fp32 rows
// of 1001 values 1000.3 had deviations of 1.2e-4 in place of none.  So an fp32 row whose
// mean is more than 8 deviations adds up its distances from it, which have no digits to
// lose, and the mean becomes the true one but for its own rounding.  (8192 rows of 1001:
// 25 us, all of them far from zero 29; 32768 of 8192 332 both.)  The sum of up to 16384
// bf16 values that lie about a mean so far from zero is exact: 8 binary digits each and
// those of their count, 14, are less than 24.
__device__ __forceinline__ bool far_from_zero(float mean, float var) { return mean * mean > 64.f * var; }
__device__ __forceinline__ void correct(float& mean, float& var, float distances, float squares, float invN) {
  const float off = distances * invN;
  var = fmaxf(fmaf(squares, invN, -off * off), 0.f);
  mean += off;
}
// Sums of the distances from `mean`, and of their squares, of the values inside the row.
template <class T, int V, Mode MODE>
__device__ __forceinline__ float2 row_distances(const Places<T, MODE>& at, int N, const float2 (&v)[V / 2], float mean) {
  float2 a = twice(0.f), s = a;
#pragma unroll
  for (int k = 0; k < V / kE<T>; ++k) {
    if (!at[k].some(N)) continue;
    float2 d[kP<T>];
#pragma unroll
    for (int q = 0; q < kP<T>; ++q) d[q] = __fadd2_rn(v[k * kP<T> + q], twice(-mean));
    own_values<T, MODE>(at[k], N, 0.f, d);
#pragma unroll
    for (int q = 0; q < kP<T>; ++q) {
      a = __fadd2_rn(a, d[q]);
      s = __ffma2_rn(d[q], d[q], s);
    }
  }
  return make_float2(a.x + a.y, s.x + s.y);
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
// shared memory, so nothing has to be waited for but its own copies.  Issue bounds
// them (two thirds of the slots): 262144 rows of 128 in bf16 27.9 us, 4.8 TB/s, of
// a million 98, 5.5.  Odd widths (129: 78 us) pay
// for shifts, for masks, and at a row's ends for stores of single values.
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
  Bits<T, MODE> own[K];
#pragma unroll
  for (int k = 0; k < K; ++k) own[k].set(at[k], N);
  Walk<T> x({p.x, p.xs}, row, groups), res({RES ? p.res : p.x, p.rs}, row, groups);
  int64_t asked = row;
  auto ask = [&](int s) {
    uint4* to = held + s * (ROW * 256) + threadIdx.x;
    if (asked < rows.M) {
      const bool end = asked == 0 || asked == rows.M - 1;
      x.template ask<K, MODE>(at, N, end, to);
      if (RES) res.template ask<K, MODE>(at, N, end, to + K * 256);
    }
    copies_commit();
    asked += groups;
    x.next += x.jump;
    if (RES) res.next += res.jump;
  };
#pragma unroll
  for (int s = 0; s < kAhead - 1; ++s) ask(s);
  float2 w[V / 2], b[V / 2];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_vector<T, MODE>(p.w, at[k], N, 1.f, w + k * P);
    load_vector<T, MODE>(p.b, at[k], N, 0.f, b + k * P);
  }
  const Count count(N);
  const float invN = count.inverse;
  int s = 0;
  T *y = p.y + row * p.N, *h = p.h + row * p.N;
  const int64_t jump = groups * p.N;
  // (the lanes of a warp stay together: shuffles are the whole warp's)
  for (int64_t lead = row - (threadIdx.x & 31) / L; lead < rows.M; lead += groups, row += groups, y += jump, h += jump) {
    ask(s == 0 ? kAhead - 1 : s - 1);
    copies_wait<kAhead - 1>();
    const uint4* from = held + s * (ROW * 256) + threadIdx.x;
    s = s == kAhead - 1 ? 0 : s + 1;
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
      input_chunk<T, RES>(own[k](from[k * 256]), RES ? own[k](from[(K + k) * 256]) : none, v + k * P);
#pragma unroll
      for (int q = 0; q < P; ++q) sum = __fadd2_rn(sum, v[k * P + q]);
      if (RES && p.h && in) store_chunk<T, MODE>(h, at[k], N, v + k * P);
    }
    const float all = lanes_sum<L>(sum.x + sum.y);
    float mean = count.mean(all);
    float var = lanes_sum<L>(row_squares<T, V, MODE>(at, N, v, mean)) * invN;
    if constexpr (sizeof(T) == 4) {
      const bool far = far_from_zero(mean, var);
      if (__any_sync(0xffffffffu, far)) {  // (shuffles are the whole warp's)
        float2 d = row_distances<T, V, MODE>(at, N, v, mean);
        d = make_float2(lanes_sum<L>(d.x), lanes_sum<L>(d.y));
        if (far) correct(mean, var, d.x, d.y, invN);
      }
    }
    const float r = rsqrtf(var + p.eps);
    if (!in) continue;
    if (t == 0 && p.mean) p.mean[row] = count.as_stored(mean, all);
    if (t == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
    for (int k = 0; k < K; ++k)
      write_chunk<T, MODE>(y, at[k], N, v + k * P, mean, r, w + k * P, b + k * P);
  }
}

// How many of a row's values warp w of a group holds.
template <class T>
__device__ __forceinline__ float warp_holds(int w, int threads, int off, int N) {
  int n = 0;
#pragma unroll
  for (int k = 0; k < kV / kE<T>; ++k) {
    const int from = (k * threads + w * 32) * kE<T>;
    n += max(0, min(from + 32 * kE<T>, off + N) - max(from, off));
  }
  return static_cast<float>(n);
}

// Threads of a block (80 registers each): 512, and where that is one group only (rows
// above 8192 values), 768.  32768 rows of 8192 in bf16 169 us with 512, 179 with 768;
// 8192 of 12288 79 and 76, with the residual 154 and 141.
constexpr int kMost = 768;
// Bytes of rows in flight on an SM.  More of them are slower, as the reads then hold
// up the writes: 32768 rows of 8192 in bf16 168 us with 64 KB, 194 with 96 and
// more; with the residual 335 with 64 KB, 370 with 128 and more.
constexpr int kFlight = 65536;

// Wider rows, a group a row at a time.  A row's mean and 1 / deviation behind one
// barrier: each warp takes its own mean and squares about it, and the warps'
// (count, sum, squares) are joined,
//   squares = sum over warps of squares_w + n_w (mean_w - mean)^2
// where two sums over the group, one after the other, would need two.
//
// Bound: HBM, beside some 5 us to start and to end.  In bf16 8192 rows of 4096 take
// 26.5 us (5.1 TB/s) and 32768 of 8192 174 (6.2, 0.94 of a copy's rate), with the
// residual 46 and 335.  A block for each row, its weights read again from L2 each
// time, took 382 for the last; 1024 threads with 64 registers
// were slower too.
template <class T, class W, Mode MODE, bool RES>
__global__ void __launch_bounds__(kMost) fwd_groups(const FwdP<T> p, const Rows rows, const Shape shape, int* err) {
  constexpr int P = kP<T>, V = kV, K = V / kE<T>, INPUTS = RES ? 2 : 1;
  extern __shared__ __align__(128) unsigned char smem[];  // w, b, the rings
  __shared__ float2 slots[2][32], counts[16];             // (sum, squares) and (n, 1 / n) of each warp
  __shared__ float2 distances[32];                        // of each warp, where a row is far from zero
  __shared__ Gave gave;
  const int N = static_cast<int>(p.N), lane = threadIdx.x & 31, nw = shape.threads >> 5;
  const Group g(shape.threads);
  const int apart = shape.threads * V, warp = g.t >> 5;
  W *w = reinterpret_cast<W*>(smem), *b = w + apart;
  Ring<T, INPUTS, MODE> ring;
  ring.in[0] = {p.x, p.xs};
  if (RES) ring.in[INPUTS - 1] = {p.res, p.rs};
  deal(ring, rows, shape, g.index, smem + 2 * sizeof(W) * apart, N);
  const Places<T, MODE> at = {g.t, g.threads, ring.off};
  if (g.t == 0) {
    gave.begin(g);
    ring.begin();
    for (int i = 0; i < ring.S; ++i) ring.issue();
  }
  if (static_cast<int>(threadIdx.x) < nw) {
    const float n = warp_holds<T>(threadIdx.x, g.threads, ring.off, N);
    counts[threadIdx.x] = make_float2(n, n > 0.f ? 1.0f / n : 0.f);
  }
  share_vector<T, W, MODE>(p.w, 1.f, w, apart, ring.off, N);
  share_vector<T, W, MODE>(p.b, 0.f, b, apart, ring.off, N);
  __syncthreads();
  const Count count(N);
  const float invN = count.inverse, inv_mine = counts[warp].y;
  const int first = g.index * nw;  // the group's slots
  int64_t row = ring.r0;
  int i = 0;
  for (; i < ring.count; ++i, row += ring.step) {
    if (!ring.wait(err)) gave.up(g, i);
    float2 v[V / 2], sum = twice(0.f), sum2 = sum;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = g.t + k * g.threads;
      if (!at[k].some(N)) {
#pragma unroll
        for (int q = 0; q < P; ++q) v[k * P + q] = twice(0.f);
        continue;
      }
      const uint4 none = make_uint4(0, 0, 0, 0);
      input_chunk<T, RES>(ring.chunk(0, c), RES ? ring.chunk(INPUTS - 1, c) : none, v + k * P);
      own_values<T, MODE>(at[k], N, 0.f, v + k * P);
#pragma unroll
      for (int q = 0; q < P; q += 2) {
        sum = __fadd2_rn(sum, v[k * P + q]);
        sum2 = __fadd2_rn(sum2, v[k * P + q + 1]);
      }
      if (RES && p.h) store_chunk<T, MODE>(p.h + row * p.N, at[k], N, v + k * P);
    }
    sum = __fadd2_rn(sum, sum2);
    const float ws = warp_sum(sum.x + sum.y);
    const float wq = warp_sum(row_squares<T, V, MODE>(at, N, v, ws * inv_mine));
    if (lane == 0) slots[i & 1][first + warp] = make_float2(ws, wq);
    g.sync();
    if (gave.is_up(g, i)) break;
    if (g.t == 0) ring.issue();  // every thread has its values of this stage
    float all = ws, var = wq * invN;
    if (nw > 1) {  // (16 lanes take a warp each, the upper half the same again)
      const int of = lane & 15;
      const float2 o = of < nw ? slots[i & 1][first + of] : twice(0.f), n = of < nw ? counts[of] : twice(0.f);
      all = lanes_sum<16>(o.x);
      const float d = fmaf(o.x, n.y, -all * invN);
      var = lanes_sum<16>(fmaf(n.x * d, d, o.y)) * invN;
    }
    float mean = count.mean(all);
    if (sizeof(T) == 4 && far_from_zero(mean, var)) {  // (the whole group: its warps have the same sums)
      const float2 d = warp_sum2(row_distances<T, V, MODE>(at, N, v, mean));
      if (lane == 0) distances[first + warp] = d;
      g.sync();
      const int of = lane & 15;
      const float2 o = of < nw ? distances[first + of] : twice(0.f);
      correct(mean, var, lanes_sum<16>(o.x), lanes_sum<16>(o.y), invN);
    }
    const float r = rsqrtf(var + p.eps);
    if (g.t == 0) {
      if (p.mean) p.mean[row] = count.as_stored(mean, all);
      if (p.rstd) p.rstd[row] = r;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) continue;
      float2 wk[P], bk[P];
      shared_chunk<T, W>(w, apart, g.t + k * g.threads, wk);
      shared_chunk<T, W>(b, apart, g.t + k * g.threads, bk);
      write_chunk<T, MODE>(p.y + row * p.N, at[k], N, v + k * P, mean, r, wk, bk);
    }
    ring.next();
  }
  if (g.t == 0 && i < ring.count) ring.drain(i);
}

// Any width, any alignment (rows above 16384 values, or tensors whose rows begin at
// different places between 16-byte boundaries): a block a row, the row read once
// for each pass, the later ones from L2.
template <class T, bool RES>
__global__ void __launch_bounds__(256) fwd_any(const FwdP<T> p) {
  __shared__ float2 slots[2][32];
  const int64_t row = blockIdx.x;
  const T* x = p.x + row * p.xs;
  const T* res = RES ? p.res + row * p.rs : nullptr;
  auto h = [&](int64_t n) { return RES ? rounded<T>(get(res + n) + get(x + n)) : get(x + n); };
  const float N = static_cast<float>(p.N);
  float mean = block_sum2(long_sums(p.N, [&](int64_t n) {
                            const float v = h(n);
                            if (RES && p.h) put(p.h + row * p.N + n, v);
                            return make_float2(v, 0.f);
                          }), slots, 0).x / N;
  auto distances = [&](int64_t n) {
    const float v = h(n) - mean;
    return make_float2(v, v * v);
  };
  float2 d = block_sum2(long_sums(p.N, distances), slots, 1);
  float var = d.y / N;
  if (far_from_zero(mean, var)) correct(mean, var, d.x, d.y, 1.0f / N);
  const float r = rsqrtf(var + p.eps);
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

// Returns -1, nothing launched, where a row's stage does not fit in shared memory.
template <class T, class W, Mode MODE, bool RES>
int launch_fwd_groups(const FwdP<T>& p, const Rows& rows, int64_t held, cudaStream_t s) {
  auto kernel = fwd_groups<T, W, MODE, RES>;
  Shape shape;
  int smem = 0;
  const int64_t blocks = plan_groups(rows, held, sizeof(T), RES ? 2 : 1, 2, sizeof(W), held > 8 * 32 * kV ? kMost : 512, 1,
                                     kFlight, shape, &smem);
  if (!blocks) return -1;
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return FRAG_ERR_CUDA;
  kernel<<<dim3(static_cast<unsigned>(blocks)), shape.groups * shape.threads, smem, s>>>(p, rows, shape,
                                                                                          device_error_word());
  return check_launch();
}

template <class T, Mode MODE, bool RES>
int launch_fwd(const FwdP<T>& p, const Rows& rows, int64_t held, cudaStream_t s) {
  constexpr Mode LANES = MODE == FULL ? PART : MODE;
  if (held <= 64) return launch_fwd_lanes<T, 8, 8, LANES, RES>(p, rows, s);
  if (held <= 128) return launch_fwd_lanes<T, 8, 16, LANES, RES>(p, rows, s);
  if (held <= 256) return launch_fwd_lanes<T, 8, 32, LANES, RES>(p, rows, s);
  if (held <= kLanes) return launch_fwd_lanes<T, 16, 32, LANES, RES>(p, rows, s);
  return by_weight<T>(p.w, p.b, [&](auto w) { return launch_fwd_groups<T, decltype(w), MODE, RES>(p, rows, held, s); });
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
  if (lay.alike && held <= kHeld) {
    const Rows rows = {M, lay.off, lay.classes()};
    const int st = by_mode(edge, p.N % (32 * kV) == 0, [&](auto mode) {
      constexpr Mode MODE = decltype(mode)::value;
      return p.res ? launch_fwd<T, MODE, true>(p, rows, held, s) : launch_fwd<T, MODE, false>(p, rows, held, s);
    });
    if (st >= 0) return st;
  }
  auto any = p.res ? fwd_any<T, true> : fwd_any<T, false>;
  any<<<dim3(static_cast<unsigned>(M)), 256, 0, s>>>(p);
  return check_launch();
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
  if (sm_count() <= 0) return FRAG_ERR_NO_DEVICE;
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

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
  int f32, aligned;
};
__device__ __forceinline__ float vector_at(const Vector& v, int64_t n, float none) {
  if (!v.p) return none;
  return v.f32 ? static_cast<const float*>(v.p)[n] : bf16_to_f(static_cast<const uint16_t*>(v.p)[n]);
}

// ------------------------------------------------------- rows in 16-byte chunks
//
// A row is cut at the 16-byte boundaries of memory into chunks of E values.  Its
// first value lies `off` values behind a boundary, so chunk c holds the columns
// c E - off to c E - off + E - 1, the first and last chunk part of them.  Rows of
// all tensors of a call have the same off, or the call takes the kernels for any
// alignment.  With rows of N values off comes again every P = E / gcd(N, E) rows:
// rows r with the same r % P are a class, and who stays within a class keeps
// fixed columns, so weights and sums over rows stay in registers for odd
// widths too.  EDGE: off or N is not a multiple of E (otherwise P = 1, off = 0).

template <class T>
constexpr int kE = 16 / sizeof(T);

template <class T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  if (sizeof(T) == 2) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f[2 * q] = bf16lo(u4_word(v, q));
      f[2 * q + 1] = bf16hi(u4_word(v, q));
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) f[q] = __uint_as_float(u4_word(v, q));
  }
}
template <class T>
__device__ __forceinline__ uint4 pack(const float* f) {
  if (sizeof(T) == 2)
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4 % kE<T>], f[5 % kE<T>]),
                      pack_bf16x2(f[6 % kE<T>], f[7 % kE<T>]));
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

// Where a thread's chunk lies in its row.
template <class T, bool EDGE>
struct Place {
  int n0;  // its first column
  __device__ __forceinline__ Place(int c, int off) : n0(c * kE<T> - (EDGE ? off : 0)) {}
  __device__ __forceinline__ bool some(int N) const { return n0 < N; }
  __device__ __forceinline__ bool all(int N) const { return EDGE ? n0 >= 0 && n0 + kE<T> <= N : n0 < N; }
  __device__ __forceinline__ bool has(int i, int N) const { return !EDGE || static_cast<unsigned>(n0 + i) < static_cast<unsigned>(N); }
};

// The chunk of a row that begins at `row`, zeros outside.
template <class T, bool EDGE>
__device__ __forceinline__ uint4 load_chunk(const T* row, const Place<T, EDGE>& at, int N) {
  if (at.all(N)) return ld_stream(row + at.n0);
  uint4 v = make_uint4(0, 0, 0, 0);
  if (EDGE && at.some(N)) {
    float f[kE<T>];
#pragma unroll
    for (int i = 0; i < kE<T>; ++i) f[i] = at.has(i, N) ? get(row + at.n0 + i) : 0.f;
    v = pack<T>(f);
  }
  return v;
}
template <class T, bool EDGE>
__device__ __forceinline__ void store_chunk(T* row, const Place<T, EDGE>& at, int N, const float* f) {
  if (at.all(N)) {
    st_global(row + at.n0, pack<T>(f));
  } else if (EDGE && at.some(N)) {
#pragma unroll
    for (int i = 0; i < kE<T>; ++i)
      if (at.has(i, N)) put(row + at.n0 + i, f[i]);
  }
}
// A vector's values at a chunk's columns.
template <class T, bool EDGE>
__device__ __forceinline__ void load_vector(const Vector& v, const Place<T, EDGE>& at, int N, float none, float* f) {
  constexpr int E = kE<T>;
  if (v.p && !EDGE && v.aligned && at.some(N)) {
    if (v.f32) {
#pragma unroll
      for (int q = 0; q < E / 4; ++q)
        unpack<float>(ld_cached(static_cast<const float*>(v.p) + at.n0 + 4 * q), f + 4 * q);
    } else if (E == 8) {
      unpack<uint16_t>(ld_cached(static_cast<const uint16_t*>(v.p) + at.n0), f);
    } else {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(v.p) + at.n0));
      f[0] = bf16lo(u.x);
      f[1] = bf16hi(u.x);
      f[2] = bf16lo(u.y);
      f[3] = bf16hi(u.y);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) f[i] = at.some(N) && at.has(i, N) ? vector_at(v, at.n0 + i, none) : 0.f;
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

// Blocks of 256 threads for rows of lanes, per SM.
constexpr int kLaneBlocks = 4;

// How a launch's rows are dealt out.
struct Rows {
  int64_t M;
  int off;      // of row 0
  int classes;  // P
  int64_t each;  // rows of a class that a block takes
};

// Sum over groups of L neighbouring lanes.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Row of h: V values a thread in chunks of E, and where those lie.
template <class T, int V, bool EDGE>
struct RowPlaces {
  int first, step, off;
  __device__ __forceinline__ Place<T, EDGE> operator[](int k) const { return Place<T, EDGE>(first + k * step, off); }
};

template <class T, int V, bool EDGE, bool RES>
__device__ __forceinline__ void load_row(const FwdP<T>& p, int64_t row, const RowPlaces<T, V, EDGE>& at, int N,
                                         uint4 (&xv)[V / kE<T>], uint4 (&rv)[V / kE<T>]) {
#pragma unroll
  for (int k = 0; k < V / kE<T>; ++k) {
    xv[k] = load_chunk<T, EDGE>(p.x + row * p.xs, at[k], N);
    if (RES) rv[k] = load_chunk<T, EDGE>(p.res + row * p.rs, at[k], N);
  }
}

// h's values (zeros outside the row), written where it is wanted; returns their sum.
template <class T, int V, bool EDGE, bool RES>
__device__ __forceinline__ float row_values(const FwdP<T>& p, int64_t row, const RowPlaces<T, V, EDGE>& at, int N,
                                            const uint4 (&xv)[V / kE<T>], const uint4 (&rv)[V / kE<T>],
                                            float (&v)[V]) {
  constexpr int E = kE<T>;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < V / E; ++k) {
    if (RES && sizeof(T) == 2) {
      unpack<T>(add_bf16x8(rv[k], xv[k]), v + k * E);
    } else {
      unpack<T>(xv[k], v + k * E);
      if (RES) {
        float r[E];
        unpack<T>(rv[k], r);
#pragma unroll
        for (int i = 0; i < E; ++i) v[k * E + i] += r[i];
      }
    }
    if (RES && p.h) store_chunk<T, EDGE>(p.h + row * p.N, at[k], N, v + k * E);
#pragma unroll
    for (int i = 0; i < E; ++i) s += v[k * E + i];
  }
  return s;
}

// Sum of the squared distances from `mean` of the values inside the row.
template <class T, int V, bool EDGE>
__device__ __forceinline__ float row_squares(const RowPlaces<T, V, EDGE>& at, int N, const float (&v)[V], float mean) {
  constexpr int E = kE<T>;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < V / E; ++k) {
    const Place<T, EDGE> a = at[k];
    if (a.all(N)) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float d = v[k * E + i] - mean;
        s = fmaf(d, d, s);
      }
    } else if (EDGE && a.some(N)) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float d = a.has(i, N) ? v[k * E + i] - mean : 0.f;
        s = fmaf(d, d, s);
      }
    }
  }
  return s;
}

// A row for each L lanes, up to V values a lane: no barrier.  Groups of lanes
// stay, with the weights in registers and the next row's loads in flight.
template <class T, int V, int L, bool EDGE, bool RES>
__global__ void __launch_bounds__(256) fwd_lanes(const FwdP<T> p, const Rows rows) {
  constexpr int E = kE<T>, K = V / E;
  const int N = static_cast<int>(p.N);
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (256 / L);  // a multiple of the classes
  int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int off = EDGE ? static_cast<int>((rows.off + row % rows.classes * N) % E) : 0;
  const int t = threadIdx.x % L;
  const RowPlaces<T, V, EDGE> at = {t, L, off};
  uint4 xv[K], rv[K];
  if (row < rows.M) load_row<T, V, EDGE, RES>(p, row, at, N, xv, rv);
  float w[V], b[V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_vector<T, EDGE>(p.w, at[k], N, 1.f, w + k * E);
    load_vector<T, EDGE>(p.b, at[k], N, 0.f, b + k * E);
  }
  const float invN = 1.0f / static_cast<float>(N);
  // (the lanes of a warp stay together: shuffles are the whole warp's)
  for (int64_t lead = row - (threadIdx.x & 31) / L; lead < rows.M; lead += groups, row += groups) {
    const bool in = row < rows.M;
    float v[V];
    if (!in) {
#pragma unroll
      for (int k = 0; k < K; ++k) xv[k] = rv[k] = make_uint4(0, 0, 0, 0);
    }
    float s;
    if (in) s = row_values<T, V, EDGE, RES>(p, row, at, N, xv, rv, v);
    else s = 0.f;
    if (row + groups < rows.M) load_row<T, V, EDGE, RES>(p, row + groups, at, N, xv, rv);
    const float mean = lanes_sum<L>(s) * invN;
    s = in ? row_squares<T, V, EDGE>(at, N, v, mean) : 0.f;
    const float r = rsqrtf(fmaf(lanes_sum<L>(s), invN, p.eps));
    if (!in) continue;
    if (t == 0 && p.mean) p.mean[row] = mean;
    if (t == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[k * E + i] = fmaf((v[k * E + i] - mean) * r, w[k * E + i], b[k * E + i]);
      store_chunk<T, EDGE>(p.y + row * p.N, at[k], N, v + k * E);
    }
  }
}

// The mean and 1 / deviation of a row whose block's threads hold sums and
// values: each warp takes its own mean and squares about it, and the warps'
// (count, sum, squares) are joined behind one barrier,
//   squares = sum over warps of squares_w + n_w (mean_w - mean)^2
// which two sums over the block, one after the other, would need two for.
template <class T, int V, bool EDGE>
__device__ __forceinline__ float2 block_stats(const RowPlaces<T, V, EDGE>& at, int N, const float (&v)[V], float s,
                                              float eps, float2 (*slots)[32], int parity) {
  constexpr int E = kE<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  // how many of the row's values warp w holds
  auto held = [&](int w) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < V / E; ++k) {
      const int from = (k * static_cast<int>(blockDim.x) + w * 32) * E;
      n += max(0, min(from + 32 * E, at.off + N) - max(from, at.off));
    }
    return static_cast<float>(n);
  };
  s = warp_sum(s);
  const float mine = held(warp);
  const float q = warp_sum(row_squares<T, V, EDGE>(at, N, v, mine > 0.f ? __fdividef(s, mine) : 0.f));
  if (lane == 0) slots[parity][warp] = make_float2(s, q);
  __syncthreads();
  const float2 o = lane < nw ? slots[parity][lane] : make_float2(0.f, 0.f);
  const float mean = warp_sum(o.x) / static_cast<float>(N);
  const float n = lane < nw ? held(lane) : 0.f;
  const float d = n > 0.f ? __fdividef(o.x, n) - mean : 0.f;
  const float var = warp_sum(fmaf(n * d, d, o.y)) / static_cast<float>(N);
  return make_float2(mean, rsqrtf(var + eps));
}

// A row for a block, V values a thread.  STAY: the block takes several rows of a
// class, with the weights at its columns in shared memory as fp32 and the next
// row's loads in flight; otherwise one row, and the weights come from L1 or L2 at
// its end.
template <class T, int V, bool EDGE, bool RES, bool STAY>
__global__ void __launch_bounds__(1024) fwd_block(const FwdP<T> p, const Rows rows) {
  constexpr int E = kE<T>, K = V / E;
  extern __shared__ __align__(16) float vectors[];  // STAY: [2][chunks E]
  __shared__ float2 slots[2][32];
  const int N = static_cast<int>(p.N);
  const int cls = EDGE ? blockIdx.x % rows.classes : 0;
  const int off = EDGE ? static_cast<int>((rows.off + static_cast<int64_t>(cls) * N) % E) : 0;
  const RowPlaces<T, V, EDGE> at = {static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x), off};
  const int64_t step = STAY ? rows.classes : 1;
  int64_t row = STAY ? blockIdx.x / rows.classes * rows.each * step + cls : blockIdx.x;
  const int64_t end = STAY ? min(rows.M, row + rows.each * step) : row + 1;
  if (row >= end) return;
  const int apart = static_cast<int>(blockDim.x) * V;  // of w's and b's in shared memory
  uint4 xv[K], rv[K];
  load_row<T, V, EDGE, RES>(p, row, at, N, xv, rv);
  if (STAY) {
#pragma unroll 1
    for (int i = threadIdx.x; i < apart; i += blockDim.x) {
      const int n = i - off;
      const bool in = n >= 0 && n < N;
      vectors[i] = in ? vector_at(p.w, n, 1.f) : 0.f;
      vectors[apart + i] = in ? vector_at(p.b, n, 0.f) : 0.f;
    }
  }  // (block_stats has a barrier before they are read)
  for (int parity = 0; row < end; row += step, parity ^= 1) {
    float v[V];
    const float s = row_values<T, V, EDGE, RES>(p, row, at, N, xv, rv, v);
    if (STAY && row + step < end) load_row<T, V, EDGE, RES>(p, row + step, at, N, xv, rv);
    const float2 st = block_stats<T, V, EDGE>(at, N, v, s, p.eps, slots, parity);
    if (threadIdx.x == 0 && p.mean) p.mean[row] = st.x;
    if (threadIdx.x == 0 && p.rstd) p.rstd[row] = st.y;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float w[E], b[E];
      if (STAY) {
        const int c = (threadIdx.x + k * blockDim.x) * E;
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
          unpack<float>(*reinterpret_cast<const uint4*>(vectors + c + 4 * q), w + 4 * q);
          unpack<float>(*reinterpret_cast<const uint4*>(vectors + apart + c + 4 * q), b + 4 * q);
        }
      } else {
        load_vector<T, EDGE>(p.w, at[k], N, 1.f, w);
        load_vector<T, EDGE>(p.b, at[k], N, 0.f, b);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) v[k * E + i] = fmaf((v[k * E + i] - st.x) * st.y, w[i], b[i]);
      store_chunk<T, EDGE>(p.y + row * p.N, at[k], N, v + k * E);
    }
  }
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

// --------------------------------------------------------------- gradient

// The values of a row's chunk that are not its own (a neighbour row's, or what
// lies between rows) are set aside: dy to 0, x to the mean.
template <class T, bool EDGE>
__device__ __forceinline__ void own_values(const Place<T, EDGE>& at, int N, float mean, float* g, float* x) {
  if (!EDGE || at.all(N)) return;
#pragma unroll
  for (int i = 0; i < kE<T>; ++i)
    if (!at.has(i, N)) {
      g[i] = 0.f;
      x[i] = mean;
    }
}

// A chunk's part of (sum of g, sum of g (x - mean)), g = dy w.
template <class T>
__device__ __forceinline__ void chunk_sums(const float* dy, const float* x, const float* w, float mean, float2& s1,
                                           float2& s2) {
  const float2 m = make_float2(-mean, -mean);
#pragma unroll
  for (int i = 0; i < kE<T>; i += 2) {
    const float2 t = __fadd2_rn(make_float2(x[i], x[i + 1]), m);
    const float2 g = __fmul2_rn(make_float2(dy[i], dy[i + 1]), make_float2(w[i], w[i + 1]));
    s1 = __fadd2_rn(s1, g);
    s2 = __ffma2_rn(g, t, s2);
  }
}

// What a row's second pass needs of its sums.
struct RowTerms {
  float r;       // rstd
  float2 mean;   // -mean, twice
  float2 a, b;   // dx = r g + a + b (x - mean)
  __device__ __forceinline__ RowTerms(float mu, float rstd, float s1, float s2, float invN) : r(rstd) {
    mean = make_float2(-mu, -mu);
    // mean(g) r, and mean(xhat g) r of xhat = (x - mean) r
    const float ca = -s1 * invN * r, cb = -((s2 * r) * invN) * r * r;
    a = make_float2(ca, ca);
    b = make_float2(cb, cb);
  }
};

// A chunk's dx (added to `o`, which holds dres or 0), and its part of dw and db.
template <class T>
__device__ __forceinline__ void chunk_grad(const float* dy, const float* x, const float* w, const RowTerms& t, float* o,
                                           float* dw, float* db) {
  const float2 r = make_float2(t.r, t.r);
#pragma unroll
  for (int i = 0; i < kE<T>; i += 2) {
    const float2 d = make_float2(dy[i], dy[i + 1]);
    const float2 far = __fadd2_rn(make_float2(x[i], x[i + 1]), t.mean);
    const float2 g = __fmul2_rn(d, make_float2(w[i], w[i + 1]));
    const float2 e = __ffma2_rn(g, r, __ffma2_rn(far, t.b, t.a));
    const float2 out = __fadd2_rn(make_float2(o[i], o[i + 1]), e);
    o[i] = out.x;
    o[i + 1] = out.y;
    const float2 aw = __ffma2_rn(d, __fmul2_rn(far, r), make_float2(dw[i], dw[i + 1]));
    dw[i] = aw.x;
    dw[i + 1] = aw.y;
    const float2 ab = __fadd2_rn(d, make_float2(db[i], db[i + 1]));
    db[i] = ab.x;
    db[i + 1] = ab.y;
  }
}

// Rows of up to 512 values: L lanes a row, V values a lane, no barrier; groups of
// lanes stay within a class, with the weights and the columns' sums in registers
// and the next row's loads in flight.  At the end a block's groups add their
// sums in shared memory, one after the other.
template <class T, int V, int L, bool EDGE, bool RES>
__global__ void __launch_bounds__(256) bwd_lanes(const BwdP<T> p, const Rows rows) {
  constexpr int E = kE<T>, K = V / E;
  __shared__ float sums[2][512];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int N = static_cast<int>(p.N);
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (256 / L);  // a multiple of the classes
  int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int off = EDGE ? static_cast<int>((rows.off + row % rows.classes * N) % E) : 0;
  const int t = threadIdx.x % L;
  const RowPlaces<T, V, EDGE> at = {t, L, off};
  uint4 dv[K], xv[K], rv[K];
  float mean = 0.f, rstd = 0.f;
  auto load = [&](int64_t n) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      dv[k] = load_chunk<T, EDGE>(p.dy + n * p.ys, at[k], N);
      xv[k] = load_chunk<T, EDGE>(p.x + n * p.xs, at[k], N);
      if (RES) rv[k] = load_chunk<T, EDGE>(p.dres + n * p.rs, at[k], N);
    }
    mean = __ldg(p.mean + n);
    rstd = __ldg(p.rstd + n);
  };
#pragma unroll
  for (int k = 0; k < K; ++k) dv[k] = xv[k] = rv[k] = make_uint4(0, 0, 0, 0);
  if (row < rows.M) load(row);
  float w[V], dw[V], db[V];
#pragma unroll
  for (int k = 0; k < K; ++k) load_vector<T, EDGE>(p.w, at[k], N, 1.f, w + k * E);
#pragma unroll
  for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.f;
  const float invN = 1.0f / static_cast<float>(N);
  // (the lanes of a warp stay together: shuffles are the whole warp's)
  for (int64_t lead = row - (threadIdx.x & 31) / L; lead < rows.M; lead += groups, row += groups) {
    const bool in = row < rows.M;
    const float mu = mean, r = rstd;
    uint4 cd[K], cx[K], cr[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      cd[k] = dv[k];
      cx[k] = xv[k];
      if (RES) cr[k] = rv[k];
    }
    if (row + groups < rows.M) load(row + groups);
    float2 s1 = make_float2(0.f, 0.f), s2 = s1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float d[E], x[E];
      unpack<T>(cd[k], d);
      unpack<T>(cx[k], x);
      own_values<T, EDGE>(at[k], N, mu, d, x);
      chunk_sums<T>(d, x, w + k * E, mu, s1, s2);
    }
    const float g1 = lanes_sum<L>(s1.x + s1.y), g2 = lanes_sum<L>(s2.x + s2.y);
    if (!in) continue;
    const RowTerms terms(mu, r, g1, g2, invN);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float d[E], x[E], o[E];
      unpack<T>(cd[k], d);
      unpack<T>(cx[k], x);
      own_values<T, EDGE>(at[k], N, mu, d, x);
      if (RES) unpack<T>(cr[k], o);
      else
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = 0.f;
      if (at[k].some(N)) chunk_grad<T>(d, x, w + k * E, terms, o, dw + k * E, db + k * E);
      store_chunk<T, EDGE>(p.dx + row * p.N, at[k], N, o);
    }
  }
  if (!p.want_dw && !p.want_db) return;
  for (int i = threadIdx.x; i < 2 * 512; i += 256) (&sums[0][0])[i] = 0.f;
  for (int q = 0; q < 256 / L; ++q) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) / L != q) continue;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (at[k].some(N) && at[k].has(i, N)) {
          sums[0][at[k].n0 + i] += dw[k * E + i];
          sums[1][at[k].n0 + i] += db[k * E + i];
        }
  }
  __syncthreads();
  float* to = p.partials + static_cast<int64_t>(blockIdx.x) * (p.want_dw + p.want_db) * N;
  for (int n = threadIdx.x; n < N; n += 256) {
    if (p.want_dw) to[n] = sums[0][n];
    if (p.want_db) to[(p.want_dw ? N : 0) + n] = sums[1][n];
  }
}

// A chunk's sums into a row of partials.
template <class T, bool EDGE>
__device__ __forceinline__ void store_sums(float* row, const Place<T, EDGE>& at, int N, const float* f) {
  if (!EDGE && at.some(N)) {
#pragma unroll
    for (int q = 0; q < kE<T> / 4; ++q)
      *reinterpret_cast<float4*>(row + at.n0 + 4 * q) = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
  } else if (EDGE && at.some(N)) {
#pragma unroll
    for (int i = 0; i < kE<T>; ++i)
      if (at.has(i, N)) row[at.n0 + i] = f[i];
  }
}

// Wider rows: a block stays for `each` rows of a class.  Thread 0 streams the
// rows' windows (their chunks, whole) of dy, x and dres into a ring of S stages by
// bulk copies; each row is read from its stage twice, for its sums and for its
// results, so a thread keeps only the weights at its 16 columns and the two sums
// of each: at most 80 registers, and several blocks an SM whose barriers
// overlap.  WIDE (more than 768 threads a block): 64 registers, the weights from L1.
//
// A window reaches up to 15 bytes past its row on either side.  Where that is not
// the tensor's own memory (before its first value, behind its last) the chunk is
// left out of the copy and its own values are written by thread 0.
struct Ring {
  int stages, slot;  // bytes of a row's window
};

template <class T>
__device__ __forceinline__ uint32_t window(unsigned char* to, const T* base, int64_t stride, int64_t row, int64_t M,
                                           int off, int N, uint64_t* bar, bool count) {
  constexpr int E = kE<T>;
  const int chunks = (off + N + E - 1) / E, over = chunks * E - off - N;
  const int first = row * stride < off ? 1 : 0;
  const int last = chunks - ((M - 1 - row) * stride < over ? 1 : 0);
  const T* from = base + row * stride;  // column 0
  const uint32_t bytes = last > first ? (last - first) * 16 : 0;
  if (count) return bytes;
  for (int c = 0; c < chunks; c += max(1, chunks - 1)) {
    if (c >= first && c < last) continue;
    for (int i = 0; i < E; ++i) {
      const int n = c * E - off + i;
      if (n >= 0 && n < N) reinterpret_cast<T*>(to)[c * E + i] = from[n];
    }
  }
  if (bytes) bulk_g2s(to + first * 16, from - off + first * E, bytes, bar);
  return bytes;
}

template <class T, bool EDGE, bool RES, bool WIDE>
__device__ __forceinline__ void bwd_ring_body(const BwdP<T>& p, const Rows& rows, const Ring& ring, int* err) {
  constexpr int E = kE<T>, V = 16, K = V / E;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float2 slots[2][32];
  __shared__ int s_abort;
  const int N = static_cast<int>(p.N);
  const int S = ring.stages, slot = ring.slot, stage_bytes = (RES ? 3 : 2) * slot;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + static_cast<size_t>(S) * stage_bytes);
  const int cls = EDGE ? blockIdx.x % rows.classes : 0;
  const int off = EDGE ? static_cast<int>((rows.off + static_cast<int64_t>(cls) * N) % E) : 0;
  const RowPlaces<T, V, EDGE> at = {static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x), off};
  const int64_t step = rows.classes;
  const int64_t r0 = blockIdx.x / rows.classes * rows.each * step + cls;
  const int count = static_cast<int>(r0 < rows.M ? min(rows.each, (rows.M - r0 + step - 1) / step) : 0);
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < S; ++i) mbar_init(&bars[i], 1);
    mbar_init_fence();
  }
  __syncthreads();
  int issued = 0;
  auto issue = [&](int i) {  // thread 0: row i into stage i % S
    if (i >= count) return;
    const int64_t row = r0 + i * step;
    unsigned char* st = smem + static_cast<size_t>(i % S) * stage_bytes;
    uint64_t* bar = &bars[i % S];
    if (EDGE) {
      uint32_t bytes = window(st, p.dy, p.ys, row, rows.M, off, N, bar, true) +
                       window(st, p.x, p.xs, row, rows.M, off, N, bar, true);
      if (RES) bytes += window(st, p.dres, p.rs, row, rows.M, off, N, bar, true);
      // (the barrier expects the bytes before any can arrive; a thread's own
      // writes come before its arrival)
      asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
      window(st, p.dy, p.ys, row, rows.M, off, N, bar, false);
      window(st + slot, p.x, p.xs, row, rows.M, off, N, bar, false);
      if (RES) window(st + 2 * slot, p.dres, p.rs, row, rows.M, off, N, bar, false);
      mbar_arrive(bar);
    } else {
      mbar_arrive_expect_tx(bar, stage_bytes);
      bulk_g2s(st, p.dy + row * p.ys, slot, bar);
      bulk_g2s(st + slot, p.x + row * p.xs, slot, bar);
      if (RES) bulk_g2s(st + 2 * slot, p.dres + row * p.rs, slot, bar);
    }
    issued = i + 1;
  };
  // Row i - 1's stage is free when all threads are in row i: S - 1 rows ahead.
  if (threadIdx.x == 0)
    for (int i = 0; i < max(1, S - 1); ++i) issue(i);
  float w[WIDE ? 1 : V], dw[V], db[V];
  if constexpr (!WIDE) {
#pragma unroll
    for (int k = 0; k < K; ++k) load_vector<T, EDGE>(p.w, at[k], N, 1.f, w + k * E);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.f;
  const float invN = 1.0f / static_cast<float>(N);
  int i = 0;
  for (; i < count; ++i) {
    const int64_t row = r0 + i * step;
    const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    const unsigned char* st = smem + static_cast<size_t>(i % S) * stage_bytes;
    if (!mbar_wait(&bars[i % S], (i / S) & 1, err)) s_abort = 1;
    float2 s1 = make_float2(0.f, 0.f), s2 = s1;
    auto chunk = [&](int k, float* d, float* x, float* wk) {
      const int c = threadIdx.x + k * blockDim.x;
      unpack<T>(*reinterpret_cast<const uint4*>(st + c * 16), d);
      unpack<T>(*reinterpret_cast<const uint4*>(st + slot + c * 16), x);
      own_values<T, EDGE>(at[k], N, mean, d, x);
      if constexpr (WIDE) {
        load_vector<T, EDGE>(p.w, at[k], N, 1.f, wk);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) wk[e] = w[k * E + e];
      }
    };
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) continue;
      float d[E], x[E], wk[E];
      chunk(k, d, x, wk);
      chunk_sums<T>(d, x, wk, mean, s1, s2);
    }
    const float2 tot = block_sum2(make_float2(s1.x + s1.y, s2.x + s2.y), slots, i & 1);
    if (s_abort) break;
    if (threadIdx.x == 0 && S > 1) issue(i + S - 1);
    const RowTerms terms(mean, rstd, tot.x, tot.y, invN);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) continue;
      float d[E], x[E], wk[E], o[E];
      chunk(k, d, x, wk);
      if (RES) unpack<T>(*reinterpret_cast<const uint4*>(st + 2 * slot + (threadIdx.x + k * blockDim.x) * 16), o);
      else
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
      chunk_grad<T>(d, x, wk, terms, o, dw + k * E, db + k * E);
      store_chunk<T, EDGE>(p.dx + row * p.N, at[k], N, o);
    }
    if (S == 1) {
      __syncthreads();
      if (threadIdx.x == 0) issue(i + 1);
    }
  }
  if (threadIdx.x == 0 && s_abort)
    for (int j = i; j < issued; ++j) mbar_wait(&bars[j % S], (j / S) & 1, nullptr);
  if (!p.want_dw && !p.want_db) return;
  float* to = p.partials + static_cast<int64_t>(blockIdx.x) * (p.want_dw + p.want_db) * N;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (p.want_dw) store_sums<T, EDGE>(to, at[k], N, dw + k * E);
    if (p.want_db) store_sums<T, EDGE>(to + (p.want_dw ? N : 0), at[k], N, db + k * E);
  }
}

template <class T, bool EDGE, bool RES>
__global__ void __maxnreg__(80) bwd_ring(const BwdP<T> p, const Rows rows, const Ring ring, int* err) {
  bwd_ring_body<T, EDGE, RES, false>(p, rows, ring, err);
}
template <class T, bool EDGE, bool RES>
__global__ void __launch_bounds__(1024) bwd_ring_wide(const BwdP<T> p, const Rows rows, const Ring ring, int* err) {
  bwd_ring_body<T, EDGE, RES, true>(p, rows, ring, err);
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
    const float g = get(dy + n) * vector_at(p.w, n, 1.f);
    s.x += g;
    s.y = fmaf((get(x + n) - mean) * r, g, s.y);
  }
  s = block_sum2(s, slots, 0);
  const float invN = 1.0f / static_cast<float>(p.N);
  const float mg = s.x * invN, mx = s.y * invN;
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) {
    const float g = get(dy + n) * vector_at(p.w, n, 1.f), xhat = (get(x + n) - mean) * r;
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

// Rows of up to so many values are a few lanes', and a block's, in the gradient.
constexpr int64_t kLanesBwd = 512, kHeldBwd = 16384;
constexpr int kSmem = 232448;  // of an SM, for its blocks

// Blocks of the ring kernel that an SM's registers hold for rows of N values.
int ring_blocks(int64_t held) {
  const int threads = static_cast<int>(ceil_div(held, 512) * 32);
  return threads > 768 ? 1 : std::min(12, 65536 / (80 * threads));
}

// Blocks of rows that the columns' sums are split over, at most.
int64_t row_blocks(int64_t M, int64_t N) {
  const int sms = sm_count();
  const int64_t per_sm = std::max(4, N <= kHeldBwd ? ring_blocks(N) : 0);
  return std::min(M + 8, (sms > 0 ? sms : 148) * per_sm);
}

// Whether rows of all of a call's tensors lie alike (the same off, row for row),
// and how.
struct Layout {
  bool alike = true;
  int off = -1, residue;
  Layout(int64_t N, int size) : residue(static_cast<int>(N % (16 / size))), size_(size) {}
  void add(const void* p, int64_t stride) {
    if (!p) return;
    const int E = 16 / size_, o = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16) / size_;
    if (off < 0) off = o;
    alike = alike && o == off && ((stride % E) + E) % E == residue;
  }
  int classes() const {
    int E = 16 / size_, r = residue;
    while (r) {
      const int t = E % r;
      E = r;
      r = t;
    }
    return 16 / size_ / E;  // E / gcd(N, E)
  }

 private:
  int size_;
};

template <class T, int V, int L, bool EDGE>
int launch_fwd_lanes(const FwdP<T>& p, Rows rows, cudaStream_t s) {
  const int per = 256 / L;  // a multiple of 8, as the classes are a divisor of 8
  const int64_t blocks = std::min<int64_t>(ceil_div(rows.M, per), static_cast<int64_t>(sm_count()) * kLaneBlocks);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (p.res) fwd_lanes<T, V, L, EDGE, true><<<grid, 256, 0, s>>>(p, rows);
  else fwd_lanes<T, V, L, EDGE, false><<<grid, 256, 0, s>>>(p, rows);
  return check_launch();
}

template <class T, bool EDGE>
int launch_fwd_lanes(const FwdP<T>& p, const Rows& rows, int64_t held, cudaStream_t s) {
  if (held <= 64) return launch_fwd_lanes<T, 8, 8, EDGE>(p, rows, s);
  if (held <= 128) return launch_fwd_lanes<T, 8, 16, EDGE>(p, rows, s);
  if (held <= 256) return launch_fwd_lanes<T, 8, 32, EDGE>(p, rows, s);
  return launch_fwd_lanes<T, 16, 32, EDGE>(p, rows, s);
}

template <class T, bool EDGE, bool RES>
int launch_fwd_block(const FwdP<T>& p, Rows rows, int64_t held, cudaStream_t s) {
  constexpr int V = 16;
  constexpr bool STAY = EDGE;
  auto kernel = fwd_block<T, V, EDGE, RES, STAY>;
  const int threads = static_cast<int>(ceil_div(held, 32 * V) * 32);
  int64_t blocks = rows.M;
  int smem = 0;
  if (STAY) {
    smem = 2 * V * threads * static_cast<int>(sizeof(float));
    if (!allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return FRAG_ERR_CUDA;
    const int per_sm = std::max(1, std::min({1024 / threads, 220 * 1024 / smem, 16}));
    const int64_t of_class = ceil_div(rows.M, rows.classes);
    const int64_t resident = std::max(1, sm_count() * per_sm / rows.classes);
    rows.each = ceil_div(of_class, std::min(of_class, resident));
    blocks = ceil_div(of_class, rows.each) * rows.classes;
  }
  kernel<<<dim3(static_cast<unsigned>(blocks)), threads, smem, s>>>(p, rows);
  return check_launch();
}

// Rows of up to so many values are held in registers.
constexpr int64_t kLanesFwd = 512, kHeldFwd = 16384;

template <class T>
int forward(const FwdP<T>& p, int64_t M, cudaStream_t s) {
  Layout lay(p.N, sizeof(T));
  lay.add(p.x, p.xs);
  lay.add(p.res, p.rs);
  lay.add(p.y, p.N);
  lay.add(p.h, p.N);
  const bool edge = lay.off || lay.residue;
  const int64_t held = p.N + (edge ? kE<T> - 1 : 0);  // values of a row's chunks, at most
  if (!lay.alike || held > kHeldFwd) {
    fwd_any<T><<<dim3(static_cast<unsigned>(M)), 256, 0, s>>>(p);
    return check_launch();
  }
  const Rows rows = {M, lay.off, lay.classes(), 1};
  if (held <= kLanesFwd)
    return edge ? launch_fwd_lanes<T, true>(p, rows, held, s) : launch_fwd_lanes<T, false>(p, rows, held, s);
  if (edge) return p.res ? launch_fwd_block<T, true, true>(p, rows, held, s) : launch_fwd_block<T, true, false>(p, rows, held, s);
  return p.res ? launch_fwd_block<T, false, true>(p, rows, held, s) : launch_fwd_block<T, false, false>(p, rows, held, s);
}

template <class T, int V, int L, bool EDGE>
int launch_bwd_lanes(const BwdP<T>& p, Rows rows, int64_t* G, cudaStream_t s) {
  const int per = 256 / L;  // a multiple of 8, as the classes are a divisor of 8
  *G = std::min<int64_t>(ceil_div(rows.M, per), static_cast<int64_t>(sm_count()) * kLaneBlocks);
  const dim3 grid(static_cast<unsigned>(*G));
  if (p.dres) bwd_lanes<T, V, L, EDGE, true><<<grid, 256, 0, s>>>(p, rows);
  else bwd_lanes<T, V, L, EDGE, false><<<grid, 256, 0, s>>>(p, rows);
  return check_launch();
}

template <class T, bool EDGE>
int launch_bwd_lanes(const BwdP<T>& p, const Rows& rows, int64_t held, int64_t* G, cudaStream_t s) {
  if (held <= 64) return launch_bwd_lanes<T, 8, 8, EDGE>(p, rows, G, s);
  if (held <= 128) return launch_bwd_lanes<T, 8, 16, EDGE>(p, rows, G, s);
  if (held <= 256) return launch_bwd_lanes<T, 8, 32, EDGE>(p, rows, G, s);
  return launch_bwd_lanes<T, 16, 32, EDGE>(p, rows, G, s);
}

template <class T, bool EDGE, bool RES>
int launch_bwd_ring(const BwdP<T>& p, Rows rows, int64_t held, int64_t* G, cudaStream_t s) {
  const int threads = static_cast<int>(ceil_div(held, 512) * 32);
  auto kernel = threads > 768 ? bwd_ring_wide<T, EDGE, RES> : bwd_ring<T, EDGE, RES>;
  // A row's chunks, whatever its off.
  const int slot = static_cast<int>(ceil_div(held, kE<T>)) * 16, stage = slot * (RES ? 3 : 2);
  // As many blocks as leave each two stages, and then as many stages as fit.
  int per_sm = ring_blocks(held), stages = 0;
  for (; per_sm >= 1; --per_sm) {
    stages = std::min(8, (kSmem / per_sm - 2048) / stage);  // (1 KB is the system's, 1 the rest of the block's)
    if (stages >= 2) break;
  }
  if (per_sm < 1) {
    per_sm = 1;
    if (stages < 1) return FRAG_ERR_SHAPE;
  }
  const int smem = stages * stage + 8 * stages;
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return FRAG_ERR_CUDA;
  const int64_t of_class = ceil_div(rows.M, rows.classes);
  const int64_t resident = std::max(1, sm_count() * per_sm / rows.classes);
  rows.each = ceil_div(of_class, std::min(of_class, resident));
  *G = ceil_div(of_class, rows.each) * rows.classes;
  kernel<<<dim3(static_cast<unsigned>(*G)), threads, smem, s>>>(p, rows, {stages, slot}, device_error_word());
  return check_launch();
}

template <class T>
int backward(const BwdP<T>& p, int64_t M, float* dw, float* db, cudaStream_t s) {
  Layout lay(p.N, sizeof(T));
  lay.add(p.dy, p.ys);
  lay.add(p.x, p.xs);
  lay.add(p.dres, p.rs);
  lay.add(p.dx, p.N);
  const bool edge = lay.off || lay.residue;
  const int64_t held = p.N + (edge ? kE<T> - 1 : 0);
  const Rows rows = {M, lay.off, lay.classes(), 1};
  int64_t G = 0;
  int st;
  if (!lay.alike || held > kHeldBwd) {
    bwd_any_dx<T><<<dim3(static_cast<unsigned>(M)), 256, 0, s>>>(p);
    if (st = check_launch(); st != FRAG_OK || (!dw && !db)) return st;
    const int64_t R = ceil_div(M, std::min(M, static_cast<int64_t>(sm_count()) * 4));
    G = ceil_div(M, R);
    const dim3 grid(static_cast<unsigned>(ceil_div(p.N, 256)), static_cast<unsigned>(G));
    bwd_any_columns<T><<<grid, 256, 0, s>>>(p, M, R);
    st = check_launch();
  } else if (held <= kLanesBwd) {
    st = edge ? launch_bwd_lanes<T, true>(p, rows, held, &G, s) : launch_bwd_lanes<T, false>(p, rows, held, &G, s);
  } else if (edge) {
    st = p.dres ? launch_bwd_ring<T, true, true>(p, rows, held, &G, s) : launch_bwd_ring<T, true, false>(p, rows, held, &G, s);
  } else {
    st = p.dres ? launch_bwd_ring<T, false, true>(p, rows, held, &G, s) : launch_bwd_ring<T, false, false>(p, rows, held, &G, s);
  }
  if (st != FRAG_OK || (!dw && !db)) return st;
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

size_t frag_layernorm_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 0;
  return align_up(static_cast<size_t>(row_blocks(M, N)) * 2 * N * sizeof(float), 256);
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
  const Vector wv = {w, wdtype == FRAG_DT_F32, aligned16(w)};
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

// layernorm_bwd.cu — the gradient of layer norm, with the sums over the rows for
// weight and bias.
#include "layernorm.cuh"

namespace frag {
namespace {

template <class T>
struct BwdP {
  const T* dy;
  const T* x;
  const T* dres;
  T* dx;
  Vector w;
  const float* mean;
  const float* rstd;
  float* partials;  // [G, vectors, width]: dw, db, as far as wanted
  int64_t width;    // N, or a row's chunks: a column then lies off places further on
  int64_t ys, xs, rs;
  int64_t N;
  int want_dw, want_db;
};

// --------------------------------------------------------------- gradient

// Rows that a thread adds up at most: a sum of n terms is off by up to n / 2 half steps
// where the terms are alike, and all the same way (1772 rows of 0.3: 1.8e-5).  For more
// rows there are more blocks than an SM holds at once, each with partials of its own.
// 262144 rows of 8192 in bf16 (885 for a thread): 2036 us, with dres 2676; in one run
// each 1880 and 2581.  Up to 128 for a thread nothing changes.
constexpr int kRun = 128;
// The blocks of a launch: `at_once`, as often as rows call for, each with `rows_at_once`.
int64_t blocks_for(int64_t M, int64_t at_once, int64_t rows_at_once) {
  return at_once * ceil_div(M, at_once * rows_at_once * kRun);
}

// A chunk: x becomes x - mean, and its part of (sum of g, sum of g (x - mean)),
// g = dy w, is added.
template <class T>
__device__ __forceinline__ void chunk_sums(const float2* dy, float2* x, const float2* w, float mean, float2& s1,
                                           float2& s2) {
#pragma unroll
  for (int q = 0; q < kP<T>; ++q) {
    x[q] = __fadd2_rn(x[q], twice(-mean));
    const float2 g = __fmul2_rn(dy[q], w[q]);
    s1 = __fadd2_rn(s1, g);
    s2 = __ffma2_rn(g, x[q], s2);
  }
}

// What a row's second pass needs of its sums: dx = r g + a + b (x - mean).
struct RowTerms {
  float2 r, a, b;
  __device__ __forceinline__ RowTerms(float rstd, float s1, float s2, float invN) {
    r = twice(rstd);
    a = twice(-s1 * invN * rstd);                           // mean(g) rstd
    b = twice(-((s2 * rstd) * invN) * rstd * rstd);         // mean(xhat g) rstd, of xhat = (x - mean) rstd
  }
};

// A chunk's dx (on top of dres, where there is one), and its part of dw and db.
template <class T, bool RES>
__device__ __forceinline__ void chunk_grad(const float2* dy, const float2* far, const float2* w, const RowTerms& t,
                                           float2* o, float2* dw, float2* db) {
#pragma unroll
  for (int q = 0; q < kP<T>; ++q) {
    float2 e = __ffma2_rn(far[q], t.b, t.a);
    e = __ffma2_rn(__fmul2_rn(dy[q], w[q]), t.r, e);
    o[q] = RES ? __fadd2_rn(o[q], e) : e;
    dw[q] = __ffma2_rn(dy[q], __fmul2_rn(far[q], t.r), dw[q]);
    db[q] = __fadd2_rn(dy[q], db[q]);
  }
}

// Rows of up to 512 values, as fwd_lanes; the columns' sums stay in registers,
// and at the end a block's groups add theirs in shared memory, one after the other.
// 262144 rows of 128 in bf16 take 41 us, of which the sums' end (the groups' turns
// and add_partials) is 4.5 and the start 5; a million rows 135, 6.0 TB/s.  Three
// blocks an SM at 80 registers; four at 64 spill.
template <class T, int V, int L, Mode MODE, bool RES>
__global__ void __launch_bounds__(256, lane_blocks(V, MODE, 3)) bwd_lanes(const BwdP<T> p, const Rows rows) {
  constexpr int E = kE<T>, P = kP<T>, K = V / E, ROW = (RES ? 3 : 2) * K;
  extern __shared__ __align__(16) uint4 held[];  // [kAhead][ROW][256], and (mean, rstd) of each row
  float* stats = reinterpret_cast<float*>(held + kAhead * ROW * 256);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int N = static_cast<int>(p.N);
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (256 / L);  // a multiple of the classes
  int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int off = MODE == EDGE ? static_cast<int>((rows.off + row % rows.classes * N) % E) : 0;
  const int t = threadIdx.x % L;
  const Places<T, MODE> at = {t, L, off};
  Bits<T, MODE> own[K];
#pragma unroll
  for (int k = 0; k < K; ++k) own[k].set(at[k], N);
  Walk<T> dy({p.dy, p.ys}, row, groups), x({p.x, p.xs}, row, groups), res({RES ? p.dres : p.x, p.rs}, row, groups);
  int64_t asked = row;
  auto ask = [&](int s) {
    uint4* to = held + s * (ROW * 256) + threadIdx.x;
    if (asked < rows.M) {
      const bool end = asked == 0 || asked == rows.M - 1;
      dy.template ask<K, MODE>(at, N, end, to);
      x.template ask<K, MODE>(at, N, end, to + K * 256);
      if (RES) res.template ask<K, MODE>(at, N, end, to + 2 * K * 256);
      if (t == 0) {  // (for all lanes of the row)
        float* st = stats + (s * 256 + threadIdx.x) / L * 2;
        copy_async4(st, p.mean + asked);
        copy_async4(st + 1, p.rstd + asked);
      }
    }
    copies_commit();
    asked += groups;
    dy.next += dy.jump;
    x.next += x.jump;
    if (RES) res.next += res.jump;
  };
#pragma unroll
  for (int s = 0; s < kAhead - 1; ++s) ask(s);
  float2 w[V / 2], dw[V / 2], db[V / 2];
#pragma unroll
  for (int k = 0; k < K; ++k) load_vector<T, MODE>(p.w, at[k], N, 1.f, w + k * P);
#pragma unroll
  for (int q = 0; q < V / 2; ++q) dw[q] = db[q] = twice(0.f);
  const float invN = 1.0f / static_cast<float>(N);
  int s = 0;
  T* dx = p.dx + row * p.N;
  const int64_t jump = groups * p.N;
  // (the lanes of a warp stay together: shuffles are the whole warp's)
  for (int64_t lead = row - (threadIdx.x & 31) / L; lead < rows.M; lead += groups, row += groups, dx += jump) {
    __syncwarp();  // (every lane has the mean and deviation that the next ones replace)
    ask(s == 0 ? kAhead - 1 : s - 1);
    copies_wait<kAhead - 1>();
    __syncwarp();  // (the first lane's copies too)
    const uint4* from = held + s * (ROW * 256) + threadIdx.x;
    const float2 st = reinterpret_cast<const float2*>(stats)[(s * 256 + threadIdx.x) / L];
    const float mean = st.x, rstd = st.y;
    s = s == kAhead - 1 ? 0 : s + 1;
    float2 d[V / 2], xv[V / 2], s1 = twice(0.f), s2 = s1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) continue;
      // (of another row's values dy is 0, and so is all that x is multiplied with)
      unpack<T>(own[k](from[k * 256]), d + k * P);
      unpack<T>(own[k](from[(K + k) * 256]), xv + k * P);
      chunk_sums<T>(d + k * P, xv + k * P, w + k * P, mean, s1, s2);
    }
    const float g1 = lanes_sum<L>(s1.x + s1.y), g2 = lanes_sum<L>(s2.x + s2.y);
    if (row >= rows.M) continue;
    const RowTerms terms(rstd, g1, g2, invN);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) continue;
      float2 o[P];
      if (RES) unpack<T>(from[(2 * K + k) * 256], o);
      chunk_grad<T, RES>(d + k * P, xv + k * P, w + k * P, terms, o, dw + k * P, db + k * P);
      store_chunk<T, MODE>(dx, at[k], N, o);
    }
  }
  if (!p.want_dw && !p.want_db) return;
  copies_wait<0>();
  __syncthreads();
  float* sums = reinterpret_cast<float*>(held);  // [2][512]
  for (int i = threadIdx.x; i < 2 * 512; i += 256) sums[i] = 0.f;
  for (int q = 0; q < 256 / L; ++q) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) / L != q) continue;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (at[k].some(N) && at[k].has(i, N)) {
          sums[at[k].n0 + i] += part(dw[k * P + i / 2], i & 1);
          sums[512 + at[k].n0 + i] += part(db[k * P + i / 2], i & 1);
        }
  }
  __syncthreads();
  float* to = p.partials + static_cast<int64_t>(blockIdx.x) * (p.want_dw + p.want_db) * N;
  for (int n = threadIdx.x; n < N; n += 256) {
    if (p.want_dw) to[n] = sums[n];
    if (p.want_db) to[(p.want_dw ? N : 0) + n] = sums[512 + n];
  }
}

// A chunk's sums into a row of partials, by their places in the row's chunks.
template <class T>
__device__ __forceinline__ void store_sums(float* row, int c, const float2* f) {
#pragma unroll
  for (int q = 0; q < kP<T>; q += 2)
    *reinterpret_cast<float4*>(row + c * kE<T> + 2 * q) = make_float4(f[q].x, f[q].y, f[q + 1].x, f[q + 1].y);
}

// Two sums over a group of up to 16 warps, in a fixed order, for every thread.
// After one exchange the lower half of a warp's lanes add the first and the upper
// half the second, so that both take one shuffle a level.  slots: [2][16][2],
// the group's at `first`.
__device__ __forceinline__ float2 group_pair(const Group& g, float a, float b, float (*slots)[2], int first) {
  const int lane = threadIdx.x & 31, nw = g.threads >> 5;
  const int upper = lane >> 4;
  float v = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((lane & 15) == 0) slots[first + (g.t >> 5)][upper] = v;
  g.sync();
  if (nw > 1) {
    v = (lane & 15) < nw ? slots[first + (lane & 15)][upper] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
}

// Wider rows, a group a row at a time.  A thread keeps its columns' two sums (64
// registers); a row is read from its stage twice, for its sums and for its results,
// as a row's own values would not fit beside them.  One block of 16 warps an SM, so
// an SM leaves one row of partials; four blocks with weights in registers left four
// and were slower.
//
// Bound: HBM once the rows are many (32768 of 8192 in bf16 251 us, 6.4 TB/s, 0.98 of
// a copy's rate); 8192 of 4096 take 41, with dres 50 (floors 31 and 41): 4.4 for
// the partials and their second launch, some 5 to start and to end.
template <class T, class W, Mode MODE, bool RES>
__global__ void __launch_bounds__(512) bwd_groups(const BwdP<T> p, const Rows rows, const Shape shape, int* err) {
  constexpr int E = kE<T>, P = kP<T>, V = kV, K = V / E, INPUTS = RES ? 3 : 2;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) unsigned char smem[];  // w, the rings; at the end dw, db
  __shared__ float slots[2][16][2];
  __shared__ Gave gave;
  const int N = static_cast<int>(p.N);
  const Group g(shape.threads);
  const int apart = shape.threads * V;
  W* w = reinterpret_cast<W*>(smem);
  Ring<T, INPUTS, MODE> ring;
  ring.in[0] = {p.dy, p.ys};
  ring.in[1] = {p.x, p.xs};
  if (RES) ring.in[INPUTS - 1] = {p.dres, p.rs};
  deal(ring, rows, shape, g.index, smem + sizeof(W) * apart, N);
  const Places<T, MODE> at = {g.t, g.threads, ring.off};
  if (g.t == 0) {
    gave.begin(g);
    ring.begin();
    // A stage is free again when every thread is in the next row: S - 1 rows ahead.
    for (int i = 0; i < max(1, ring.S - 1); ++i) ring.issue();
  }
  share_vector<T, W, MODE>(p.w, 1.f, w, apart, ring.off, N);
  float2 dw[V / 2], db[V / 2];
#pragma unroll
  for (int q = 0; q < V / 2; ++q) dw[q] = db[q] = twice(0.f);
  int64_t row = ring.r0;
  float mean = 0.f, rstd = 0.f;
  if (ring.count) {
    mean = __ldg(p.mean + row);
    rstd = __ldg(p.rstd + row);
  }
  __syncthreads();
  const float invN = 1.0f / static_cast<float>(N);
  const int first = g.index * (g.threads >> 5);
  int i = 0;
  for (; i < ring.count; ++i, row += ring.step) {
    if (!ring.wait(err)) gave.up(g, i);
    // A chunk's dy, x and weights.
    auto take = [&](int k, float2* d, float2* x, float2* wk) {
      const int c = g.t + k * g.threads;
      unpack<T>(ring.chunk(0, c), d);
      unpack<T>(ring.chunk(1, c), x);
      own_values<T, MODE>(at[k], N, 0.f, d);
      own_values<T, MODE>(at[k], N, mean, x);
      shared_chunk<T, W>(w, apart, c, wk);
    };
    float2 s1 = twice(0.f), s2 = s1;
    constexpr int AT_ONCE = sizeof(T) == 4 ? 2 : K;
#pragma unroll AT_ONCE
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) continue;
      float2 d[P], x[P], wk[P];
      take(k, d, x, wk);
      chunk_sums<T>(d, x, wk, mean, s1, s2);
    }
    const float2 tot = group_pair(g, s1.x + s1.y, s2.x + s2.y, slots[i & 1], first);
    if (gave.is_up(g, i)) break;
    if (g.t == 0 && ring.S > 1) ring.issue();
    const RowTerms terms(rstd, tot.x, tot.y, invN);
    float next_mean = 0.f, next_rstd = 0.f;
    if (i + 1 < ring.count) {
      next_mean = __ldg(p.mean + row + ring.step);
      next_rstd = __ldg(p.rstd + row + ring.step);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) continue;
      float2 d[P], x[P], wk[P], o[P];
      take(k, d, x, wk);
#pragma unroll
      for (int q = 0; q < P; ++q) x[q] = __fadd2_rn(x[q], twice(-mean));
      if (RES) unpack<T>(ring.chunk(INPUTS - 1, g.t + k * g.threads), o);
      chunk_grad<T, RES>(d, x, wk, terms, o, dw + k * P, db + k * P);
      store_chunk<T, MODE>(p.dx + row * p.N, at[k], N, o);
    }
    mean = next_mean;
    rstd = next_rstd;
    if (ring.S == 1) {
      g.sync();
      if (g.t == 0) ring.issue();
    }
    ring.next();
  }
  if (g.t == 0 && i < ring.count) ring.drain(i);
  if (!p.want_dw && !p.want_db) return;
  float* to = p.partials + static_cast<int64_t>(blockIdx.x) * (p.want_dw + p.want_db) * p.width;
  float* to_db = to + (p.want_dw ? p.width : 0);
  if (shape.groups == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at[k].some(N)) continue;
      if (p.want_dw) store_sums<T>(to, g.t + k * g.threads, dw + k * P);
      if (p.want_db) store_sums<T>(to_db, g.t + k * g.threads, db + k * P);
    }
    return;
  }
  // All groups' sums into shared memory, a column's added in the groups' order.
  __syncthreads();
  float2* sums = reinterpret_cast<float2*>(smem) + g.index * (V * g.threads) + g.t;
#pragma unroll
  for (int q = 0; q < V / 2; ++q) {
    sums[q * g.threads] = dw[q];
    sums[(V / 2 + q) * g.threads] = db[q];
  }
  __syncthreads();
  sums = reinterpret_cast<float2*>(smem) + g.t;
  for (int k = g.index; k < K; k += shape.groups) {
    if (!at[k].some(N)) continue;
    float2 sw[P], sb[P];
#pragma unroll
    for (int j = 0; j < P; ++j) sw[j] = sb[j] = twice(0.f);
    for (int i = 0; i < shape.groups; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) {
        sw[j] = __fadd2_rn(sw[j], sums[(i * V + k * P + j) * g.threads]);
        sb[j] = __fadd2_rn(sb[j], sums[(i * V + V / 2 + k * P + j) * g.threads]);
      }
    if (p.want_dw) store_sums<T>(to, g.t + k * g.threads, sw);
    if (p.want_db) store_sums<T>(to_db, g.t + k * g.threads, sb);
  }
}

// Any width, any alignment, as fwd_any: dx a block a row, then the columns' sums in a
// second pass over dy and x.
template <class T>
__global__ void __launch_bounds__(256) bwd_any_dx(const BwdP<T> p) {
  __shared__ float2 slots[2][32];
  const int64_t row = blockIdx.x;
  const T* dy = p.dy + row * p.ys;
  const T* x = p.x + row * p.xs;
  const float mean = p.mean[row], r = p.rstd[row];
  auto sums = [&](auto weight) {
    return long_sums(p.N, [&](int64_t n) {
      const float g = get(dy + n) * weight(n);
      return make_float2(g, (get(x + n) - mean) * r * g);
    });
  };
  float2 s;  // (what the weights are is asked once)
  if (!p.w.p) s = sums([](int64_t) { return 1.f; });
  else if (p.w.f32) s = sums([&](int64_t n) { return static_cast<const float*>(p.w.p)[n]; });
  else s = sums([&](int64_t n) { return bf16_to_f(static_cast<const uint16_t*>(p.w.p)[n]); });
  s = block_sum2(s, slots, 0);
  const float invN = 1.0f / static_cast<float>(p.N);
  const float mg = s.x * invN, mx = s.y * invN;
  for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) {
    const float g = get(dy + n) * vector_at(p.w, n, 1.f), xhat = (get(x + n) - mean) * r;
    const float d = (g - mg - xhat * mx) * r;
    put(p.dx + row * p.N + n, p.dres ? get(p.dres + row * p.rs + n) + d : d);
  }
}

// Columns of a block of rows, a thread each, by kRun rows.
template <class T>
__global__ void __launch_bounds__(256) bwd_any_columns(const BwdP<T> p, int64_t M, int64_t R) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (n >= p.N) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * R, r1 = min(M, r0 + R);
  float dw = 0.f, db = 0.f;
  for (int64_t row = r0; row < r1;) {
    float rw = 0.f, rb = 0.f;
#pragma unroll 4
    for (const int64_t end = min(r1, row + kRun); row < end; ++row) {
      const float g = get(p.dy + row * p.ys + n);
      rw = fmaf(g, (get(p.x + row * p.xs + n) - p.mean[row]) * p.rstd[row], rw);
      rb += g;
    }
    dw += rw;
    db += rb;
  }
  float* to = p.partials + static_cast<int64_t>(blockIdx.y) * (p.want_dw + p.want_db) * p.N;
  if (p.want_dw) to[n] = dw;
  if (p.want_db) to[(p.want_dw ? p.N : 0) + n] = db;
}

// How the partials lie: row g's column n at n + (off + g N) % E of `width` places
// (E = 1: at n).
struct Partials {
  const float* p;
  int64_t G, N, width;
  int vectors, off, E;
};

// The G rows of partials added in a fixed order: 32 columns a block, warp w adds the
// rows w, w + WARPS, ..., AT_ONCE in flight and then those to what it has, then the
// warps' sums in order.  The
// first N columns go to `first`, the others to `second`.  The launch, which waits
// for the other's end, costs 3 us however few the rows, up to 4.6 with them: latency.
template <int WARPS, int AT_ONCE>
__global__ void __launch_bounds__(32 * WARPS) add_partials(const Partials in, float* first, float* second) {
  __shared__ float red[WARPS][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane, n = col < in.N ? col : col - in.N;
  const bool is = col < in.vectors * in.N;
  const float* from = in.p + (col < in.N ? 0 : in.width) + n;
  const int step = static_cast<int>(in.N % in.E), G = static_cast<int>(in.G);
  const int64_t apart = in.vectors * in.width;
  float a = 0.f;
  if (is) {
    for (int g0 = warp; g0 < G; g0 += WARPS * AT_ONCE) {
      const float* row = from + g0 * apart;
      float v[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j, row += WARPS * apart)
        v[j] = g0 + WARPS * j < G ? row[(in.off + (g0 + WARPS * j) * step) & (in.E - 1)] : 0.f;
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) s += v[j];
      a += s;
    }
  }
  red[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && is) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += red[w][lane];
    if (col < in.N) first[n] = s;
    else second[n] = s;
  }
}

int launch_add_partials(const Partials& in, float* dw, float* db, cudaStream_t s) {
  const int64_t columns = in.vectors * in.N;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ceil_div(columns, 32)));
  // A block of 32 warps fills an SM's registers.  Columns for more than one round of
  // such blocks (the partials are then a row an SM) take half as large ones.
  const bool many = columns > 32LL * sm_count();
  cfg.blockDim = dim3(many ? 512 : 1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, many ? add_partials<16, 10> : add_partials<32, 16>, in, dw ? dw : db, db));
}

// Blocks of rows that the columns' sums are split over, at most: blocks_for's at_once and
// one for each kRun rows of a group, or of a block of 8 rows at once; for any row 4 an SM.
int64_t row_blocks(int64_t M, int64_t N) {
  const int sms = sm_count();
  const int64_t more = N > kHeld ? 0 : M / (N <= kLanes - 7 ? 8 * kRun : kRun);
  return std::min<int64_t>(M + 8, (sms > 0 ? sms : 148) * 4 + more);
}

template <class T, int V, int L, Mode MODE, bool RES>
int launch_bwd_lanes(const BwdP<T>& p, const Rows& rows, int64_t* G, cudaStream_t s) {
  const int per = 256 / L;  // a multiple of 8, as the classes are a divisor of 8
  const int smem = kAhead * 256 * ((RES ? 3 : 2) * V * static_cast<int>(sizeof(T)) + 8);
  auto kernel = bwd_lanes<T, V, L, MODE, RES>;
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return FRAG_ERR_CUDA;
  const int64_t resident = static_cast<int64_t>(sm_count()) * std::min(lane_blocks(V, MODE, 3), kSmem / (smem + 1024));
  *G = std::min(ceil_div(rows.M, per), blocks_for(rows.M, resident, per));
  kernel<<<dim3(static_cast<unsigned>(*G)), 256, smem, s>>>(p, rows);
  return check_launch();
}

// Returns -1, nothing launched, where a row's stage does not fit in shared memory.
template <class T, class W, Mode MODE, bool RES>
int launch_bwd_groups(const BwdP<T>& p, const Rows& rows, int64_t held, int64_t* G, cudaStream_t s) {
  auto kernel = bwd_groups<T, W, MODE, RES>;
  Shape shape;
  int smem = 0;
  *G = plan_groups(rows, held, sizeof(T), RES ? 3 : 2, 1, sizeof(W), 512, 2, 1 << 20, shape, &smem);
  if (!*G) return -1;
  *G = blocks_for(rows.M, *G, shape.groups);
  if (shape.groups > 1) smem = std::max(smem, shape.groups * shape.threads * kV * 8);  // the sums at the end
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem)) return FRAG_ERR_CUDA;
  kernel<<<dim3(static_cast<unsigned>(*G)), shape.groups * shape.threads, smem, s>>>(p, rows, shape,
                                                                                      device_error_word());
  return check_launch();
}

template <class T, Mode MODE, bool RES>
int launch_bwd(const BwdP<T>& p, const Rows& rows, int64_t held, int64_t* G, cudaStream_t s) {
  constexpr Mode LANES = MODE == FULL ? PART : MODE;
  if (held <= 64) return launch_bwd_lanes<T, 8, 8, LANES, RES>(p, rows, G, s);
  if (held <= 128) return launch_bwd_lanes<T, 8, 16, LANES, RES>(p, rows, G, s);
  if (held <= 256) return launch_bwd_lanes<T, 8, 32, LANES, RES>(p, rows, G, s);
  if (held <= kLanes) return launch_bwd_lanes<T, 16, 32, LANES, RES>(p, rows, G, s);
  return by_weight<T>(p.w, {}, [&](auto w) { return launch_bwd_groups<T, decltype(w), MODE, RES>(p, rows, held, G, s); });
}

template <class T>
int backward(BwdP<T> p, int64_t M, float* dw, float* db, cudaStream_t s) {
  Partials sums = {p.partials, 0, p.N, p.N, p.want_dw + p.want_db, 0, 1};
  Layout lay(p.N, sizeof(T));
  lay.add(p.dy, p.ys);
  lay.add(p.x, p.xs);
  lay.add(p.dres, p.rs);
  lay.add(p.dx, p.N);
  const bool edge = lay.off || lay.residue;
  const int64_t held = p.N + (edge ? kE<T> - 1 : 0);
  int64_t G = 0;
  int st = -1;
  if (lay.alike && held <= kHeld) {
    const Rows rows = {M, lay.off, lay.classes()};
    if (edge && held > kLanes) {  // (the groups write their partials by chunks)
      sums.width = p.width = ceil_div(held, kE<T>) * kE<T>;
      sums.off = lay.off;
      sums.E = kE<T>;
    }
    st = by_mode(edge, p.N % (32 * kV) == 0, [&](auto mode) {
      constexpr Mode MODE = decltype(mode)::value;
      return p.dres ? launch_bwd<T, MODE, true>(p, rows, held, &G, s) : launch_bwd<T, MODE, false>(p, rows, held, &G, s);
    });
  }
  if (st < 0) {
    sums.width = p.N;
    sums.E = 1;
    bwd_any_dx<T><<<dim3(static_cast<unsigned>(M)), 256, 0, s>>>(p);
    if (st = check_launch(); st != FRAG_OK || (!dw && !db)) return st;
    const int64_t R = ceil_div(M, std::min(M, static_cast<int64_t>(sm_count()) * 4));
    G = ceil_div(M, R);
    const dim3 grid(static_cast<unsigned>(ceil_div(p.N, 256)), static_cast<unsigned>(G));
    bwd_any_columns<T><<<grid, 256, 0, s>>>(p, M, R);
    st = check_launch();
  }
  if (st != FRAG_OK || (!dw && !db)) return st;
  sums.G = G;
  return launch_add_partials(sums, dw, db, s);
}

}  // namespace
}  // namespace frag

using namespace frag;

extern "C" {

size_t frag_layernorm_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 0;
  return align_up(static_cast<size_t>(row_blocks(M, N)) * 2 * (N + 16) * sizeof(float), 256);
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
  if (sm_count() <= 0) return FRAG_ERR_NO_DEVICE;
  const Vector wv = {w, wdtype == FRAG_DT_F32, aligned16(w)};
  float* ws = static_cast<float*>(workspace);
  if (dtype == FRAG_DT_F32)
    return backward<float>({static_cast<const float*>(dy), static_cast<const float*>(x),
                            static_cast<const float*>(dres), static_cast<float*>(dx), wv, mean, rstd, ws, N, dy_stride,
                            x_stride, dres_stride, N, dw != nullptr, db != nullptr},
                           M, dw, db, s);
  return backward<uint16_t>({static_cast<const uint16_t*>(dy), static_cast<const uint16_t*>(x),
                             static_cast<const uint16_t*>(dres), static_cast<uint16_t*>(dx), wv, mean, rstd, ws, N,
                             dy_stride, x_stride, dres_stride, N, dw != nullptr, db != nullptr},
                            M, dw, db, s);
}

}  // extern "C"

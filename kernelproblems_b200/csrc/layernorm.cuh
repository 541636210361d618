// layernorm.cuh — (residual add +) layer norm, and its gradient with the sums
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
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

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
// widths too.
enum Mode {
  FULL,  // off = 0, P = 1, and every thread has all of its chunks
  PART,  // off = 0, P = 1
  EDGE   // off or N is not a multiple of E
};

template <class T>
constexpr int kE = 16 / sizeof(T);
// A chunk's values, in pairs: fp32 arithmetic takes two in one instruction.
template <class T>
constexpr int kP = kE<T> / 2;

template <class T>
__device__ __forceinline__ void unpack(const uint4& v, float2* f) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int q = 0; q < 4; ++q) f[q] = bf16x2_to_f2(u4_word(v, q));
  } else {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
}
template <class T>
__device__ __forceinline__ uint4 pack(const float2* f) {
  if (sizeof(T) == 2)
    return make_uint4(f2_to_bf16x2(f[0]), f2_to_bf16x2(f[1]), f2_to_bf16x2(f[2 % kP<T>]), f2_to_bf16x2(f[3 % kP<T>]));
  return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
}
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }
__device__ __forceinline__ float& part(float2& v, int i) { return i ? v.y : v.x; }

// Where a thread's chunk lies in its row.
template <class T, Mode MODE>
struct Place {
  int n0;  // its first column
  __device__ __forceinline__ Place(int c, int off) : n0(c * kE<T> - (MODE == EDGE ? off : 0)) {}
  __device__ __forceinline__ bool some(int N) const { return MODE == FULL || n0 < N; }
  __device__ __forceinline__ bool all(int N) const { return MODE == EDGE ? n0 >= 0 && n0 + kE<T> <= N : some(N); }
  __device__ __forceinline__ bool has(int i, int N) const {
    return MODE != EDGE || static_cast<unsigned>(n0 + i) < static_cast<unsigned>(N);
  }
};
// A thread's chunks of a row.
template <class T, Mode MODE>
struct Places {
  int first, step, off;
  __device__ __forceinline__ Place<T, MODE> operator[](int k) const {
    return Place<T, MODE>(first + k * step, off);
  }
};

// Of a chunk that other values share: those outside the row become `other`.
template <class T, Mode MODE>
__device__ __forceinline__ void own_values(const Place<T, MODE>& at, int N, float other, float2* f) {
  if constexpr (MODE == EDGE) {
    if (at.all(N)) return;
#pragma unroll
    for (int i = 0; i < kE<T>; ++i)
      if (!at.has(i, N)) part(f[i / 2], i & 1) = other;
  }
}

template <class T, Mode MODE>
__device__ __forceinline__ void store_chunk(T* row, const Place<T, MODE>& at, int N, float2* f) {
  if (at.all(N)) {
    st_stream(row + at.n0, pack<T>(f));
  } else if (MODE == EDGE && at.some(N)) {
#pragma unroll
    for (int i = 0; i < kE<T>; ++i)
      if (at.has(i, N)) put(row + at.n0 + i, part(f[i / 2], i & 1));
  }
}

// A vector's values at a chunk's columns, 0 outside the row.
template <class T, Mode MODE>
__device__ __forceinline__ void load_vector(const Vector& v, const Place<T, MODE>& at, int N, float none, float2* f) {
  if (v.p && MODE != EDGE && v.aligned && at.some(N)) {
    if (v.f32) {
#pragma unroll
      for (int q = 0; q < kP<T>; q += 2)
        unpack<float>(ld_cached(static_cast<const float*>(v.p) + at.n0 + 2 * q), f + q);
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(v.p) + at.n0;
      if (sizeof(T) == 2) {
        unpack<T>(ld_cached(p), f);
      } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        f[0] = bf16x2_to_f2(u.x);
        f[1] = bf16x2_to_f2(u.y);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kE<T>; ++i) {
    const bool in = at.some(N) && at.has(i, N);
    const int n = in ? at.n0 + i : 0;
    float x = none;
    if (v.p) x = v.f32 ? __ldg(static_cast<const float*>(v.p) + n) : bf16_to_f(__ldg(static_cast<const uint16_t*>(v.p) + n));
    part(f[i / 2], i & 1) = in ? x : 0.f;
  }
}

// A thread's part of a row's two sums, for rows of any length: `term` gives value n's.
// A row of a million values is 4096 a thread, whose squares in one sum would be off by
// up to 1e-4; in runs of 64, added up in 64 bits, by 2e-6.  (4096 rows of 20000 in bf16:
// forward 190 us, gradient 419, with the residual 611 and 471; all in one sum 200, 385, 633
// and 489.)
template <class F>
__device__ __forceinline__ float2 long_sums(int64_t N, F&& term) {
  constexpr int RUN = 64;
  const int64_t apart = blockDim.x;
  double a = 0.0, b = 0.0;
  float2 s = make_float2(0.f, 0.f);
  auto add = [&](int64_t n) {
    const float2 t = term(n);
    s.x += t.x;
    s.y += t.y;
  };
  int64_t n = threadIdx.x;
  if (N > 2 * RUN * apart) {  // (else one run of both)
    for (; n + (RUN - 1) * apart < N; n += RUN * apart) {
#pragma unroll 16
      for (int i = 0; i < RUN; ++i) add(n + i * apart);
      a += s.x;
      b += s.y;
      s = make_float2(0.f, 0.f);
    }
  }
  for (; n < N; n += apart) add(n);
  return make_float2(static_cast<float>(a + s.x), static_cast<float>(b + s.y));
}

// How a launch's rows are dealt out.
struct Rows {
  int64_t M;
  int off;      // of row 0
  int classes;  // P
};

// One of a call's inputs: rows of N values, `stride` apart.
template <class T>
struct Input {
  const T* p;
  int64_t stride;
};

// ------------------------------------------- a thread's own ring: short rows

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// A thread's way down its rows of one input, every `jump`-th value of it: asks for
// the K chunks of a row, to `to`, 256 threads' chunks apart.  A chunk that the row
// shares with another is read whole, except where it reaches out of the tensor:
// rows a whole chunk or more apart, only the first and the last row (`end`) can.
template <class T>
struct Walk {
  const T* next;
  int64_t jump;
  bool apart;
  __device__ __forceinline__ Walk(const Input<T>& in, int64_t row, int64_t rows)
      : next(in.p + row * in.stride), jump(rows * in.stride), apart(in.stride >= kE<T>) {}
  template <int K, Mode MODE>
  __device__ __forceinline__ void ask(const Places<T, MODE>& at, int N, bool end, uint4* to) const {
    const bool inner = MODE != EDGE || (apart && !end);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Place<T, MODE> a = at[k];
      if (!a.some(N)) continue;
      if (inner || a.all(N)) {
        copy_async16(to + k * 256, next + a.n0);
      } else {
        for (int i = 0; i < kE<T>; ++i)
          if (a.has(i, N)) reinterpret_cast<T*>(to + k * 256)[i] = next[a.n0 + i];
      }
    }
  }
};

// The bits of a chunk that are its row's, for a thread whose columns stay.
template <class T, Mode MODE>
struct Bits {
  uint4 mask;
  __device__ __forceinline__ void set(const Place<T, MODE>& at, int N) {
    if constexpr (MODE == EDGE) {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kE<T>; ++i)
        if (at.has(i, N)) w[i * static_cast<int>(sizeof(T)) / 4] |= sizeof(T) == 4 ? ~0u : 0xffffu << (16 * (i & 1));
      mask = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  // Zeros for the values of another row.
  __device__ __forceinline__ uint4 operator()(const uint4& v) const {
    if constexpr (MODE == EDGE)
      return make_uint4(v.x & mask.x, v.y & mask.y, v.z & mask.z, v.w & mask.w);
    else return v;
  }
};

// Sum over groups of L neighbouring lanes.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ------------------------------------------- wider rows: groups of a block's warps

// A block fills an SM.  Its threads make groups, each with rows of its own: 32
// values a thread, a named barrier, and a ring of S stages that the group's first
// thread streams its next rows' windows (their chunks, whole) of up to three
// inputs into by bulk copies.  All rows of a block are of one class, so the groups
// share the weights at their columns in shared memory.  Groups that wait for
// nothing but their own rows fill one another's latencies, and the gradient's sums
// over rows leave an SM as one row of partials.
//
// A window reaches up to 15 bytes past its row on either side.  Where that is not
// the tensor's own memory (before its first value, behind its last) the chunk is
// left out of the copy and its own values are written by the first thread.
constexpr int kV = 32;
struct Shape {
  int groups, threads;  // of a block, of a group
  int stages, slot;     // bytes of a row's window
};

// A group's threads, and a barrier of theirs.
struct Group {
  int index, t, threads;
  __device__ __forceinline__ explicit Group(int n) : threads(n) {
    index = threadIdx.x / n;
    t = threadIdx.x - index * n;
  }
  __device__ __forceinline__ void sync() const {
    if (threads == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(threads) : "memory");
  }
};

// Whether a thread of a group gave up its wait for row i.  All of them leave the loop at
// the same row, behind its barrier: a flag of its own for every other row, as one that is
// already at the next row's wait (and gives up there) must not be heard at this one.  The
// others would go, and it would wait at its barrier for good.
struct Gave {
  int flags[2][32];
  __device__ __forceinline__ void begin(const Group& g) { flags[0][g.index] = flags[1][g.index] = 0; }
  __device__ __forceinline__ void up(const Group& g, int i) { flags[i & 1][g.index] = 1; }
  __device__ __forceinline__ bool is_up(const Group& g, int i) const {
    return *static_cast<const volatile int*>(&flags[i & 1][g.index]);
  }
};

template <class T, int INPUTS, Mode MODE>
struct Ring {
  unsigned char* smem;
  uint64_t* bars;
  int S, slot, count, off, N;
  int64_t r0, step, M;
  Input<T> in[INPUTS];
  int cur, phase;    // the row that every thread is at: its stage, the barrier's parity
  int issued, into;  // thread 0: rows asked for, the next one's stage
  uint32_t bytes;    // of a row's windows

  __device__ __forceinline__ unsigned char* stage(int s) const { return smem + s * (INPUTS * slot); }
  // Chunk c of the current row.
  __device__ __forceinline__ uint4 chunk(int input, int c) const {
    return *reinterpret_cast<const uint4*>(stage(cur) + input * slot + c * 16);
  }

  __device__ __forceinline__ void begin() {  // thread 0
    for (int i = 0; i < S; ++i) mbar_init(&bars[i], 1);
    mbar_init_fence();
  }

  // The next row into the next stage (thread 0).
  __device__ __forceinline__ void issue() {
    if (issued >= count) return;
    uint64_t* bar = &bars[into];
    unsigned char* to = stage(into);
    const int64_t r = r0 + issued * step;
    // (rows a whole chunk or more apart: only the first and the last row's windows
    // can reach out of a tensor)
    bool inner = true;
    if (MODE == EDGE) {
      inner = r > 0 && r < M - 1;
#pragma unroll
      for (int k = 0; k < INPUTS; ++k) inner = inner && in[k].stride >= kE<T>;
    }
    if (inner) {
      mbar_arrive_expect_tx(bar, INPUTS * bytes);
#pragma unroll
      for (int k = 0; k < INPUTS; ++k)
        bulk_g2s_hint(to + k * slot, in[k].p + r * in[k].stride - off, bytes, bar, l2_policy_evict_first());
    } else {
      issue_parts(*this, bar, to, r);
    }
    ++issued;
    into = into + 1 == S ? 0 : into + 1;
  }
  // (by value: the members of the ring that the rows go by stay in registers)
  static __device__ __noinline__ void issue_parts(const Ring ring, uint64_t* bar, unsigned char* to, int64_t r) {
    constexpr int E = kE<T>;
    const int chunks = static_cast<int>(ring.bytes / 16), over = chunks * E - ring.off - ring.N;
    uint32_t expect = 0;
    for (int k = 0; k < INPUTS; ++k) expect += 16 * (chunks - ring.before(k, r) - ring.behind(k, r, over));
    // (a thread's own writes come before its arrival, the bytes are expected
    // before any can come in)
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(expect)
                 : "memory");
    for (int k = 0; k < INPUTS; ++k) {
      const int first = ring.before(k, r), last = chunks - ring.behind(k, r, over);
      const T* from = ring.in[k].p + r * ring.in[k].stride - ring.off;  // the window's begin
      T* own = reinterpret_cast<T*>(to + k * ring.slot);
      if (first)
        for (int n = ring.off; n < E; ++n) own[n] = from[n];
      if (last < chunks)
        for (int n = last * E; n < ring.off + ring.N; ++n) own[n] = from[n];
      bulk_g2s(to + k * ring.slot + first * 16, from + first * E, (last - first) * 16, bar);
    }
    // (the copy of a row S later goes over what was written here)
    proxy_fence_shared();
    mbar_arrive(bar);
  }
  // Whether the window's first, or last, chunk is left out of the copy.
  __device__ __forceinline__ int before(int k, int64_t r) const { return r * in[k].stride < off; }
  __device__ __forceinline__ int behind(int k, int64_t r, int over) const { return (M - 1 - r) * in[k].stride < over; }

  // Waits for the current row (every thread).
  __device__ __forceinline__ bool wait(int* err) { return mbar_wait(&bars[cur], phase, err); }
  __device__ __forceinline__ void next() {
    if (++cur == S) {
      cur = 0;
      phase ^= 1;
    }
  }
  // Waits for what is in flight from row i, the current one, on (thread 0, after a
  // wait ran out).
  __device__ __forceinline__ void drain(int i) {
    for (; i < issued; ++i, next()) mbar_wait(&bars[cur], phase, nullptr);
  }
};

// A group's share of the rows: every n-th of the class, so that what the groups
// are at lies together in memory.
template <class T, int INPUTS, Mode MODE>
__device__ __forceinline__ void deal(Ring<T, INPUTS, MODE>& ring, const Rows& rows, const Shape& shape, int group,
                                     unsigned char* smem, int N) {
  const int P = MODE == EDGE ? rows.classes : 1, cls = MODE == EDGE ? blockIdx.x % P : 0;
  const int stage = INPUTS * shape.slot;
  ring.S = shape.stages;
  ring.slot = shape.slot;
  ring.smem = smem + group * (shape.stages * stage);
  ring.bars = reinterpret_cast<uint64_t*>(smem + shape.groups * (shape.stages * stage)) + group * shape.stages;
  ring.off = MODE == EDGE ? static_cast<int>((rows.off + static_cast<int64_t>(cls) * N) % kE<T>) : 0;
  ring.N = N;
  ring.M = rows.M;
  ring.step = static_cast<int64_t>(gridDim.x) * shape.groups;  // (the grid is a multiple of P)
  ring.r0 = cls + static_cast<int64_t>(P) * (group * (gridDim.x / P) + blockIdx.x / P);
  ring.count = ring.r0 < rows.M ? static_cast<int>((rows.M - ring.r0 + ring.step - 1) / ring.step) : 0;
  ring.bytes = (ring.off + N + kE<T> - 1) / kE<T> * 16;
  ring.cur = ring.phase = ring.issued = ring.into = 0;
}

// A vector at the block's columns, `count` of them, into shared memory; 0 outside
// the row.  W: as fp32, or as bf16 where it is (half the space and accesses, for a
// conversion each time); fp32 values of an 8-value chunk lie in two planes, so that
// neighbouring threads read neighbouring 16 bytes.
template <class T, class W, Mode MODE>
__device__ __forceinline__ void share_vector(const Vector& v, float none, W* to, int count, int off, int N) {
  for (int c = threadIdx.x; c < count / kE<T>; c += blockDim.x) {
    float2 f[kP<T>];
    load_vector<T, MODE == FULL ? PART : MODE>(v, {c, off}, N, none, f);
    uint4* at = reinterpret_cast<uint4*>(to) + c;
    if constexpr (sizeof(W) == 2) {
      *at = pack<T>(f);
    } else {
#pragma unroll
      for (int q = 0; q < kP<T>; q += 2) at[q / 2 * (count / kE<T>)] = pack<float>(f + q);
    }
  }
}
template <class T, class W>
__device__ __forceinline__ void shared_chunk(const W* vector, int count, int c, float2* f) {
  const uint4* at = reinterpret_cast<const uint4*>(vector) + c;
  if constexpr (sizeof(W) == 2) {
    unpack<T>(*at, f);
  } else {
#pragma unroll
    for (int q = 0; q < kP<T>; q += 2) unpack<float>(at[q / 2 * (count / kE<T>)], f + q);
  }
}

// Rows that a thread's own ring holds.
constexpr int kAhead = 3;
// Blocks an SM, as far as registers go: `most` of eight values a lane.
constexpr int lane_blocks(int V, Mode mode, int most) { return most - (V == 8 && mode != EDGE ? 0 : 1); }

// Rows of up to so many values are a few lanes' (16 values a lane, what registers
// hold beside weights and sums), and of up to so many a group's (512 threads of 32).
// 65536 rows in bf16, us by lanes and by groups: of 512 27 and 42 (gradient 39 and
// 56), of 300 36 and 58 (52 and 75); in fp32 of 512 48 and 50 (71 and 72).  4096 rows
// of 16384 by groups 52 (gradient 83), of 20000 by the kernels for any row 190 (419);
// 8192 of 4096 27 and 84 (42 and 152).
constexpr int64_t kLanes = 512, kHeld = 16384;
constexpr int kSmem = 232448;  // of an SM, for its blocks

int group_threads(int64_t held) { return static_cast<int>(ceil_div(held, 32 * kV) * 32); }

// The groups of a launch's blocks, and their stages: as many groups as `most`
// threads are that leave each `least` stages beside `vectors` shared ones, and then
// as many stages as `flight` bytes are.  Returns the blocks, 0 where not one stage
// fits.
int64_t plan_groups(const Rows& rows, int64_t held, int size, int inputs, int vectors, int vector_size, int most,
                    int least, int flight, Shape& shape, int* smem) {
  const int E = 16 / size;
  shape.threads = group_threads(held);
  shape.slot = static_cast<int>(ceil_div(held, E)) * 16;
  const int shared = vectors * shape.threads * kV * vector_size, stage = shape.slot * inputs;
  const int64_t sms = std::max(1, sm_count() / rows.classes) * rows.classes;  // (blocks: a multiple of the classes)
  // (15 named barriers; rows fewer than groups leave some without)
  int groups = std::min(most / shape.threads, shape.threads == 32 ? 32 : 15);
  groups = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(groups, ceil_div(rows.M, sms))));
  for (;; --groups) {
    shape.stages = std::min({8, (kSmem - 2048 - shared) / (stage * groups), std::max(least, flight / (stage * groups))});
    if (shape.stages >= least || groups == 1) break;
  }
  if (shape.stages < 1) return 0;
  shape.groups = groups;
  *smem = shared + groups * shape.stages * (stage + 8);
  return std::min(ceil_div(rows.M, rows.classes) * rows.classes, sms);
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

// The type that a call's weights are kept in, as a constant: bf16 only beside bf16
// rows (of all ones, where there are none).
template <class T, class F>
int by_weight(const Vector& w, const Vector& b, F&& f) {
  if constexpr (sizeof(T) == 2)
    if (!(w.p && w.f32) && !(b.p && b.f32)) return f(uint16_t{});
  return f(float{});
}

// The templates' mode, as a constant.
template <class F>
int by_mode(bool edge, bool full, F&& f) {
  if (edge) return f(std::integral_constant<Mode, EDGE>());
  return full ? f(std::integral_constant<Mode, FULL>()) : f(std::integral_constant<Mode, PART>());
}

bool known(int dtype) { return dtype == FRAG_DT_BF16 || dtype == FRAG_DT_F32; }
bool whole(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == FRAG_DT_F32 ? 4 : 2) == 0; }

}  // namespace
}  // namespace frag

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

#ifndef FWD_V
#define FWD_V 32
#define FWD_REGS 128
#endif
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
    st_global(row + at.n0, pack<T>(f));
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
  for (int i = 0; i < kE<T>; ++i)
    part(f[i / 2], i & 1) = at.some(N) && at.has(i, N) ? vector_at(v, at.n0 + i, none) : 0.f;
}

// How a launch's rows are dealt out.
struct Rows {
  int64_t M;
  int off;       // of row 0
  int classes;   // P
  int64_t each;  // rows of a class that a block takes
};

// One of a call's inputs: rows of N values, `stride` apart.
template <class T>
struct Input {
  const T* p;
  int64_t stride;
};

// Whether a row's chunk c is memory of the tensor from its first value to its
// last (the chunk may be shared with the row before or behind): 0 yes, otherwise
// it is not read as a whole.
__device__ __forceinline__ bool outside(int64_t row, int64_t stride, int64_t M, int before, int behind) {
  return row * stride < before || (M - 1 - row) * stride < behind;
}

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

// Asks for a thread's K chunks of a row, to `to`, 256 threads' chunks apart.
template <class T, int K, Mode MODE>
__device__ __forceinline__ void ask_row(const Input<T>& in, int64_t row, int64_t M, const Places<T, MODE>& at, int N,
                                        uint4* to) {
  const T* from = in.p + row * in.stride;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const Place<T, MODE> a = at[k];
    if (!a.some(N)) continue;
    if (MODE == EDGE && !a.all(N) && outside(row, in.stride, M, max(0, -a.n0), max(0, a.n0 + kE<T> - N))) {
      for (int i = 0; i < kE<T>; ++i)
        if (a.has(i, N)) reinterpret_cast<T*>(to + k * 256)[i] = from[a.n0 + i];
    } else {
      copy_async16(to + k * 256, from + a.n0);
    }
  }
}

// Sum over groups of L neighbouring lanes.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ------------------------------------------- a block's ring: a row a stage

// Thread 0 streams the windows (a row's chunks, whole) of a block's rows of up
// to three inputs into a ring of S stages by bulk copies, one mbarrier a stage.
// A window reaches up to 15 bytes past its row on either side.  Where that is not
// the tensor's own memory (before its first value, behind its last) the chunk is
// left out of the copy and its own values are written by thread 0.
struct RingShape {
  int stages, slot;  // bytes of a row's window
};

template <class T, int INPUTS, Mode MODE>
struct Ring {
  unsigned char* smem;
  uint64_t* bars;
  int S, slot, count, off, N, issued;
  int64_t r0, step, M;
  Input<T> in[INPUTS];

  __device__ __forceinline__ unsigned char* stage(int i) const {
    return smem + static_cast<size_t>(i % S) * (INPUTS * slot);
  }
  __device__ __forceinline__ uint4 chunk(int i, int input, int c) const {
    return *reinterpret_cast<const uint4*>(stage(i) + input * slot + c * 16);
  }
  __device__ __forceinline__ int64_t row(int i) const { return r0 + i * step; }

  __device__ __forceinline__ void begin() {  // thread 0
    for (int i = 0; i < S; ++i) mbar_init(&bars[i], 1);
    mbar_init_fence();
  }

  // Row i into its stage (thread 0).
  __device__ __forceinline__ void issue(int i) {
    if (i >= count) return;
    uint64_t* bar = &bars[i % S];
    unsigned char* to = stage(i);
    const int64_t r = row(i);
    if (MODE != EDGE) {
      mbar_arrive_expect_tx(bar, INPUTS * slot);
#pragma unroll
      for (int k = 0; k < INPUTS; ++k) bulk_g2s(to + k * slot, in[k].p + r * in[k].stride, slot, bar);
    } else {
      constexpr int E = kE<T>;
      const int chunks = (off + N + E - 1) / E, over = chunks * E - off - N;
      uint32_t bytes = 0;
#pragma unroll
      for (int k = 0; k < INPUTS; ++k) bytes += 16 * (chunks - ends(k, r, over, false) - ends(k, r, over, true));
      // (a thread's own writes come before its arrival, the bytes are expected
      // before any can come in)
      asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
                   : "memory");
#pragma unroll
      for (int k = 0; k < INPUTS; ++k) {
        const int first = ends(k, r, over, false), last = chunks - ends(k, r, over, true);
        const T* from = in[k].p + r * in[k].stride - off;  // the window's begin
        T* own = reinterpret_cast<T*>(to + k * slot);
        if (first)
          for (int n = off; n < E; ++n) own[n] = from[n];
        if (last < chunks)
          for (int n = last * E; n < off + N; ++n) own[n] = from[n];
        bulk_g2s(to + k * slot + first * 16, from + first * E, (last - first) * 16, bar);
      }
      mbar_arrive(bar);
    }
    issued = i + 1;
  }
  // Whether the window's first (or last) chunk is left out of the copy.
  __device__ __forceinline__ int ends(int k, int64_t r, int over, bool last) const {
    return last ? (M - 1 - r) * in[k].stride < over : r * in[k].stride < off;
  }

  // Waits for row i (every thread).
  __device__ __forceinline__ bool wait(int i, int* err) { return mbar_wait(&bars[i % S], (i / S) & 1, err); }
  // Waits for what is in flight from row i on (thread 0, after a wait ran out).
  __device__ __forceinline__ void drain(int i) {
    for (; i < issued; ++i) mbar_wait(&bars[i % S], (i / S) & 1, nullptr);
  }
};

// A block's share of the rows: `each` of one class.
template <class T, int INPUTS, Mode MODE>
__device__ __forceinline__ void deal(Ring<T, INPUTS, MODE>& ring, const Rows& rows, const RingShape& shape,
                                     unsigned char* smem, int N) {
  const int cls = MODE == EDGE ? blockIdx.x % rows.classes : 0;
  ring.smem = smem;
  ring.S = shape.stages;
  ring.slot = shape.slot;
  ring.bars = reinterpret_cast<uint64_t*>(smem + static_cast<size_t>(shape.stages) * (INPUTS * shape.slot));
  ring.off = MODE == EDGE ? static_cast<int>((rows.off + static_cast<int64_t>(cls) * N) % kE<T>) : 0;
  ring.N = N;
  ring.M = rows.M;
  ring.step = rows.classes;
  ring.r0 = blockIdx.x / rows.classes * rows.each * rows.classes + cls;
  ring.count = ring.r0 < rows.M
                   ? static_cast<int>(min(rows.each, (rows.M - ring.r0 + rows.classes - 1) / rows.classes)) : 0;
  ring.issued = 0;
}

// Rows that a thread's own ring holds.
constexpr int kAhead = 4;
// Blocks an SM, as far as registers go: `most` of eight values a lane.
constexpr int lane_blocks(int V, Mode mode, int most) { return most - (V == 8 && mode != EDGE ? 0 : 1); }

// Rows of up to so many values are a few lanes', and a block's.
constexpr int64_t kLanes = 512, kHeld = 16384;
constexpr int kSmem = 232448;  // of an SM, for its blocks

int ring_threads(int64_t held) { return static_cast<int>(ceil_div(held, 512) * 32); }
// Blocks of a ring kernel that an SM's registers hold.
int ring_blocks(int threads, int registers) { return std::max(1, std::min(12, 65536 / (registers * threads))); }

// The ring of a launch and its blocks: as many an SM as leave each two stages, and
// then as many stages as fit.  Returns the blocks, 0 where not one stage fits.
int64_t plan_ring(Rows& rows, RingShape& shape, int* smem, int inputs, int slot, int per_sm) {
  const int stage = slot * inputs;
  shape.slot = slot;
  for (;; --per_sm) {
    shape.stages = std::min(8, (kSmem / per_sm - 2048) / stage);  // (1 KB is the system's, 1 the rest of the block's)
    if (shape.stages >= 2 || per_sm == 1) break;
  }
  if (shape.stages < 1) return 0;
  *smem = shape.stages * stage + 8 * shape.stages;
  const int64_t of_class = ceil_div(rows.M, rows.classes);
  const int64_t resident = std::max(1, sm_count() * per_sm / rows.classes);
  rows.each = ceil_div(of_class, std::min(of_class, resident));
  return ceil_div(of_class, rows.each) * rows.classes;
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

// orthogonal_small.cu — the Newton-Schulz chain of matrices with a side of at
// most 128, one cluster of blocks a matrix, in one launch.
//
// Block c of the cluster holds up to 256 columns of X (taken as s <= 128 rows
// of the long side l; a tall matrix is read transposed) as hi and lo in shared
// memory, from the first step to the last:
//   A  each block multiplies its columns into a partial X X' (tensor memory ->
//      shared memory), sums every C-th column of all blocks' partials in block
//      order over the cluster, and writes it, a row of the symmetric A, to all
//   B  every block makes b A + c A A for itself, in A's place
//   X  every block updates its own columns where they are
// Only A crosses blocks: two or three cluster barriers a step, nothing in global
// memory.
//
// Results in bf16 take the chain's arithmetic (single fp16 operands, B's
// diagonal in 32 bits): an error of 0.6 to 1.5e-3 under a rounding of 1.7e-3.
// Where the result is stored in 32 bits (FINE), A and B are kept as two fp16
// numbers like X and each product takes hi hi, hi lo and lo hi: 1.5 to 1.7e-6 of
// the step at 96 x 160 and 128 x 2048, for 12 to 25 us more.  X's lo is an operand there and not scaled up: an
// element of X is off by up to 2^-33, which shows where the norm is far below eps.
//
// The same 64-column block of X is A's K-major operand (rows of k) and X's
// MN-major one (rows across k), so it is stored once.
//
// Bound: latency.  A step takes 4 us in one block (96 x 160: 31 us for five
// steps and the rest) and 9 over eight (128 x 2048: 59), where the sum of A over
// the cluster is the larger part; the launch, reading the matrix and writing the
// result take 11 to 15.  The same sizes through orthogonal.cu's chain: 92, 128.
#include <algorithm>
#include <mutex>

#include "orthogonal.cuh"

namespace frag {
namespace {

constexpr int kSide = 128;
constexpr int kMaxBlocks = 4;                 // of 64 columns a block holds
constexpr int kBlock = kSide * 64 * 2;        // bytes of one, 16 bits
constexpr int kPart = kSide * kSide * 4;      // partial A, columns of 128 rows; then A's (and B's) lo
constexpr int kASize = kSide * kSide * 2;     // hi of A, then of B: two 64-column blocks
constexpr int kSmallThreads = 256;
constexpr int kMaxCluster = 16;

struct SmallP {
  PrepP prep;
  ResultP res;
  int s, l, tall, blocks, steps;  // blocks: of 64 columns in each block of the cluster
  int* err;
  float co[3 * kMaxSteps];
};

struct SmallShared {
  uint64_t bar;
  uint32_t tmem;
  int abort;
  float slots[2][32];
  float sum;           // of this block's squares
  float2 coef[kSide];  // hi's and lo's factors by row (not FINE)
};

__device__ __forceinline__ uint32_t small_tail(int blocks) { return 2 * blocks * kBlock + kPart + kASize; }

// How a block's threads walk its part of the matrix in memory order: lines
// (matrix rows) over warps, V neighbouring elements a lane, N pieces of work
// in flight a thread.  A line is a row of X, or a column when it is tall.
template <int V>
struct Walk {
  static constexpr int kLines = V == 8 ? 8 : 2, kSteps = V == 8 ? 1 : 8;
  int lines, length, per, first;  // per: lines of a warp's pass
  __device__ Walk(const SmallP& p, int cols) {
    lines = p.tall ? cols : p.s;
    length = p.tall ? p.s : cols;
    per = V == 8 && p.tall ? 2 : 1;  // 128 elements are half a warp's
    first = (threadIdx.x >> 5) * per + (per == 2 ? (threadIdx.x & 31) >> 4 : 0);
  }
  __device__ int stride() const { return per * (kSmallThreads / 32); }
  __device__ int pos(int b) const { return (per == 2 ? threadIdx.x & 15 : (threadIdx.x & 31) + 32 * b) * V; }
};

// Place of X's element (i, j) in hi's (or lo's) columns.
__device__ __forceinline__ uint32_t place(int i, int j) { return unit((j >> 6) * kBlock, i, (j & 63) >> 3) + (j & 7) * 2; }

template <int V, int MODE>
__device__ __forceinline__ void small_out(const SmallP& p, uint32_t hi, uint32_t lo, int e, int c0, int cols) {
  const ResultP& q = p.res;
  const Walk<V> w(p, cols);
  for (int l0 = w.first; l0 - w.first < w.lines; l0 += w.kLines * w.stride()) {
    float old[w.kLines][w.kSteps][V];
    if (MODE == UPDATE) {
#pragma unroll
      for (int a = 0; a < w.kLines; ++a)
#pragma unroll
        for (int b = 0; b < w.kSteps; ++b) {
          const int line = l0 + a * w.stride(), pos = w.pos(b);
          if (line < w.lines && pos < w.length)
            load_elems<V>(q.par, e * q.par.sb + static_cast<int64_t>(p.tall ? c0 + line : line) * q.par.sr +
                                     static_cast<int64_t>(p.tall ? pos : c0 + pos) * q.par.sc, old[a][b]);
        }
    }
#pragma unroll
    for (int a = 0; a < w.kLines; ++a)
#pragma unroll
      for (int b = 0; b < w.kSteps; ++b) {
        const int line = l0 + a * w.stride(), pos = w.pos(b);
        if (line >= w.lines || pos >= w.length) continue;
        float v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          // the first four floats of an 8-column unit lie in hi's place, the others in lo's
          const int i = p.tall ? pos + k : line, j = p.tall ? line : pos + k;
          v[k] = ld_shared_f(unit((j & 4 ? lo : hi) + (j >> 6) * kBlock, i, (j & 63) >> 3) + (j & 3) * 4) *
                 (1.0f / kXScale);
          if (MODE == UPDATE) v[k] = q.keep * old[a][b][k] - q.rate * v[k];
        }
        store_elems<V>(q.out, e * q.out.sb + static_cast<int64_t>(p.tall ? c0 + line : line) * q.out.sr +
                                  (p.tall ? pos : c0 + pos), v);
      }
  }
}

// Reads the block's part of the matrix (and makes the new momentum), returns
// this thread's sum of squares; a value's 32 bits wait in hi's and lo's places
// until the norm is known.
template <int V>
__device__ __forceinline__ float small_in(const SmallP& p, uint32_t hi, uint32_t lo, int e, int c0, int cols) {
  const PrepP& q = p.prep;
  const Walk<V> w(p, cols);
  float ss = 0.f;
  for (int l0 = w.first; l0 - w.first < w.lines; l0 += w.kLines * w.stride()) {
    float v[w.kLines][w.kSteps][V], m[w.kLines][w.kSteps][V];
#pragma unroll
    for (int a = 0; a < w.kLines; ++a)
#pragma unroll
      for (int b = 0; b < w.kSteps; ++b) {
        const int line = l0 + a * w.stride(), pos = w.pos(b);
        if (line < w.lines && pos < w.length)
          prep_value<V>(q, e, p.tall ? c0 + line : line, p.tall ? pos : c0 + pos, v[a][b], m[a][b]);
      }
#pragma unroll
    for (int a = 0; a < w.kLines; ++a)
#pragma unroll
      for (int b = 0; b < w.kSteps; ++b) {
        const int line = l0 + a * w.stride(), pos = w.pos(b);
        if (line >= w.lines || pos >= w.length) continue;
        if (q.has_mom)
          store_elems<V>(q.mom_out, e * q.mom_out.sb + static_cast<int64_t>(p.tall ? c0 + line : line) * q.mom_out.sr +
                                        (p.tall ? pos : c0 + pos), m[a][b]);
        uint32_t bits[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          ss = fmaf(v[a][b][k], v[a][b][k], ss);
          bits[k] = __float_as_uint(v[a][b][k]);
        }
        if (V == 8 && !p.tall) {
          uint32_t h[4], l[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t x = bits[(2 * k) % V], y = bits[(2 * k + 1) % V];
            h[k] = x >> 16 | (y & 0xffff0000u);
            l[k] = (x & 0xffffu) | y << 16;
          }
          st_shared(hi + place(line, pos), make_uint4(h[0], h[1], h[2], h[3]));
          st_shared(lo + place(line, pos), make_uint4(l[0], l[1], l[2], l[3]));
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const uint32_t o = p.tall ? place(pos + k, line) : place(line, pos + k);
            st_shared_h(hi + o, __ushort_as_half(static_cast<unsigned short>(bits[k] >> 16)));
            st_shared_h(lo + o, __ushort_as_half(static_cast<unsigned short>(bits[k])));
          }
        }
      }
  }
  return ss;
}

template <int V, bool FINE>
__global__ void __launch_bounds__(kSmallThreads, 1) small_chain(const __grid_constant__ SmallP p, int C) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t hi = smem_u32(smem_raw), lo = hi + p.blocks * kBlock, part = lo + p.blocks * kBlock;
  const uint32_t am = part + kPart, al = part;  // A's hi and lo
  SmallShared& sh = *reinterpret_cast<SmallShared*>(smem_raw + small_tail(p.blocks));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int quad = warp & 3, half = warp >> 2, r = quad * 32 + lane;
  constexpr float lo_scale = FINE ? 1.0f : kLoScale;  // of X's lo
  const int c = static_cast<int>(blockIdx.x) % C, e = static_cast<int>(blockIdx.x) / C;
  const int c0 = c * p.blocks * 64, cols = max(0, min(p.blocks * 64, p.l - c0));
  volatile int* const abort_flag = &sh.abort;

  if (threadIdx.x == 0) {
    sh.abort = 0;
    mbar_init(&sh.bar, 1);
    mbar_init_fence();
  }
  if (warp == 0) tmem_alloc<1>(&sh.tmem, 512);
  // zeros past the matrix's rows and columns
  for (int i = threadIdx.x; i < static_cast<int>(small_tail(p.blocks)) / 16; i += kSmallThreads)
    st_shared(hi + i * 16, make_uint4(0, 0, 0, 0));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  float ss = small_in<V>(p, hi, lo, e, c0, cols);
  ss = block_sum(ss, sh.slots, 0);
  if (threadIdx.x == 0) sh.sum = ss;
  cluster_sync();
  if (C > 1) {
    ss = 0.f;
    for (int q = 0; q < C; ++q) ss += ld_cluster_f(cluster_address(smem_u32(&sh.sum), q));
  }
  const float f = kXScale / (sqrtf(ss) + p.prep.eps);
  for (int i = threadIdx.x; i < p.blocks * (kBlock / 16); i += kSmallThreads) {
    const uint4 a = ld_shared(hi + i * 16), b = ld_shared(lo + i * 16);
    uint4 oh, ol;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t aw = u4_word(a, w), bw = u4_word(b, w);
      const float x0 = __uint_as_float(aw << 16 | (bw & 0xffffu)) * f;
      const float x1 = __uint_as_float((aw & 0xffff0000u) | bw >> 16) * f;
      const __half2 h = __floats2half2_rn(x0, x1);
      const float2 back = __half22float2(h);
      const __half2 rest = __floats2half2_rn((x0 - back.x) * lo_scale, (x1 - back.y) * lo_scale);
      reinterpret_cast<uint32_t*>(&oh)[w] = *reinterpret_cast<const uint32_t*>(&h);
      reinterpret_cast<uint32_t*>(&ol)[w] = *reinterpret_cast<const uint32_t*>(&rest);
    }
    st_shared(hi + i * 16, oh);
    st_shared(lo + i * 16, ol);
  }

  uint32_t phase = 0;
  // what the block has written to shared memory is seen by thread 0's products
  auto publish = [&]() {
    proxy_fence_shared();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  auto wait = [&]() {  // the products are done (bounded; after that the block only keeps step with the others)
    if (!*abort_flag && !mbar_wait(&sh.bar, phase, p.err)) *abort_flag = 1;
    phase ^= 1;
    __syncwarp();
    tc_fence_after();
  };
  const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  const int k16 = (p.s + 15) / 16;
  // eight values' hi and lo in two units (the lo of A and B is used if FINE)
  auto split8 = [](const float* v, uint4& oh, uint4& ol) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const __half2 t = __floats2half2_rn(v[2 * q], v[2 * q + 1]);
      const float2 back = __half22float2(t);
      const __half2 rest = __floats2half2_rn((v[2 * q] - back.x) * lo_scale, (v[2 * q + 1] - back.y) * lo_scale);
      reinterpret_cast<uint32_t*>(&oh)[q] = *reinterpret_cast<const uint32_t*>(&t);
      reinterpret_cast<uint32_t*>(&ol)[q] = *reinterpret_cast<const uint32_t*>(&rest);
    }
  };
  constexpr float a_scale = kAScale / (kXScale * kXScale);
  // operands: X's columns along and across k, A and B (and their lo); a block
  // of 64 columns further is kBlock / 16 more
  const uint64_t xh = smem_desc(hi, false), xl = smem_desc(lo, false);
  const uint64_t yh = smem_desc(hi, true, kBlock), yl = smem_desc(lo, true, kBlock);
  const uint64_t ah = smem_desc(am, false), ax = smem_desc(al, false);
  constexpr uint64_t kNext = kBlock >> 4;
  const uint32_t id_a = instr_desc_f16(kSide, kSide, false, false);
  const uint32_t id_x = instr_desc_f16(kSide, 64 * p.blocks, false, true);

  for (int step = 0; step < p.steps; ++step) {
    const float ca = p.co[3 * step], cb = p.co[3 * step + 1], cc = p.co[3 * step + 2] / kAScale;
    // ---- A = X X'
    publish();
    if (threadIdx.x == 0) {
      uint64_t o = 0;
      for (int b = 0; b < p.blocks; ++b, o += kNext)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint64_t h = xh + o + 2 * k, l = xl + o + 2 * k;
          mma_f16<1>(tmem, h, h, id_a, b + k > 0);
          if (!FINE) continue;
          mma_f16<1>(tmem, h, l, id_a, true);
          mma_f16<1>(tmem, l, h, id_a, true);
        }
      mma_commit<1>(&sh.bar);
    }
    wait();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float v[32];
      tmem_load32(lanes + half * 64 + g * 32, v);
      if (C == 1) {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] *= a_scale;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint4 oh = pack_h8(v + 8 * u), ol;
          if (FINE) split8(v + 8 * u, oh, ol);
          st_shared(unit(am + half * kBlock, r, g * 4 + u), oh);
          if (FINE) st_shared(unit(al + half * kBlock, r, g * 4 + u), ol);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(part + ((half * 64 + g * 32 + k) * kSide + r) * 4), "f"(v[k])
                       : "memory");
      }
    }
    if (C > 1) {
      cluster_sync();
      // columns c, c + C, ... of all partials, at most eight a warp: rows of A
      constexpr int kRowsOfWarp = 8;
      float4 t[kRowsOfWarp];
#pragma unroll
      for (int n = 0; n < kRowsOfWarp; ++n) {
        const int j = c + C * (warp + n * (kSmallThreads / 32));
        t[n] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j >= p.s) continue;
        const uint32_t from = part + (j * kSide + 4 * lane) * 4;
        for (int q0 = 0; q0 < C; q0 += 8) {
          float4 x[8];
#pragma unroll
          for (int q = 0; q < 8; ++q)
            x[q] = q0 + q < C ? ld_cluster_f4(cluster_address(from, q0 + q)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int q = 0; q < 8; ++q) t[n].x += x[q].x, t[n].y += x[q].y, t[n].z += x[q].z, t[n].w += x[q].w;
        }
      }
      if (FINE) cluster_sync();  // every partial is read: lo takes its place
#pragma unroll
      for (int n = 0; n < kRowsOfWarp; ++n) {
        const int j = c + C * (warp + n * (kSmallThreads / 32));
        if (j >= p.s) continue;
        const float v[8] = {t[n].x * a_scale, t[n].y * a_scale, t[n].z * a_scale, t[n].w * a_scale, 0.f, 0.f, 0.f, 0.f};
        uint4 oh, ol;
        split8(v, oh, ol);
        const uint32_t to = unit((lane >> 4) * kBlock, j, (lane & 15) >> 1) + (lane & 1) * 8;
        for (int q = 0; q < C; ++q) {
          st_cluster_u2(cluster_address(am + to, q), oh.x, oh.y);
          if (FINE) st_cluster_u2(cluster_address(al + to, q), ol.x, ol.y);
        }
      }
      // rows past the matrix hold partials where lo has to be zero
      for (int i = threadIdx.x; FINE && i < 2 * (kSide - p.s) * 8; i += kSmallThreads)
        st_shared(al + (i / ((kSide - p.s) * 8)) * kBlock + p.s * 128 + (i % ((kSide - p.s) * 8)) * 16,
                  make_uint4(0, 0, 0, 0));
      proxy_fence();
      cluster_sync();
    }
    // ---- B = b A + c A A
    publish();
    if (threadIdx.x == 0) {
      for (int k = 0; k < k16; ++k) {
        const uint64_t o = (k >> 2) * kNext + (k & 3) * 2;
        mma_f16<1>(tmem + kSide, ah + o, ah + o, id_a, k > 0);
        if (!FINE) continue;
        mma_f16<1>(tmem + kSide, ah + o, ax + o, id_a, true);
        mma_f16<1>(tmem + kSide, ax + o, ah + o, id_a, true);
      }
      mma_commit<1>(&sh.bar);
    }
    wait();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float v[32];
      tmem_load32(lanes + kSide + half * 64 + g * 32, v);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t uh = unit(am + half * kBlock, r, g * 4 + u), ul = unit(al + half * kBlock, r, g * 4 + u);
        const uint4 h = ld_shared(uh), l = FINE ? ld_shared(ul) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t hw = u4_word(h, q), lw = u4_word(l, q);
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&hw));
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&lw));
          v[8 * u + 2 * q] = fmaf(v[8 * u + 2 * q], cc, cb * (FINE ? x.x + y.x : x.x));
          v[8 * u + 2 * q + 1] = fmaf(v[8 * u + 2 * q + 1], cc, cb * (FINE ? x.y + y.y : x.y));
        }
        uint4 oh = pack_h8(v + 8 * u), ol;
        if (FINE) split8(v + 8 * u, oh, ol);
        st_shared(uh, oh);
        if (FINE) st_shared(ul, ol);
      }
      const int j = half * 64 + g * 32;
      if (!FINE && r >= j && r < j + 32) {
        float d = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) d = j + k == r ? v[k] : d;
        const float rest = d - __half2float(__float2half_rn(d));
        sh.coef[r] = make_float2(ca + rest * (1.0f / kAScale),
                                 (step >= p.steps - 2 ? ca + d * (1.0f / kAScale) : ca) * (1.0f / lo_scale));
      }
    }
    // ---- X = a X + B X
    publish();
    if (threadIdx.x == 0) {
      for (int k = 0; k < k16; ++k) {
        const uint64_t o = (k >> 2) * kNext + (k & 3) * 2, ox = static_cast<uint64_t>(k) * 128;
        mma_f16<1>(tmem + 2 * kSide, ah + o, yh + ox, id_x, k > 0);
        if (!FINE) continue;
        mma_f16<1>(tmem + 2 * kSide, ax + o, yh + ox, id_x, true);
        mma_f16<1>(tmem + 2 * kSide, ah + o, yl + ox, id_x, true);
      }
      mma_commit<1>(&sh.bar);
    }
    wait();
    const bool last = step + 1 == p.steps;
    const float2 coef = FINE ? make_float2(ca, ca) : sh.coef[r], k2 = make_float2(1.0f / kAScale, 1.0f / kAScale);
    const float2 fh = make_float2(coef.x, coef.x), fl = make_float2(coef.y, coef.y);
    for (int b = 0; b < p.blocks; ++b) {
      float v[32];
      tmem_load32(lanes + 2 * kSide + b * 64 + half * 32, v);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t uh = unit(hi + b * kBlock, r, half * 4 + u), ul = unit(lo + b * kBlock, r, half * 4 + u);
        const uint4 h = ld_shared(uh), l = ld_shared(ul);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t hw = u4_word(h, q), lw = u4_word(l, q);
          float2* y = reinterpret_cast<float2*>(v + 8 * u + 2 * q);
          *y = __ffma2_rn(__half22float2(*reinterpret_cast<const __half2*>(&lw)), fl, __fmul2_rn(*y, k2));
          *y = __ffma2_rn(__half22float2(*reinterpret_cast<const __half2*>(&hw)), fh, *y);
        }
        uint4 oh, ol;
        const float* y = v + 8 * u;
        if (last) {  // 32 bits a value: four in each place
          oh = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
          ol = make_uint4(__float_as_uint(y[4]), __float_as_uint(y[5]), __float_as_uint(y[6]), __float_as_uint(y[7]));
        } else {
          split8(y, oh, ol);
        }
        st_shared(uh, oh);
        st_shared(ul, ol);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (p.res.last == UPDATE) small_out<V, UPDATE>(p, hi, lo, e, c0, cols);
  else small_out<V, LAST>(p, hi, lo, e, c0, cols);
  if (warp == 0) {
    __syncwarp();
    tmem_free<1>(tmem, 512);
  }
  cluster_sync();  // no block leaves while another may still read its shared memory
}

int small_smem(int blocks) { return 2 * blocks * kBlock + kPart + kASize + static_cast<int>(sizeof(SmallShared)); }

void cluster_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int grid, int C, int smem, cudaStream_t s) {
  cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(C);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
}

// Whether a cluster of C blocks fits on the device (asked once for each C).
bool cluster_fits(int C) {
  static std::mutex mu;
  static int known[64][kMaxCluster + 1] = {};  // 1: no, 2: yes
  const int d = current_device();
  if (d < 0 || d >= 64) return false;
  std::lock_guard<std::mutex> lk(mu);
  if (known[d][C]) return known[d][C] == 2;
  for (const void* kern :
       {reinterpret_cast<const void*>(small_chain<1, false>), reinterpret_cast<const void*>(small_chain<1, true>),
        reinterpret_cast<const void*>(small_chain<8, false>), reinterpret_cast<const void*>(small_chain<8, true>)}) {
    if (!allow_dynamic_smem(kern, small_smem(kMaxBlocks))) return false;
    if (C > 8 && cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
  }
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[1];
  cluster_config(cfg, attr, C, C, small_smem(kMaxBlocks), nullptr);
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, small_chain<8, true>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return false;  // asked again by the next call
  }
  known[d][C] = n > 0 ? 2 : 1;
  return n > 0;
}

// Blocks of a cluster whose matrix has this long side.
int cluster_blocks(int64_t longer) { return static_cast<int>(ceil_div(ceil_div(longer, 64), kMaxBlocks)); }

}  // namespace

bool small_takes(int64_t m, int64_t n) {
  const int64_t longer = std::max(m, n);
  return std::min(m, n) <= kSide && longer <= static_cast<int64_t>(kMaxCluster) * kMaxBlocks * 64 &&
         cluster_fits(cluster_blocks(longer));
}

int orthogonalise_small(const PrepP& prep, int64_t E, int steps, const float* co, const ResultP& res, cudaStream_t s) {
  const int64_t small = std::min(prep.rows, prep.cols), longer = std::max(prep.rows, prep.cols);
  const int C = cluster_blocks(longer);
  SmallP p = {};
  p.prep = prep;
  p.res = res;
  p.s = static_cast<int>(small);
  p.l = static_cast<int>(longer);
  p.tall = prep.rows > prep.cols;
  p.blocks = static_cast<int>(ceil_div(ceil_div(longer, 64), C));
  p.steps = steps;
  p.err = device_error_word();
  for (int i = 0; i < 3 * steps; ++i) p.co[i] = co[i];
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[1];
  cluster_config(cfg, attr, static_cast<int>(E) * C, C, small_smem(p.blocks), s);
  const int64_t m = prep.rows, n = prep.cols;
  const bool wide_access = chunked(prep.g, E, m, n) && chunked(res.out, E, m, n) &&
                           (res.last != UPDATE || chunked(res.par, E, m, n)) &&
                           (!prep.has_mom || (chunked(prep.mom, E, m, n) && chunked(prep.mom_out, E, m, n)));
  auto kern = res.out.f32 ? (wide_access ? small_chain<8, true> : small_chain<1, true>)
                          : (wide_access ? small_chain<8, false> : small_chain<1, false>);
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p, C));
}

}  // namespace frag

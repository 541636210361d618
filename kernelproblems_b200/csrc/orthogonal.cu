// orthogonal.cu — Newton-Schulz orthogonalisation of a gradient and the weight
// update made of it.
//
// Math (s = the smaller side, X = G / (|G|_F + eps), quintic step (a, b, c)):
//   A = X X' (s x s; X'X when the matrix is tall),  B = b A + c A A
//   X <- a X + B X  (X B when tall), `steps` times
// Singular vectors stay, singular values go towards 1.  muon: momentum
// m' = mu m + (1 - mu) g, u = mu m' + (1 - mu) g (or m'), and
// p' = (1 - lr wd) p - lr scale O(u).
//
// Products run on the tensor cores with fp16 operands and fp32 accumulators.
// What the 16 bits are, and why it is enough:
//  - X = hi + lo, two fp16 numbers: 22 bits where |x| is above 2^-22, 2^-44
//    below (an element of the largest matrices is 2^-16).  a X uses both, B X
//    uses hi: an error of B X lies along directions that are already large, which later
//    steps do not amplify, while an error of a X is multiplied by a^5 = 485
//    along small ones.  On a gradient of 16 strong directions and a rest of 2%
//    (512 x 2048), relative error of the result against 64 bits: bf16
//    throughout 0.27, one fp16 0.035, hi + lo 0.0003.
//  - everything is kept times a power of two (X 2^8, A and B 2^10), so that
//    the first step's small entries (1/sqrt(mn) of a unit norm) stay clear of
//    fp16's subnormals, and the largest (|B| <= 24 for steep schedules) of 65504;
//    lo times another 2^11.  Where the norm is far below eps, X stays small
//    through all steps and hi is subnormal; lo carries it then.
//  - B's diagonal (near -2.7 at the end, against small off-diagonal entries)
//    carries most of B's rounding error: its residual is kept in 32 bits and
//    added in the epilogue, as is the diagonal's product with lo in the last
//    two steps (earlier, lo along small directions would be amplified).
#include <math.h>

#include <algorithm>
#include <mutex>

#include "orthogonal.cuh"

namespace frag {

bool make_map_3d(CUtensorMap* map, const void* base, int64_t x, int64_t y, int64_t z, int64_t stride_y,
                 int64_t stride_z, int box_x, int box_y) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::mutex mu;
  static Encode encode = nullptr;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!encode) {
      void* fn = nullptr;
      cudaDriverEntryPointQueryResult how;
      const cudaError_t e =
          cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &how);
      if (e != cudaSuccess || how != cudaDriverEntryPointSuccess) {
        set_last_cuda_error(e == cudaSuccess ? cudaErrorUnknown : e);
        cudaGetLastError();
        return false;
      }
      encode = reinterpret_cast<Encode>(fn);
    }
  }
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(x), static_cast<cuuint64_t>(y), static_cast<cuuint64_t>(z)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride_y) * 2, static_cast<cuuint64_t>(stride_z) * 2};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_x), static_cast<cuuint32_t>(box_y), 1};
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r =
      encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_cuda_error(cudaErrorInvalidValue);
    return false;
  }
  return true;
}

namespace {

constexpr int kRows = 128;          // rows of C a block holds
constexpr int kChunk = 64;          // columns the epilogue takes at a time
constexpr int kOperand = 128 * kTileK * 2;  // bytes of one operand of a stage
constexpr int kStageBytes = 2 * kOperand;
constexpr int kSet = 2 * kRows * kChunk * 2;  // two 16-bit chunks
// Shared memory: stages of operands and sets of chunks.  Five stages and two
// sets take 7 to 13% longer below 1100 x 1100: chunks then wait for stores.
constexpr int kStages = 4, kSets = 3;
constexpr int kEpiWarps = 8;
// a loading warp, an issuing warp, the epilogue, and a warp that moves its chunks
constexpr int kThreads = 64 + 32 * kEpiWarps + 32;

struct ChainP {
  // X's two buffers by 64 columns x 128 rows and by 64 x 64, lo, A and B
  CUtensorMap xk[2], xm[2], lo, ak, bk, a64, b64;
  int m, n, s, l, E, tall, steps, split, narrow;
  float2* diag;        // [E, s] B's diagonal in 32 bits and its rounding residual
  float* partials;     // split GRAM sums
  unsigned* counters;  // finished phases of all blocks, abort, and arrived parts of each split tile
  ResultP res;
  int* err;
  float co[3 * kMaxSteps];
};

// One phase's product C[i, j] = sum_k P[i, k] Q[j, k] as a list of work items:
// tiles of TM rows and `tn` columns.  A symmetric product takes the tiles that
// reach the diagonal or lie below it; a narrow one (pairs of blocks, 128
// columns) has twice as many of them.
template <int CG>
struct Work {
  static constexpr int TM = kRows * CG, TN = 128 * CG;
  int I, J, ks, split, ti_count, tj_count, per, items, E, tn, ratio;
  bool sym, cols_fast;
  __device__ Work(const ChainP& p, int mode) {
    sym = mode == GRAM || mode == POLY;
    I = sym ? p.s : p.m;
    J = sym ? p.s : p.n;
    E = p.E;
    ks = ((mode == GRAM ? p.l : p.s) + kTileK - 1) / kTileK;
    split = mode == GRAM ? p.split : 1;
    ratio = CG == 2 && sym && p.narrow ? 2 : 1;
    tn = TN / ratio;
    ti_count = (I + TM - 1) / TM;
    tj_count = (J + tn - 1) / tn;
    per = sym ? ratio * ti_count * (ti_count - 1) / 2 + tj_count : ti_count * tj_count;
    items = per * E * split;
    // the long side's tiles go last, so that blocks at work share the operands
    cols_fast = p.tall;
  }
  // Item w: batch, tile and part of k.  Parts of a tile are neighbours.
  __device__ void at(int w, int& e, int& ti, int& tj, int& z) const {
    int t = w / split;
    z = w - t * split;
    e = t / per;
    t -= e * per;
    if (sym) {  // row ti has ratio (ti + 1) tiles (the last row tj_count)
      ti = static_cast<int>((sqrtf(8.0f * t / ratio + 1.0f) - 1.0f) * 0.5f);
      while (ratio * ti * (ti + 1) / 2 > t) --ti;
      while (ratio * (ti + 1) * (ti + 2) / 2 <= t) ++ti;
      tj = t - ratio * ti * (ti + 1) / 2;
    } else if (cols_fast) {
      ti = t / tj_count;
      tj = t - ti * tj_count;
    } else {
      tj = t / ti_count;
      ti = t - tj * ti_count;
    }
  }
  // Whether a tile lies wholly below the diagonal: its transpose is written too.
  __device__ bool mirrored(int ti, int tj) const { return sym && tj < ratio * ti; }
  // Chunks of the block's rows from i0 on in the tile's columns from j0 on.
  __device__ int chunks(int i0, int j0) const {
    return i0 < I ? min(tn / kChunk, (J - j0 + kChunk - 1) / kChunk) : 0;
  }
  __device__ int k_begin(int z) const { return static_cast<int>(static_cast<int64_t>(ks) * z / split); }
};

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory"); }

struct __align__(16) Shared {
  uint64_t full[kStages], empty[kStages], done[2], freed[2], aux[kSets], written[kSets], drain;
  alignas(16) float2 cols[kEpiWarps][32];  // a tall matrix's factors of a warp's 32 columns
  uint32_t tmem;
  int abort;
};
constexpr int kSmem = kStages * kStageBytes + kSets * kSet + sizeof(Shared);
static_assert(kSmem <= 227 * 1024, "a block's shared memory");
constexpr int kLead = 64;  // the epilogue's first thread

// The epilogue's view: what it does with 32 accumulator columns of one row of
// a chunk.  `set` is the chunk's 32 KB of shared memory: hi and lo (STEP), A
// (POLY), overwritten by the results that a bulk store then takes.
//
// X's element becomes  ca (hi + lo) + (acc + d_res hi + f d lo) / 2^10
//                    = acc / 2^10 + hi (ca + d_res / 2^10) + lo (ca + f d / 2^10):
// two factors for a row (`coef`), or for a column when the matrix is tall
// (`cols`, this warp's 32 of them in shared memory); lo's is made for the
// stored lo, 2^11 times as large.
template <int MODE>
__device__ __forceinline__ void finish32(const ChainP& p, int step, uint32_t set, int e, int i, int j, int r, int half,
                                         bool mirror, float2 coef, const float4* cols, float (&v)[32]) {
  const uint32_t lo = set + kSet / 2;
  if (MODE == GRAM || MODE == POLY) {
    if (MODE == GRAM) {
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] *= kAScale / (kXScale * kXScale);
    } else {
      const float2 cb = make_float2(p.co[3 * step + 1], p.co[3 * step + 1]);
      const float2 cc = make_float2(p.co[3 * step + 2] / kAScale, p.co[3 * step + 2] / kAScale);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint4 a = ld_shared(unit(set, r, half * 4 + u));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float2* f = reinterpret_cast<float2*>(v + 8 * u + 2 * q);
          const uint32_t w = u4_word(a, q);
          *f = __ffma2_rn(*f, cc, __fmul2_rn(cb, __half22float2(*reinterpret_cast<const __half2*>(&w))));
        }
      }
      if (i >= j && i < j + 32 && i < p.s) {
        float d = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) d = j + k == i ? v[k] : d;
        p.diag[static_cast<int64_t>(e) * p.s + i] = make_float2(d, d - __half2float(__float2half_rn(d)));
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) st_shared(unit(set, r, half * 4 + u), pack_h8(v + 8 * u));
    if (mirror) {
      // the transposed chunk, 64 rows of 128: two boxes of 64 columns
      const uint32_t box = lo + (r >> 6) * (kChunk * 128) + half * 32 * 128 + (r & 7) * 2;
      const int c = (r & 63) >> 3;
#pragma unroll
      for (int k = 0; k < 32; ++k) st_shared_h(unit(box, k, c), __float2half_rn(v[k]));
    }
    return;
  }
  const float2 scale = make_float2(1.0f / kAScale, 1.0f / kAScale);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint32_t ah = unit(set, r, half * 4 + u), al = unit(lo, r, half * 4 + u);
    const uint4 h = ld_shared(ah), l = ld_shared(al);
    uint4 oh, ol;
    uint32_t* const wh = reinterpret_cast<uint32_t*>(&oh);
    uint32_t* const wl = reinterpret_cast<uint32_t*>(&ol);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float2 ch = make_float2(coef.x, coef.x), cl = make_float2(coef.y, coef.y);
      if (p.tall) {
        const float4 t = cols[4 * u + q];
        ch = make_float2(t.x, t.z);
        cl = make_float2(t.y, t.w);
      }
      const uint32_t hw = u4_word(h, q), lw = u4_word(l, q);
      float2* f = reinterpret_cast<float2*>(v + 8 * u + 2 * q);
      float2 y = __ffma2_rn(__half22float2(*reinterpret_cast<const __half2*>(&hw)), ch, __fmul2_rn(*f, scale));
      y = __ffma2_rn(__half22float2(*reinterpret_cast<const __half2*>(&lw)), cl, y);
      if (MODE == STEP) {
        const __half2 hi = __float22half2_rn(y);
        // (y - hi) 2^11, exact before it is rounded
        const __half2 rest = __float22half2_rn(__ffma2_rn(__half22float2(hi), make_float2(-kLoScale, -kLoScale),
                                                          __fmul2_rn(y, make_float2(kLoScale, kLoScale))));
        wh[q] = *reinterpret_cast<const uint32_t*>(&hi);
        wl[q] = *reinterpret_cast<const uint32_t*>(&rest);
      } else {
        *f = y;
      }
    }
    if (MODE == STEP) {
      st_shared(ah, oh);
      st_shared(al, ol);
    }
  }
  if (MODE != STEP) {
    // 32 floats in the place of this thread's hi and lo
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint4 w = make_uint4(__float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]), __float_as_uint(v[4 * u + 2]),
                                 __float_as_uint(v[4 * u + 3]));
      st_shared(unit(u < 4 ? set : lo, r, half * 4 + (u & 3)), w);
    }
  }
}

// The last step's 32 rows and 32 columns of a warp, 32 floats a thread in
// shared memory, to the caller's tensors: row by row, lanes along it.
template <int MODE>
__device__ __forceinline__ void write_out(const ChainP& p, uint32_t set, int e, int i0, int j, int r0, int half) {
  const int lane = threadIdx.x & 31;
  const int col = j + lane, rows = min(32, p.m - i0);
  if (col >= p.n) return;
  const uint32_t from = lane < 16 ? set : set + kSet / 2;
  const int64_t o = static_cast<int64_t>(e) * p.res.out.sb + static_cast<int64_t>(i0) * p.res.out.sr + col;
  const int64_t q = static_cast<int64_t>(e) * p.res.par.sb + static_cast<int64_t>(i0) * p.res.par.sr +
                    static_cast<int64_t>(col) * p.res.par.sc;
#pragma unroll 8
  for (int r = 0; r < rows; ++r) {
    float v = ld_shared_f(unit(from, r0 + r, half * 4 + ((lane & 15) >> 2)) + (lane & 3) * 4) * (1.0f / kXScale);
    if (MODE == UPDATE) v = p.res.keep * load_elem(p.res.par, q + r * p.res.par.sr) - p.res.rate * v;
    store_elem(p.res.out, o + r * p.res.out.sr, v);
  }
}

// Every wait below is bounded (mbar_wait); after one runs out the block's
// roles leave their loops, and so do the other blocks where they wait for phases.

// The loading thread: both operands' k-slices of every work item, in order.
template <int CG>
__device__ __forceinline__ bool load_phase(const ChainP& p, Shared& sh, uint32_t smem, int mode, int cur, int rank,
                                           int64_t& n) {
  const Work<CG> w(p, mode);
  const bool p_mn = mode == GRAM && p.tall, q_mn = mode == GRAM ? p.tall : mode >= STEP && !p.tall;
  const CUtensorMap* mp = mode == GRAM ? (p.tall ? &p.xm[cur] : &p.xk[cur])
                          : mode == POLY ? &p.ak : p.tall ? &p.xk[cur] : &p.bk;
  const CUtensorMap* mq = mode == GRAM ? mp : mode == POLY ? &p.ak : p.tall ? &p.bk : &p.xm[cur];
  const bool half_q = w.ratio == 2;  // a block's 64 rows of Q: the maps by 64 x 64
  if (half_q) mq = mode == GRAM ? &p.xm[cur] : &p.a64;
  const uint32_t bytes = CG * (kOperand + kOperand / w.ratio);
  volatile int* const abort_flag = &sh.abort;
  for (int t = blockIdx.x / CG; t < w.items; t += gridDim.x / CG) {
    int e, ti, tj, z;
    w.at(t, e, ti, tj, z);
    const int i0 = ti * w.TM + rank * kRows, j0 = tj * w.tn + rank * (w.tn / CG);
    for (int k = w.k_begin(z); k < w.k_begin(z + 1); ++k, ++n) {
      const int st = static_cast<int>(n % kStages);
      if (n >= kStages && !mbar_wait(&sh.empty[st], static_cast<uint32_t>(n / kStages - 1) & 1, p.err)) return false;
      if (*abort_flag) return false;
      const uint32_t sp = smem + st * kStageBytes, sq = sp + kOperand;
      if (rank == 0) mbar_arrive_expect_tx(&sh.full[st], bytes);
      if (p_mn) {
        tma_load_3d<CG>(sp, mp, &sh.full[st], i0, k * kTileK, e);
        tma_load_3d<CG>(sp + kOperand / 2, mp, &sh.full[st], i0 + 64, k * kTileK, e);
      } else {
        tma_load_3d<CG>(sp, mp, &sh.full[st], k * kTileK, i0, e);
      }
      if (q_mn) {
        tma_load_3d<CG>(sq, mq, &sh.full[st], j0, k * kTileK, e);
        if (!half_q) tma_load_3d<CG>(sq + kOperand / 2, mq, &sh.full[st], j0 + 64, k * kTileK, e);
      } else {
        tma_load_3d<CG>(sq, mq, &sh.full[st], k * kTileK, j0, e);
      }
    }
  }
  return true;
}

// The issuing thread (of a pair's first block): a work item's products into
// one of two accumulators.
template <int CG>
__device__ __forceinline__ bool issue_phase(const ChainP& p, Shared& sh, uint32_t smem, uint32_t tmem, int mode,
                                            int64_t& n, int64_t& c) {
  const Work<CG> w(p, mode);
  const bool p_mn = mode == GRAM && p.tall, q_mn = mode == GRAM ? p.tall : mode >= STEP && !p.tall;
  const uint32_t idesc = instr_desc_f16(w.TM, w.tn, p_mn, q_mn);
  const uint64_t ka = desc_k16(p_mn), kb = desc_k16(q_mn);
  const uint64_t first_a = smem_desc(smem, p_mn), first_b = smem_desc(smem + kOperand, q_mn);
  volatile int* const abort_flag = &sh.abort;
  for (int t = blockIdx.x / CG; t < w.items; t += gridDim.x / CG, ++c) {
    int e, ti, tj, z;
    w.at(t, e, ti, tj, z);
    const int acc = static_cast<int>(c & 1);
    if (c >= 2 && !mbar_wait(&sh.freed[acc], static_cast<uint32_t>(c / 2 - 1) & 1, p.err)) return false;
    tc_fence_after();
    const uint32_t d = tmem + acc * w.TN;
    const int k0 = w.k_begin(z), k1 = w.k_begin(z + 1);
    for (int k = k0; k < k1; ++k, ++n) {
      const int st = static_cast<int>(n % kStages);
      if (*abort_flag || !mbar_wait(&sh.full[st], static_cast<uint32_t>(n / kStages) & 1, p.err)) return false;
      tc_fence_after();
      const uint64_t da = first_a + st * (kStageBytes >> 4), db = first_b + st * (kStageBytes >> 4);
#pragma unroll
      for (int kk = 0; kk < kTileK / 16; ++kk)
        mma_f16<CG>(d, da + kk * ka, db + kk * kb, idesc, k > k0 || kk > 0);
      mma_commit<CG>(&sh.empty[st]);
    }
    mma_commit<CG>(&sh.done[acc]);
  }
  return true;
}

// A bounded wait that gives the block up when it runs out.  The epilogue's
// warps never leave their loops early (they meet at barriers): once the block
// is given up they run through them without waiting.
__device__ __forceinline__ void wait_or_abort(uint64_t* bar, uint32_t parity, Shared& sh, int* err) {
  volatile int* const abort_flag = &sh.abort;
  if (!*abort_flag && !mbar_wait(bar, parity, err)) *abort_flag = 1;
  __syncwarp();
}

// Add to a counter that other blocks wait on: all that this thread has seen
// written is seen by those that see the sum.
__device__ __forceinline__ void count_up(unsigned* count) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(count) : "memory");
}
// Wait until *count reaches `target` (bounded), or the call is given up.
__device__ __forceinline__ bool wait_count(const ChainP& p, const unsigned* count, unsigned target) {
  const long long t0 = clock64();
  for (int i = 0;; ++i) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(count) : "memory");
    if (v >= target) return true;
    if (i & 15) continue;
    if (*static_cast<volatile unsigned*>(p.counters + 1)) return false;
    if (clock64() - t0 > kWaitCycles) {
      if (p.err) atomicOr(p.err, FRAG_DEVFLAG_WAIT_TIMEOUT);
      atomicExch(p.counters + 1, 1u);
      return false;
    }
  }
}

// Walks the chunks that this block finishes in a phase, in the order of its
// work items.
template <int CG>
struct Cursor {
  const Work<CG>& w;
  const int rank;
  int t, g, step, chunks, e, i0, j0;
  bool mirror;
  __device__ Cursor(const Work<CG>& w_, int rank_) : w(w_), rank(rank_), t(blockIdx.x / CG) { item(); }
  __device__ void item() {
    for (; t < w.items; t += gridDim.x / CG) {
      int ti, tj, z;
      w.at(t, e, ti, tj, z);
      i0 = ti * w.TM + rank * kRows;
      j0 = tj * w.tn;
      chunks = w.chunks(i0, j0);
      mirror = w.mirrored(ti, tj);
      g = w.split > 1 ? z : 0;  // a tile in parts: each of its blocks finishes some chunks
      step = w.split;
      if (g < chunks) return;
    }
  }
  __device__ bool valid() const { return t < w.items; }
  __device__ void next() {
    g += step;
    if (g < chunks) return;
    t += gridDim.x / CG;
    item();
  }
  __device__ int col() const { return j0 + g * kChunk; }
};

// The moving thread: brings each chunk's inputs into a set, all but one of
// them ahead of the epilogue, and stores its results.  `v` counts chunks.
template <int CG>
__device__ __forceinline__ void move_phase(const ChainP& p, Shared& sh, uint32_t sets, int mode, int cur, int rank,
                                           int64_t& v) {
  const Work<CG> w(p, mode);
  volatile int* const abort_flag = &sh.abort;
  int64_t ahead = v;
  Cursor<CG> in(w, rank), out(w, rank);
  auto bring = [&]() {
    if (!in.valid() || *abort_flag) return;
    uint64_t* const bar = &sh.aux[ahead % kSets];
    const uint32_t set = sets + static_cast<uint32_t>(ahead % kSets) * kSet;
    if (mode == GRAM) {
      mbar_arrive(bar);  // nothing to bring: the set is free
    } else {
      mbar_arrive_expect_tx(bar, mode == POLY ? kSet / 2 : kSet);
      tma_load_3d<1>(set, mode == POLY ? &p.ak : &p.xk[cur], bar, in.col(), in.i0, in.e);
      if (mode != POLY) tma_load_3d<1>(set + kSet / 2, &p.lo, bar, in.col(), in.i0, in.e);
    }
    ++ahead;
    in.next();
  };
  for (int i = 0; i < kSets - 1; ++i) bring();
  for (; out.valid(); ++v, out.next()) {
    const uint32_t set = sets + static_cast<uint32_t>(v % kSets) * kSet;
    if (*abort_flag || !mbar_wait(&sh.written[v % kSets], static_cast<uint32_t>(v / kSets) & 1, p.err)) {
      *abort_flag = 1;
      break;
    }
    if (mode == STEP) {
      tma_store_3d(&p.xk[cur ^ 1], set, out.col(), out.i0, out.e);
      tma_store_3d(&p.lo, set + kSet / 2, out.col(), out.i0, out.e);
    } else if (mode < STEP) {
      tma_store_3d(mode == GRAM ? &p.ak : &p.bk, set, out.col(), out.i0, out.e);
      if (out.mirror) {
        const CUtensorMap* to = mode == GRAM ? &p.a64 : &p.b64;
        tma_store_3d(to, set + kSet / 2, out.i0, out.col(), out.e);
        if (out.i0 + 64 < w.I) tma_store_3d(to, set + kSet / 2 + kChunk * 128, out.i0 + 64, out.col(), out.e);
      }
    }
    bulk_commit();
    bulk_wait_read<1>();  // the chunk before this one is out of its set
    bring();
  }
  bulk_wait<0>();  // the phase's results are written
  if (*abort_flag)  // no copy is left on its way into this block
    for (int64_t i = ahead > kSets ? ahead - kSets : 0; i < ahead; ++i)
      mbar_wait(&sh.aux[i % kSets], static_cast<uint32_t>(i / kSets) & 1, nullptr);
}

// The epilogue warps.  `c` counts accumulators, `u` chunks.
template <int CG, int MODE>
__device__ __forceinline__ void finish_phase(const ChainP& p, Shared& sh, uint32_t sets, uint32_t tmem, int step,
                                             int rank, int64_t& c, int64_t& u) {
  const Work<CG> w(p, MODE);
  const int ew = (threadIdx.x >> 5) - 2, lane = threadIdx.x & 31;
  const int quad = (threadIdx.x >> 5) & 3, half = ew >> 2;  // accumulator lanes of this warp; columns of a chunk
  const int r = quad * 32 + lane;
  volatile int* const abort_flag = &sh.abort;
  auto release = [&](int acc) {  // the accumulator is read: the next item's products may overwrite it
    tc_fence_before();
    __syncwarp();
    if (lane == 0) CG == 1 ? mbar_arrive(&sh.freed[acc]) : mbar_arrive_first(&sh.freed[acc]);
  };
  // hi's and lo's factors in row (or column) d of batch e; lo's meets the
  // diagonal in the last two steps only
  auto factors = [&](int e, int d) {
    const float2 v = __ldcg(p.diag + static_cast<int64_t>(e) * p.s + d);
    const float ca = p.co[3 * step];
    return make_float2(ca + v.y * (1.0f / kAScale),
                       (step >= p.steps - 2 ? ca + v.x * (1.0f / kAScale) : ca) * (1.0f / kLoScale));
  };
  for (int t = blockIdx.x / CG; t < w.items; t += gridDim.x / CG, ++c) {
    int e, ti, tj, z;
    w.at(t, e, ti, tj, z);
    const int acc = static_cast<int>(c & 1);
    const int i0 = ti * w.TM + rank * kRows, j0 = tj * w.tn, i = i0 + r;
    const int chunks = w.chunks(i0, j0);
    const bool mirror = w.mirrored(ti, tj);
    const uint32_t ta = tmem + (static_cast<uint32_t>(quad * 32) << 16) + acc * w.TN + half * 32;
    wait_or_abort(&sh.done[acc], static_cast<uint32_t>(c / 2) & 1, sh, p.err);
    tc_fence_after();
    const bool parts = MODE == GRAM && w.split > 1;
    const float* part = nullptr;
    if (parts) {
      // This part's sums go out as columns of 128 rows; when all parts of the
      // tile have arrived, each of its blocks finishes some of the chunks,
      // adding the parts in order.
      const int64_t tile = static_cast<int64_t>(t / w.split) * CG + rank;
      part = p.partials + tile * w.split * (kRows * w.tn);
      float* mine = p.partials + (tile * w.split + z) * (kRows * w.tn);
      for (int g = 0; g < chunks; ++g) {
        float v[32];
        tmem_load32(ta + g * kChunk, v);
#pragma unroll
        for (int k = 0; k < 32; ++k) __stcg(mine + (g * kChunk + half * 32 + k) * kRows + r, v[k]);
      }
      release(acc);
      __threadfence();
      epi_sync();
      if (threadIdx.x == kLead) {
        count_up(p.counters + 2 + tile);
        if (!wait_count(p, p.counters + 2 + tile, static_cast<unsigned>(w.split) * (step + 1))) *abort_flag = 1;
      }
      epi_sync();
    }
    float2 coef = make_float2(0.f, 0.f);
    if (MODE >= STEP && !p.tall && i < p.m) coef = factors(e, i);
    for (int g = parts ? z : 0; g < chunks; g += parts ? w.split : 1, ++u) {
      const int b = static_cast<int>(u % kSets), j = j0 + g * kChunk;
      const uint32_t set = sets + b * kSet;
      float v[32];
      if (parts) {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = 0.f;
        const float* from = part + (g * kChunk + half * 32) * kRows + r;
#pragma unroll
        for (int k0 = 0; k0 < 32; k0 += 16)
          for (int q0 = 0; q0 < w.split; q0 += 4) {
            float f[4][16];  // loads of four parts in flight
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int k = 0; k < 16; ++k)
                f[q][k] = q0 + q < w.split
                              ? __ldcg(from + (static_cast<int64_t>(q0 + q) * w.tn + k0 + k) * kRows) : 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int k = 0; k < 16; ++k) v[k0 + k] += f[q][k];
          }
      } else {
        tmem_load32(ta + g * kChunk, v);
        if (g == chunks - 1) release(acc);
      }
      if (MODE >= STEP && p.tall) {
        const int col = j + half * 32 + lane;
        __syncwarp();
        sh.cols[ew][lane] = col < p.n ? factors(e, col) : coef;
        __syncwarp();
      }
      wait_or_abort(&sh.aux[b], static_cast<uint32_t>(u / kSets) & 1, sh, p.err);
      finish32<MODE>(p, step, set, e, i, j + half * 32, r, half, mirror, coef,
                     reinterpret_cast<const float4*>(sh.cols[ew]), v);
      if (MODE <= STEP) {
        proxy_fence_shared();
      } else {
        __syncwarp();
        write_out<MODE>(p, set, e, i0 + quad * 32, j + half * 32, quad * 32, half);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.written[b]);
    }
    if (chunks == 0 && !parts) release(acc);
  }
}

// All steps in one launch: every block walks each phase's work items (A, then
// B, then X), and a count of finished blocks parts the phases.  One block per
// SM; CG = 2: pairs of blocks share 256 x 256 tiles, each holding half of the
// operands.
//
// Bound: large matrices by the operands' way from L2: a pair's tile takes 64 KB
// for each 64 of k, and every phase of 4096 x 14336 moves 9.5 to 10.5 TB/s (A
// 191 us for 2.0 GB, B 58 for 0.57, X 395 for 3.8): 1.3 to 1.5 PFLOP/s while it
// runs, 0.92 over the useful operations of a whole update (the last round of
// tiles is part empty; the power limit).  Small ones by latency: a phase of one
// item a block takes 7 to 9 us, of which 2 are counting, 1.3 the first load,
// 0.3 each k-slice, 2.5 the epilogue and its stores.
template <int CG>
__global__ void __launch_bounds__(kThreads, 1) chain(const __grid_constant__ ChainP p) {
  // stages, sets, and the rest behind them: no static shared memory, so that
  // the stages start on the swizzle's 1024 bytes
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw + kStages * kStageBytes + kSets * kSet);
  const uint32_t smem = smem_u32(smem_raw);
  const uint32_t sets = smem + kStages * kStageBytes;
  const int warp = threadIdx.x >> 5;
  const int rank = CG == 1 ? 0 : static_cast<int>(cluster_rank());
  constexpr int kColumns = 2 * 128 * CG;
  if (threadIdx.x == 0) {
    sh.abort = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.done[i], 1);
      mbar_init(&sh.freed[i], CG * kEpiWarps);
    }
    for (int i = 0; i < kSets; ++i) {
      mbar_init(&sh.aux[i], 1);
      mbar_init(&sh.written[i], kEpiWarps);
    }
    mbar_init(&sh.drain, 1);
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc<CG>(&sh.tmem, kColumns);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* const abort_flag = &sh.abort;
  const bool loads = warp == 0 && elect_one(), issues = warp == 1 && rank == 0 && elect_one();
  const bool moves = warp == 2 + kEpiWarps && elect_one();
  int64_t n = 0, c = 0, u = 0;  // k-slices, accumulators, chunks so far
  // Phase f may start when every block's mover has counted phase f - 1.  The
  // loading thread waits for that; the others follow it from barrier to
  // barrier, and no part of the block waits for another to end a phase.
  auto phases = [&](auto body) {
    for (int f = 0; f < 3 * p.steps; ++f) {
      const int step = f / 3, ph = f - 3 * step;
      const int mode = ph < STEP ? ph : step + 1 < p.steps ? static_cast<int>(STEP) : p.res.last;
      if (!body(f, step, mode)) {
        *abort_flag = 1;
        atomicExch(p.counters + 1, 1u);
        return;
      }
    }
  };
  auto started = [&](int f) {
    if (f > 0 && !wait_count(p, p.counters, static_cast<unsigned>(f) * gridDim.x)) return false;
    proxy_fence();
    return true;
  };
  if (warp == 0) {
    if (loads)
      phases([&](int f, int step, int mode) {
        return started(f) && load_phase<CG>(p, sh, smem, mode, step & 1, rank, n);
      });
  } else if (warp == 1) {
    if (issues) phases([&](int, int, int mode) { return issue_phase<CG>(p, sh, smem, tmem, mode, n, c); });
  } else if (warp == 2 + kEpiWarps) {
    if (moves)
      phases([&](int f, int step, int mode) {
        // A has to be there; X and lo have been since the phase before A's
        if (mode == POLY && !started(f)) return false;
        const int64_t before = u;
        move_phase<CG>(p, sh, sets, mode, step & 1, rank, u);
        // a block with nothing to do in a phase may not count ahead of the others
        if (u == before && !started(f)) return false;
        count_up(p.counters);
        return !*abort_flag;
      });
  } else {
    for (int step = 0; step < p.steps; ++step) {
      finish_phase<CG, GRAM>(p, sh, sets, tmem, step, rank, c, u);
      finish_phase<CG, POLY>(p, sh, sets, tmem, step, rank, c, u);
      if (step + 1 < p.steps) finish_phase<CG, STEP>(p, sh, sets, tmem, step, rank, c, u);
      else if (p.res.last == LAST) finish_phase<CG, LAST>(p, sh, sets, tmem, step, rank, c, u);
      else finish_phase<CG, UPDATE>(p, sh, sets, tmem, step, rank, c, u);
    }
  }
  __syncthreads();
  // nothing is in flight when shared memory and accumulators are given up
  if (loads)
    for (int64_t i = n > kStages ? n - kStages : 0; i < n && rank == 0; ++i)
      mbar_wait(&sh.full[i % kStages], static_cast<uint32_t>(i / kStages) & 1, nullptr);
  if (issues) mma_commit<CG>(&sh.drain);
  if (warp == 1 && (rank == 0 ? issues : elect_one())) mbar_wait(&sh.drain, 0, p.err);
  __syncthreads();
  if (CG == 2) cluster_sync();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free<CG>(tmem, kColumns);
  }
}

// ------------------------------------------------------------- preparation

// Sums of squares, a block's in a fixed order.
template <int V>
__global__ void __launch_bounds__(256) prep_norm(const PrepP p) {
  __shared__ float slots[2][32];
  const int64_t e = blockIdx.y;
  const uint32_t per = static_cast<uint32_t>(p.cols / V);
  const uint32_t total = static_cast<uint32_t>(p.rows * per), stride = gridDim.x * blockDim.x;
  if (blockIdx.x == 0 && e == 0)
    for (int i = threadIdx.x; i < p.count; i += blockDim.x) p.counters[i] = 0;
  float ss = 0.f;
#pragma unroll 4
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
    const uint32_t r = i / per;
    float u[V], m[V];
    prep_value<V>(p, e, r, (i - r * per) * V, u, m);
#pragma unroll
    for (int k = 0; k < V; ++k) ss = fmaf(u[k], u[k], ss);
  }
  ss = block_sum(ss, slots, 0);
  if (threadIdx.x == 0) p.partials[e * gridDim.x + blockIdx.x] = ss;
}

// X = u / (|u| + eps) as hi + lo, and the new momentum.
template <int V>
__global__ void __launch_bounds__(256) prep_scale(const PrepP p, int blocks) {
  __shared__ float slots[2][32];
  const int64_t e = blockIdx.y;
  const uint32_t per = static_cast<uint32_t>(p.cols / V);
  const uint32_t total = static_cast<uint32_t>(p.rows * per), stride = gridDim.x * blockDim.x;
  float ss = 0.f;
  for (int i = threadIdx.x; i < blocks; i += blockDim.x) ss += p.partials[e * blocks + i];
  const float f = kXScale / (sqrtf(block_sum(ss, slots, 0)) + p.eps);
#pragma unroll 4
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
    const uint32_t r = i / per, c = (i - r * per) * V;
    float u[V], m[V];
    prep_value<V>(p, e, r, c, u, m);
    if (p.has_mom) store_elems<V>(p.mom_out, (e * p.rows + r) * p.cols + c, m);
    const int64_t o = (e * p.rows + r) * p.ldx + c;
    if (V == 8) {
      float l[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = u[k % V] * f;
        u[k % V] = x;
        l[k] = (x - __half2float(__float2half_rn(x))) * kLoScale;
      }
      *reinterpret_cast<uint4*>(p.hi + o) = pack_h8(u);
      *reinterpret_cast<uint4*>(p.lo + o) = pack_h8(l);
    } else {
      const float x = u[0] * f;
      const __half h = __float2half_rn(x);
      p.hi[o] = h;
      p.lo[o] = __float2half_rn((x - __half2float(h)) * kLoScale);
    }
  }
}

// -------------------------------------------------------------------- host

struct Plan {
  int64_t s, l, ldx, lds, tiles;
  size_t hi0, hi1, lo, a, b, diag, partials, sums, counters, bytes;
  int blocks, pairs, groups, narrow, split, count;
};

// Blocks (or pairs of them) that are resident at once, one per SM.
int resident(bool pairs) {
  static std::mutex mu;
  static int cache[64][2] = {};
  const int d = current_device();
  if (d < 0 || d >= 64) return 0;
  std::lock_guard<std::mutex> lk(mu);
  int& n = cache[d][pairs];
  if (n) return n;
  if (!pairs) return n = sm_count();
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(chain<2>), kSmem)) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * sm_count());
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, chain<2>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return n = std::min(clusters, sm_count() / 2);
}

int64_t chain_tiles(int64_t E, int64_t rows, int64_t cols, int64_t side, bool sym) {
  const int64_t ti = ceil_div(rows, side), tj = ceil_div(cols, side);
  return E * (sym ? ti * (ti + 1) / 2 : ti * tj);
}

Plan make_plan(int64_t E, int64_t m, int64_t n) {
  Plan q;
  q.s = std::min(m, n);
  q.l = std::max(m, n);
  q.ldx = ceil_div(n, 8) * 8;
  q.lds = ceil_div(q.s, 8) * 8;
  // Pairs of blocks and 256 x 256 tiles where X has enough of them to keep three
  // quarters of the pairs busy, single blocks and 128 x 128 tiles below.  A
  // step, single against pairs: 1536 x 1536 (36 tiles) 46 and 53 us, 2048 x
  // 2048 (64) 70 and 63, 4096 x 4096 405 and 270.
  q.pairs = resident(true) > 0 && 4 * chain_tiles(E, m, n, 256, false) >= 3 * resident(true);
  q.groups = resident(q.pairs);
  const int64_t side = q.pairs ? 256 : 128;
  q.tiles = chain_tiles(E, q.s, q.s, side, true);
  // A's and B's tiles at half the width where pairs outnumber them two to one.
  // Five steps, full against half: 1024 x 4096 246 and 240 us, 2048 x 2048 331
  // and 310, 1536 x 2560 290 and 282; but 1100 x 5000, whose A is then split into
  // fewer parts, 326 and 340.
  q.narrow = q.pairs && 2 * q.tiles <= q.groups;
  if (q.narrow) q.tiles = E * (ceil_div(q.s, 256) * (ceil_div(q.s, 256) - 1) + ceil_div(q.s, 128));
  // A's few tiles with a long k: each in up to four parts of at least six
  // k-slices (a part costs about 5 us, a slice 0.3), one work item a group.  A
  // step of 1024 x 4096 in 1, 2, 4 and 8 parts: 63, 55, 49 and 49 us.
  const int64_t ks = ceil_div(q.l, kTileK);
  q.split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({q.groups / std::max<int64_t>(1, q.tiles), ks / 6, 4})));
  const size_t x = align_up(static_cast<size_t>(E) * m * q.ldx * 2, 256);
  const size_t a = align_up(static_cast<size_t>(E) * q.s * q.lds * 2, 256);
  q.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(1184, ceil_div(m * n, 2048))));
  q.count = 2 + (q.split > 1 ? static_cast<int>(q.tiles) * (q.pairs ? 2 : 1) : 0);
  q.hi0 = 0;
  q.hi1 = x;
  q.lo = 2 * x;
  q.a = 3 * x;
  q.b = q.a + a;
  q.diag = q.b + a;
  q.partials = q.diag + align_up(static_cast<size_t>(E) * q.s * sizeof(float2), 256);
  q.counters = q.partials + align_up(static_cast<size_t>(E) * q.blocks * sizeof(float), 256);
  q.sums = q.counters + align_up(static_cast<size_t>(q.count) * sizeof(unsigned), 256);
  q.bytes = q.sums + (q.split > 1 ? static_cast<size_t>(q.tiles) * q.split * side * (q.narrow ? 128 : side) * sizeof(float) : 0);
  return q;
}

template <int CG>
int launch_chain(const ChainP& p, int groups, cudaStream_t s) {
  auto kern = chain<CG>;
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kern), kSmem)) return FRAG_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups * CG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;  // blocks wait for one another: every one is resident
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 1 ? 1 : 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p));
}

int orthogonalise(const PrepP& prep, int64_t E, int64_t m, int64_t n, int steps, const float* co, Elem out,
                  const Elem* par, float keep, float rate, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  const ResultP res = {par ? UPDATE : LAST, out, par ? *par : Elem{}, keep, rate};
  if (small_takes(m, n)) return orthogonalise_small(prep, E, steps, co, res, s);
  const Plan q = make_plan(E, m, n);
  if (!workspace || workspace_bytes < q.bytes) return FRAG_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FRAG_ERR_ALIGN;
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  if (q.groups <= 0) return FRAG_ERR_NO_DEVICE;
  PrepP pp = prep;
  pp.ldx = q.ldx;
  pp.hi = reinterpret_cast<__half*>(ws + q.hi0);
  pp.lo = reinterpret_cast<__half*>(ws + q.lo);
  pp.partials = reinterpret_cast<float*>(ws + q.partials);
  pp.counters = reinterpret_cast<unsigned*>(ws + q.counters);
  pp.count = q.count;
  ChainP p = {};
  __half* hi[2] = {pp.hi, reinterpret_cast<__half*>(ws + q.hi1)};
  __half* A = reinterpret_cast<__half*>(ws + q.a);
  __half* B = reinterpret_cast<__half*>(ws + q.b);
  bool maps = make_map_3d(&p.lo, pp.lo, n, m, E, q.ldx, m * q.ldx, kChunk, kRows);
  for (int i = 0; i < 2; ++i)
    maps = maps && make_map_3d(&p.xk[i], hi[i], n, m, E, q.ldx, m * q.ldx, kTileK, kRows) &&
           make_map_3d(&p.xm[i], hi[i], n, m, E, q.ldx, m * q.ldx, 64, kTileK);
  maps = maps && make_map_3d(&p.ak, A, q.s, q.s, E, q.lds, q.s * q.lds, kTileK, kRows) &&
         make_map_3d(&p.bk, B, q.s, q.s, E, q.lds, q.s * q.lds, kTileK, kRows) &&
         make_map_3d(&p.a64, A, q.s, q.s, E, q.lds, q.s * q.lds, 64, 64) &&
         make_map_3d(&p.b64, B, q.s, q.s, E, q.lds, q.s * q.lds, 64, 64);
  if (!maps) return FRAG_ERR_CUDA;
  p.m = static_cast<int>(m);
  p.n = static_cast<int>(n);
  p.s = static_cast<int>(q.s);
  p.l = static_cast<int>(q.l);
  p.E = static_cast<int>(E);
  p.tall = m > n;
  p.steps = steps;
  p.split = q.split;
  p.narrow = q.narrow;
  p.diag = reinterpret_cast<float2*>(ws + q.diag);
  p.partials = reinterpret_cast<float*>(ws + q.sums);
  p.counters = pp.counters;
  p.res = res;
  p.err = device_error_word();
  for (int i = 0; i < 3 * steps; ++i) p.co[i] = co[i];

  const dim3 grid(static_cast<unsigned>(q.blocks), static_cast<unsigned>(E));
  if (chunked(pp.g, E, m, n) && (!pp.has_mom || (chunked(pp.mom, E, m, n) && chunked(pp.mom_out, E, m, n)))) {
    prep_norm<8><<<grid, 256, 0, s>>>(pp);
    prep_scale<8><<<grid, 256, 0, s>>>(pp, q.blocks);
  } else {
    prep_norm<1><<<grid, 256, 0, s>>>(pp);
    prep_scale<1><<<grid, 256, 0, s>>>(pp, q.blocks);
  }
  const int st = check_launch();
  if (st != FRAG_OK) return st;
  // no more groups than the busiest phase has items
  const int64_t side = q.pairs ? 256 : 128;
  const int64_t most = std::max<int64_t>(q.tiles * q.split, chain_tiles(E, m, n, side, false));
  const int groups = static_cast<int>(std::min<int64_t>(q.groups, most));
  return q.pairs ? launch_chain<2>(p, groups, s) : launch_chain<1>(p, groups, s);
}

int check_sizes(int64_t E, int64_t m, int64_t n, int steps, const float* co) {
  if (E < 0 || m < 0 || n < 0 || steps < 1 || !co) return FRAG_ERR_INVALID_ARG;
  if (m > (1 << 24) || n > (1 << 24) || E > 65535 || steps > kMaxSteps) return FRAG_ERR_SHAPE;
  if (m > 0 && n > 0 && (chain_tiles(E, m, n, 128, false) > (1 << 24) || m * n > 0x7fffffffLL)) return FRAG_ERR_SHAPE;
  return FRAG_OK;
}

bool elem_of(const frag_matrix* t, Elem& e) {
  if (!t || !t->data || (t->dtype != FRAG_DT_BF16 && t->dtype != FRAG_DT_F32)) return false;
  e = Elem{t->data, t->dtype == FRAG_DT_F32, t->stride_batch, t->stride_row, t->stride_col};
  return true;
}

}  // namespace
}  // namespace frag

using namespace frag;

extern "C" {

size_t frag_orthogonalize_workspace_bytes(int64_t E, int64_t m, int64_t n) {
  if (E <= 0 || m <= 0 || n <= 0) return 0;
  return small_takes(m, n) ? 0 : make_plan(E, m, n).bytes;
}

int frag_orthogonalize(const frag_matrix* g, void* out, int64_t E, int64_t m, int64_t n, int steps,
                       const float* coefficients, float eps, void* workspace, size_t workspace_bytes,
                       frag_stream_t stream) {
  const int bad = check_sizes(E, m, n, steps, coefficients);
  if (bad != FRAG_OK) return bad;
  if (E == 0 || m == 0 || n == 0) return FRAG_OK;
  PrepP prep = {};
  if (!elem_of(g, prep.g) || !out) return FRAG_ERR_INVALID_ARG;
  prep.rows = m;
  prep.cols = n;
  prep.eps = eps;
  const Elem o{out, 0, m * n, n, 1};
  return orthogonalise(prep, E, m, n, steps, coefficients, o, nullptr, 0.f, 0.f,
                       workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

int frag_muon_update(const frag_matrix* param, const frag_matrix* grad, const frag_matrix* momentum, void* param_out,
                     void* momentum_out, int64_t E, int64_t m, int64_t n, float lr, float mu, int nesterov,
                     float weight_decay, float scale, int steps, const float* coefficients, float eps,
                     void* workspace, size_t workspace_bytes, frag_stream_t stream) {
  const int bad = check_sizes(E, m, n, steps, coefficients);
  if (bad != FRAG_OK) return bad;
  if (E == 0 || m == 0 || n == 0) return FRAG_OK;
  PrepP prep = {};
  Elem par;
  if (!elem_of(param, par) || !elem_of(grad, prep.g) || !elem_of(momentum, prep.mom)) return FRAG_ERR_INVALID_ARG;
  if (!param_out || !momentum_out) return FRAG_ERR_INVALID_ARG;
  prep.mom_out = Elem{momentum_out, prep.mom.f32, m * n, n, 1};
  prep.has_mom = 1;
  prep.nesterov = nesterov;
  prep.mu = mu;
  prep.rows = m;
  prep.cols = n;
  prep.eps = eps;
  const Elem o{param_out, par.f32, m * n, n, 1};
  return orthogonalise(prep, E, m, n, steps, coefficients, o, &par, 1.0f - lr * weight_decay, lr * scale,
                       workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"

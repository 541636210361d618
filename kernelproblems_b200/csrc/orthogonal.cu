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
//  - X = hi + lo, two fp16 numbers (22 bits).  a X uses both, B X uses hi: an
//    error of B X lies along directions that are already large, which later
//    steps do not amplify, while an error of a X is multiplied by a^5 = 485
//    along small ones.  On a gradient of 16 strong directions and a rest of 2%
//    (512 x 2048), relative error of the result against 64 bits: bf16
//    throughout 0.27, one fp16 0.035, hi + lo 0.0003.
//  - everything is kept times a power of two (X 2^8, A and B 2^10), so that
//    the first step's small entries (1/sqrt(mn) of a unit norm) stay clear of
//    fp16's subnormals, and the largest (|B| <= 24 for steep schedules) of 65504.
//  - B's diagonal (near -2.7 at the end, against small off-diagonal entries)
//    carries most of B's rounding error: its residual is kept in 32 bits and
//    added in the epilogue, as is the diagonal's product with lo in the last
//    two steps (earlier, lo along small directions would be amplified).
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <mutex>

#include "tc.cuh"

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

constexpr float kXScale = 256.0f;   // X is kept times 2^8
constexpr float kAScale = 1024.0f;  // A and B times 2^10
constexpr int kRows = 128;          // rows of C a block holds
constexpr int kChunk = 64;          // columns the epilogue takes at a time
constexpr int kOperand = 128 * kTileK * 2;  // bytes of one operand of a stage
constexpr int kStageBytes = 2 * kOperand;
constexpr int kStages = 4;
constexpr int kSet = 2 * kRows * kChunk * 2;  // two 16-bit chunks
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;  // a loading warp, an issuing warp, the epilogue
constexpr int kSmem = kStages * kStageBytes + 2 * kSet + 1024;

// GRAM A = X X', POLY B = b A + c A A, STEP X <- a X + B X; the last step's
// STEP writes the result (LAST) or the weights (UPDATE) instead of X.
enum Mode { GRAM = 0, POLY = 1, STEP = 2, LAST = 3, UPDATE = 4 };

struct Elem {  // a tensor of bf16 or fp32 elements with strides
  void* p;
  int f32;
  int64_t sb, sr, sc;
};
__device__ __forceinline__ float load_elem(const Elem& e, int64_t i) {
  return e.f32 ? static_cast<const float*>(e.p)[i] : bf16_to_f(static_cast<const uint16_t*>(e.p)[i]);
}
__device__ __forceinline__ void store_elem(const Elem& e, int64_t i, float v) {
  if (e.f32) static_cast<float*>(e.p)[i] = v;
  else static_cast<uint16_t*>(e.p)[i] = f_to_bf16(v);
}

constexpr int kMaxSteps = 32;

struct ChainP {
  // X's two buffers by 64 columns x 128 rows and by 64 x 64, lo, A and B
  CUtensorMap xk[2], xm[2], lo, ak, bk, a64, b64;
  int m, n, s, l, E, tall, steps, split;
  float2* diag;        // [E, s] B's diagonal in 32 bits and its rounding residual
  float* partials;     // split GRAM sums
  unsigned* counters;  // grid barrier, abort, and an arrival count for each split tile
  int last;            // LAST or UPDATE
  Elem out, par;
  float keep, rate;  // p' = keep p - rate O
  int* err;
  float co[3 * kMaxSteps];
};

__device__ __forceinline__ void unpack_h8(const uint4& v, float* f) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack_h8(const float* f) {
  uint4 v;
  __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  return v;
}
__device__ __forceinline__ uint4 ld_shared(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void st_shared(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float ld_shared_f(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void st_shared_h(uint32_t a, __half v) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(a), "h"(__half_as_ushort(v)) : "memory");
}
// 16-byte unit u of row r of a chunk (128-byte rows under the 128-byte swizzle).
__device__ __forceinline__ uint32_t unit(uint32_t base, int r, int u) { return base + r * 128 + ((u ^ (r & 7)) << 4); }

// One phase's product C[i, j] = sum_k P[i, k] Q[j, k] as a list of work items.
template <int CG>
struct Work {
  static constexpr int TM = kRows * CG, TN = 128 * CG;
  int I, J, ks, split, ti_count, tj_count, per, items, E;
  bool sym, cols_fast;
  __device__ Work(const ChainP& p, int mode) {
    sym = mode == GRAM || mode == POLY;
    I = sym ? p.s : p.m;
    J = sym ? p.s : p.n;
    E = p.E;
    ks = ((mode == GRAM ? p.l : p.s) + kTileK - 1) / kTileK;
    split = mode == GRAM ? p.split : 1;
    ti_count = (I + TM - 1) / TM;
    tj_count = (J + TN - 1) / TN;
    per = sym ? ti_count * (ti_count + 1) / 2 : ti_count * tj_count;
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
    if (sym) {
      ti = static_cast<int>((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
      while (ti * (ti + 1) / 2 > t) --ti;
      while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
      tj = t - ti * (ti + 1) / 2;
    } else if (cols_fast) {
      ti = t / tj_count;
      tj = t - ti * tj_count;
    } else {
      tj = t / ti_count;
      ti = t - tj * ti_count;
    }
  }
  __device__ int k_begin(int z) const { return static_cast<int>(static_cast<int64_t>(ks) * z / split); }
};

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory"); }

struct Shared {
  uint64_t full[kStages], empty[kStages], done[2], freed[2], aux[2], drain;
  int64_t aux_issued[2];  // the last chunk prepared in each set, plus one
  uint32_t tmem;
  int abort;
};
constexpr int kLead = 64;  // the epilogue's thread that moves chunks

// The epilogue's view: what it does with 32 accumulator columns of one row of
// a chunk.  `set` is the chunk's 32 KB of shared memory: hi and lo (STEP), A
// (POLY), overwritten by the results that a bulk store then takes.
template <int MODE>
__device__ __forceinline__ void finish32(const ChainP& p, int step, uint32_t set, int e, int i, int j, int r, int half,
                                         bool mirror, float2 dr, float (&v)[32]) {
  const uint32_t lo = set + kSet / 2;
  if (MODE == GRAM || MODE == POLY) {
    if (MODE == GRAM) {
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] *= kAScale / (kXScale * kXScale);
    } else {
      const float cb = p.co[3 * step + 1], cc = p.co[3 * step + 2] / kAScale;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float a[8];
        unpack_h8(ld_shared(unit(set, r, half * 4 + u)), a);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[8 * u + k] = cb * a[k] + cc * v[8 * u + k];
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
      const uint32_t box = lo + (r >> 6) * (kChunk * 128);
      const int c = r & 63;
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const int jr = half * 32 + k;
        st_shared_h(unit(box, jr, c >> 3) + (c & 7) * 2, __float2half_rn(v[k]));
      }
    }
    return;
  }
  const float ca = p.co[3 * step];
  const float lf = step >= p.steps - 2 ? 1.0f / kAScale : 0.0f;  // the diagonal's product with lo
  float2 dc = dr;
  if (p.tall) {  // column j + lane's, handed round below
    const int col = j + (threadIdx.x & 31);
    dc = col < p.n ? __ldcg(p.diag + static_cast<int64_t>(e) * p.s + col) : make_float2(0.f, 0.f);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    float h[8], l[8];
    unpack_h8(ld_shared(unit(set, r, half * 4 + u)), h);
    unpack_h8(ld_shared(unit(lo, r, half * 4 + u)), l);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float2 d = dr;
      if (p.tall) {
        d.x = __shfl_sync(0xffffffffu, dc.x, 8 * u + k);
        d.y = __shfl_sync(0xffffffffu, dc.y, 8 * u + k);
      }
      v[8 * u + k] = ca * (h[k] + l[k]) + (v[8 * u + k] + d.y * h[k]) * (1.0f / kAScale) + lf * (d.x * l[k]);
    }
  }
  if (MODE == STEP) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      st_shared(unit(set, r, half * 4 + u), pack_h8(v + 8 * u));
#pragma unroll
      for (int k = 0; k < 8; ++k) v[8 * u + k] -= __half2float(__float2half_rn(v[8 * u + k]));
      st_shared(unit(lo, r, half * 4 + u), pack_h8(v + 8 * u));
    }
  } else {
    // 32 floats in the place of this thread's hi and lo
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint4 w = make_uint4(__float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]), __float_as_uint(v[4 * u + 2]),
                                 __float_as_uint(v[4 * u + 3]));
      st_shared(unit(u < 4 ? set : lo, r, half * 4 + (u & 3)), w);
    }
  }
}

// The last step's chunk, 32 floats a thread in shared memory, to the caller's
// tensors: a warp a row, lanes along it.
template <int MODE>
__device__ __forceinline__ void write_out(const ChainP& p, uint32_t set, int e, int i0, int j0, int warp) {
  const int lane = threadIdx.x & 31;
#pragma unroll 4
  for (int r = warp; r < kRows; r += kEpiWarps) {
    const int i = i0 + r;
    if (i >= p.m) break;
    const int64_t o = static_cast<int64_t>(e) * p.out.sb + static_cast<int64_t>(i) * p.out.sr;
    const int64_t q = static_cast<int64_t>(e) * p.par.sb + static_cast<int64_t>(i) * p.par.sr;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = j0 + 32 * h + lane;
      if (j >= p.n) continue;
      float v = ld_shared_f(unit(lane < 16 ? set : set + kSet / 2, r, h * 4 + ((lane & 15) >> 2)) + (lane & 3) * 4);
      v *= 1.0f / kXScale;
      if (MODE == UPDATE) v = p.keep * load_elem(p.par, q + static_cast<int64_t>(j) * p.par.sc) - p.rate * v;
      store_elem(p.out, o + j, v);
    }
  }
}

// Every wait below is bounded (mbar_wait); after one runs out the block's
// roles leave their loops, and so do the other blocks at the grid barrier.

// The loading thread: both operands' k-slices of every work item, in order.
template <int CG>
__device__ __forceinline__ bool load_phase(const ChainP& p, Shared& sh, uint32_t smem, int mode, int cur, int rank,
                                           int64_t& n) {
  const Work<CG> w(p, mode);
  const bool p_mn = mode == GRAM && p.tall, q_mn = mode == GRAM ? p.tall : mode >= STEP && !p.tall;
  const CUtensorMap* mp = mode == GRAM ? (p.tall ? &p.xm[cur] : &p.xk[cur])
                          : mode == POLY ? &p.ak : p.tall ? &p.xk[cur] : &p.bk;
  const CUtensorMap* mq = mode == GRAM ? mp : mode == POLY ? &p.ak : p.tall ? &p.bk : &p.xm[cur];
  volatile int* const abort_flag = &sh.abort;
  for (int t = blockIdx.x / CG; t < w.items; t += gridDim.x / CG) {
    int e, ti, tj, z;
    w.at(t, e, ti, tj, z);
    const int i0 = ti * w.TM + rank * kRows, j0 = tj * w.TN + rank * 128;
    for (int k = w.k_begin(z); k < w.k_begin(z + 1); ++k, ++n) {
      const int st = static_cast<int>(n % kStages);
      if (n >= kStages && !mbar_wait(&sh.empty[st], static_cast<uint32_t>(n / kStages - 1) & 1, p.err)) return false;
      if (*abort_flag) return false;
      const uint32_t sp = smem + st * kStageBytes, sq = sp + kOperand;
      if (rank == 0) mbar_arrive_expect_tx(&sh.full[st], CG * kStageBytes);
      if (p_mn) {
        tma_load_3d<CG>(sp, mp, &sh.full[st], i0, k * kTileK, e);
        tma_load_3d<CG>(sp + kOperand / 2, mp, &sh.full[st], i0 + 64, k * kTileK, e);
      } else {
        tma_load_3d<CG>(sp, mp, &sh.full[st], k * kTileK, i0, e);
      }
      if (q_mn) {
        tma_load_3d<CG>(sq, mq, &sh.full[st], j0, k * kTileK, e);
        tma_load_3d<CG>(sq + kOperand / 2, mq, &sh.full[st], j0 + 64, k * kTileK, e);
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
  const uint32_t idesc = instr_desc_f16(w.TM, w.TN, p_mn, q_mn);
  const uint64_t ka = desc_k16(p_mn), kb = desc_k16(q_mn);
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
      const uint32_t sp = smem + st * kStageBytes;
      const uint64_t da = smem_desc(sp, p_mn), db = smem_desc(sp + kOperand, q_mn);
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

// Wait until *count reaches `target` (bounded), or the call is given up.
__device__ __forceinline__ bool wait_count(const ChainP& p, volatile unsigned* count, unsigned target) {
  volatile unsigned* const given_up = p.counters + 1;
  const long long t0 = clock64();
  while (*count < target) {
    if (*given_up) return false;
    if (clock64() - t0 > kWaitCycles) {
      if (p.err) atomicOr(p.err, FRAG_DEVFLAG_WAIT_TIMEOUT);
      atomicExch(p.counters + 1, 1u);
      return false;
    }
  }
  __threadfence();
  return true;
}

// The epilogue warps.  `c` counts accumulators, `u` chunks (of shared memory).
template <int CG, int MODE>
__device__ __forceinline__ void finish_phase(const ChainP& p, Shared& sh, uint32_t sets, uint32_t tmem, int step,
                                             int cur, int rank, int64_t& c, int64_t& u) {
  const Work<CG> w(p, MODE);
  const int ew = (threadIdx.x >> 5) - 2, lane = threadIdx.x & 31;
  const int quad = (threadIdx.x >> 5) & 3, half = ew >> 2;  // accumulator lanes of this warp; columns of a chunk
  const int r = quad * 32 + lane;
  const bool lead = threadIdx.x == kLead;
  volatile int* const abort_flag = &sh.abort;
  // chunk v, columns j.. of rows i0.. of batch e: its set is free (the store
  // of two chunks ago has read it) and its inputs are on their way
  auto prepare = [&](int64_t v, int e, int i0, int j) {
    const int b = static_cast<int>(v & 1);
    const uint32_t set = sets + b * kSet;
    if (*abort_flag) return;
    if (MODE == GRAM) {
      bulk_wait_read<1>();
      mbar_arrive(&sh.aux[b]);
    } else {
      bulk_wait_read<0>();
      mbar_arrive_expect_tx(&sh.aux[b], MODE == POLY ? kSet / 2 : kSet);
      if (MODE == POLY) {
        tma_load_3d<1>(set, &p.ak, &sh.aux[b], j, i0, e);
      } else {
        tma_load_3d<1>(set, &p.xk[cur], &sh.aux[b], j, i0, e);
        tma_load_3d<1>(set + kSet / 2, &p.lo, &sh.aux[b], j, i0, e);
      }
    }
    sh.aux_issued[b] = v + 1;
  };
  auto release = [&](int acc) {  // the accumulator is read: the next item's products may overwrite it
    tc_fence_before();
    __syncwarp();
    if (lane == 0) CG == 1 ? mbar_arrive(&sh.freed[acc]) : mbar_arrive_first(&sh.freed[acc]);
  };
  for (int t = blockIdx.x / CG; t < w.items; t += gridDim.x / CG, ++c) {
    int e, ti, tj, z;
    w.at(t, e, ti, tj, z);
    const int acc = static_cast<int>(c & 1);
    const int i0 = ti * w.TM + rank * kRows, j0 = tj * w.TN, i = i0 + r;
    const int chunks = i0 < w.I ? min(w.TN / kChunk, (w.J - j0 + kChunk - 1) / kChunk) : 0;
    const bool mirror = w.sym && ti != tj;
    const uint32_t ta = tmem + (static_cast<uint32_t>(quad * 32) << 16) + acc * w.TN + half * 32;
    if (MODE != GRAM && lead && chunks > 0) prepare(u, e, i0, j0);
    wait_or_abort(&sh.done[acc], static_cast<uint32_t>(c / 2) & 1, sh, p.err);
    tc_fence_after();
    const bool parts = MODE == GRAM && w.split > 1;
    const float* part = nullptr;
    if (parts) {
      // This part's sums go out as columns of 128 rows; when all parts of the
      // tile have arrived, each of its blocks finishes some of the chunks,
      // adding the parts in order.
      const int64_t tile = static_cast<int64_t>(t / w.split) * CG + rank;
      part = p.partials + tile * w.split * (kRows * w.TN);
      float* mine = p.partials + (tile * w.split + z) * (kRows * w.TN);
      for (int g = 0; g < chunks; ++g) {
        float v[32];
        tmem_load32(ta + g * kChunk, v);
#pragma unroll
        for (int k = 0; k < 32; ++k) __stcg(mine + (g * kChunk + half * 32 + k) * kRows + r, v[k]);
      }
      release(acc);
      __threadfence();
      epi_sync();
      if (lead) {
        atomicAdd(p.counters + 2 + tile, 1u);
        if (!wait_count(p, p.counters + 2 + tile, static_cast<unsigned>(w.split) * (step + 1))) *abort_flag = 1;
      }
      epi_sync();
    }
    const float2 dr = MODE >= STEP && !p.tall && i < p.m ? __ldcg(p.diag + static_cast<int64_t>(e) * p.s + i)
                                                         : make_float2(0.f, 0.f);
    for (int g = parts ? z : 0; g < chunks; g += parts ? w.split : 1, ++u) {
      const int b = static_cast<int>(u & 1), j = j0 + g * kChunk;
      const uint32_t set = sets + b * kSet;
      if (lead) {
        if (MODE == GRAM) prepare(u, e, i0, j);
        else if (g + 1 < chunks) prepare(u + 1, e, i0, j + kChunk);
      }
      float v[32];
      if (parts) {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = 0.f;
        for (int q = 0; q < w.split; ++q) {
          const float* from = part + (static_cast<int64_t>(q) * w.TN + g * kChunk + half * 32) * kRows + r;
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] += __ldcg(from + k * kRows);
        }
      } else {
        tmem_load32(ta + g * kChunk, v);
        if (g == chunks - 1) release(acc);
      }
      wait_or_abort(&sh.aux[b], static_cast<uint32_t>(u / 2) & 1, sh, p.err);
      finish32<MODE>(p, step, set, e, i, j + half * 32, r, half, mirror, dr, v);
      if (MODE <= STEP) {
        proxy_fence();
        epi_sync();
        if (lead) {
          if (MODE == STEP) {
            tma_store_3d(&p.xk[cur ^ 1], set, j, i0, e);
            tma_store_3d(&p.lo, set + kSet / 2, j, i0, e);
          } else {
            tma_store_3d(MODE == GRAM ? &p.ak : &p.bk, set, j, i0, e);
            if (mirror) {
              const CUtensorMap* to = MODE == GRAM ? &p.a64 : &p.b64;
              tma_store_3d(to, set + kSet / 2, i0, j, e);
              if (i0 + 64 < w.I) tma_store_3d(to, set + kSet / 2 + kChunk * 128, i0 + 64, j, e);
            }
          }
          bulk_commit();
        }
      } else {
        epi_sync();
        write_out<MODE>(p, set, e, i0, j, ew);
        epi_sync();
      }
    }
    if (chunks == 0 && !parts) release(acc);
  }
}

// All steps in one launch: every block walks each phase's work items (A, then
// B, then X), with a grid barrier between phases.  One block per SM; CG = 2:
// pairs of blocks share 256 x 256 tiles, each holding half of the operands.
template <int CG>
__global__ void __launch_bounds__(kThreads, 1) chain(const __grid_constant__ ChainP p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ __align__(8) Shared sh;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sets = smem + kStages * kStageBytes;
  const int warp = threadIdx.x >> 5;
  const int rank = CG == 1 ? 0 : static_cast<int>(cluster_rank());
  constexpr int kColumns = 2 * 128 * CG;
  if (threadIdx.x == 0) {
    sh.abort = 0;
    sh.aux_issued[0] = sh.aux_issued[1] = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.done[i], 1);
      mbar_init(&sh.freed[i], CG * kEpiWarps);
      mbar_init(&sh.aux[i], 1);
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
  int64_t n = 0, c = 0, u = 0;
  unsigned phase = 0;
  bool ok = true;
  for (int step = 0; step < p.steps && ok; ++step) {
    const int cur = step & 1;
    for (int ph = 0; ph < 3; ++ph) {
      const int mode = ph < STEP ? ph : step + 1 < p.steps ? static_cast<int>(STEP) : p.last;
      bool good = true;
      if (warp == 0) {
        if (loads) good = load_phase<CG>(p, sh, smem, mode, cur, rank, n);
      } else if (warp == 1) {
        if (issues) good = issue_phase<CG>(p, sh, smem, tmem, mode, n, c);
      } else {
        switch (mode) {
          case GRAM: finish_phase<CG, GRAM>(p, sh, sets, tmem, step, cur, rank, c, u); break;
          case POLY: finish_phase<CG, POLY>(p, sh, sets, tmem, step, cur, rank, c, u); break;
          case STEP: finish_phase<CG, STEP>(p, sh, sets, tmem, step, cur, rank, c, u); break;
          case LAST: finish_phase<CG, LAST>(p, sh, sets, tmem, step, cur, rank, c, u); break;
          default: finish_phase<CG, UPDATE>(p, sh, sets, tmem, step, cur, rank, c, u);
        }
        if (threadIdx.x == kLead) bulk_wait<0>();  // this phase's stores are written
        proxy_fence();
        __threadfence();
      }
      if (!good) *abort_flag = 1;
      __syncthreads();
      if (step + 1 == p.steps && ph == 2) break;
      if (threadIdx.x == 0) {
        // every block has finished the phase
        ++phase;
        if (*abort_flag) atomicExch(p.counters + 1, 1u);
        __threadfence();
        atomicAdd(p.counters, 1u);
        if (!wait_count(p, p.counters, phase * gridDim.x)) *abort_flag = 1;
      }
      __syncthreads();
      proxy_fence();
      if (*abort_flag) {
        ok = false;
        break;
      }
    }
  }
  // nothing is in flight when shared memory and accumulators are given up
  if (loads)
    for (int64_t i = n > kStages ? n - kStages : 0; i < n && rank == 0; ++i)
      mbar_wait(&sh.full[i % kStages], static_cast<uint32_t>(i / kStages) & 1, nullptr);
  if (threadIdx.x == kLead && *abort_flag)
    for (int b = 0; b < 2; ++b)
      if (sh.aux_issued[b]) mbar_wait(&sh.aux[b], static_cast<uint32_t>((sh.aux_issued[b] - 1) / 2) & 1, nullptr);
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

struct PrepP {
  Elem g, mom, mom_out;
  int has_mom, nesterov;
  float mu;
  int64_t rows, cols, ldx;  // of one matrix
  float eps;
  __half* hi;
  __half* lo;
  float* partials;  // [E, blocks]
  unsigned* counters;
  int count;  // of them, cleared for the chain of products
};

// The matrix to be orthogonalised at (r, c): the gradient or the momentum's
// look-ahead; m' in `m`.
__device__ __forceinline__ float prep_value(const PrepP& p, int64_t e, int64_t r, int64_t c, float& m) {
  const float g = load_elem(p.g, e * p.g.sb + r * p.g.sr + c * p.g.sc);
  if (!p.has_mom) return g;
  m = p.mu * load_elem(p.mom, e * p.mom.sb + r * p.mom.sr + c * p.mom.sc) + (1.0f - p.mu) * g;
  return p.nesterov ? p.mu * m + (1.0f - p.mu) * g : m;
}

// Sums of squares, a block's in a fixed order.
__global__ void __launch_bounds__(256) prep_norm(const PrepP p) {
  __shared__ float slots[2][32];
  const int64_t e = blockIdx.y, total = p.rows * p.cols;
  if (blockIdx.x == 0 && e == 0)
    for (int i = threadIdx.x; i < p.count; i += blockDim.x) p.counters[i] = 0;
  float ss = 0.f;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / p.cols;
    float m;
    const float u = prep_value(p, e, r, i - r * p.cols, m);
    ss = fmaf(u, u, ss);
  }
  ss = block_sum(ss, slots, 0);
  if (threadIdx.x == 0) p.partials[e * gridDim.x + blockIdx.x] = ss;
}

// X = u / (|u| + eps) as hi + lo, and the new momentum.
__global__ void __launch_bounds__(256) prep_scale(const PrepP p, int blocks) {
  __shared__ float slots[2][32];
  const int64_t e = blockIdx.y, total = p.rows * p.cols;
  float ss = 0.f;
  for (int i = threadIdx.x; i < blocks; i += blockDim.x) ss += p.partials[e * blocks + i];
  const float f = kXScale / (sqrtf(block_sum(ss, slots, 0)) + p.eps);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / p.cols, c = i - r * p.cols;
    float m;
    const float x = prep_value(p, e, r, c, m) * f;
    if (p.has_mom) store_elem(p.mom_out, (e * p.rows + r) * p.cols + c, m);
    const __half h = __float2half_rn(x);
    const int64_t o = (e * p.rows + r) * p.ldx + c;
    p.hi[o] = h;
    p.lo[o] = __float2half_rn(x - __half2float(h));
  }
}

// -------------------------------------------------------------------- host

struct Plan {
  int64_t s, l, ldx, lds, tiles;
  size_t hi0, hi1, lo, a, b, diag, partials, sums, counters, bytes;
  int blocks, pairs, groups, split, count;
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
  // Pairs of blocks and 256 x 256 tiles where X has enough of them to keep the
  // pairs busy; single blocks and 128 x 128 tiles below.
  q.pairs = resident(true) > 0 && chain_tiles(E, m, n, 256, false) >= resident(true) / 2;
  q.groups = resident(q.pairs);
  const int64_t side = q.pairs ? 256 : 128;
  q.tiles = chain_tiles(E, q.s, q.s, side, true);
  // A's few tiles with a long k: each in `split` parts of at least four
  // k-slices, one work item a group.
  const int64_t ks = ceil_div(q.l, kTileK);
  q.split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({q.groups / std::max<int64_t>(1, q.tiles), ks / 4, 8})));
  const size_t x = align_up(static_cast<size_t>(E) * m * q.ldx * 2, 256);
  const size_t a = align_up(static_cast<size_t>(E) * q.s * q.lds * 2, 256);
  q.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(1024, ceil_div(m * n, 4096))));
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
  q.bytes = q.sums + (q.split > 1 ? static_cast<size_t>(q.tiles) * q.split * side * side * sizeof(float) : 0);
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
  attr[0].id = cudaLaunchAttributeCooperative;  // the grid barrier needs every block resident
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 1 ? 1 : 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p));
}

int orthogonalise(const PrepP& prep, const Plan& q, int64_t E, int64_t m, int64_t n, int steps, const float* co,
                  Elem out, const Elem* par, float keep, float rate, unsigned char* ws, cudaStream_t s) {
  if (q.groups <= 0) return FRAG_ERR_NO_DEVICE;
  PrepP pp = prep;
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
  p.diag = reinterpret_cast<float2*>(ws + q.diag);
  p.partials = reinterpret_cast<float*>(ws + q.sums);
  p.counters = pp.counters;
  p.last = par ? UPDATE : LAST;
  p.out = out;
  if (par) p.par = *par;
  p.keep = keep;
  p.rate = rate;
  p.err = device_error_word();
  for (int i = 0; i < 3 * steps; ++i) p.co[i] = co[i];

  const dim3 grid(static_cast<unsigned>(q.blocks), static_cast<unsigned>(E));
  prep_norm<<<grid, 256, 0, s>>>(pp);
  prep_scale<<<grid, 256, 0, s>>>(pp, q.blocks);
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
  if (m > 0 && n > 0 && chain_tiles(E, m, n, 128, false) > (1 << 24)) return FRAG_ERR_SHAPE;
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
  return make_plan(E, m, n).bytes;
}

int frag_orthogonalize(const frag_matrix* g, void* out, int64_t E, int64_t m, int64_t n, int steps,
                       const float* coefficients, float eps, void* workspace, size_t workspace_bytes,
                       frag_stream_t stream) {
  const int bad = check_sizes(E, m, n, steps, coefficients);
  if (bad != FRAG_OK) return bad;
  if (E == 0 || m == 0 || n == 0) return FRAG_OK;
  PrepP prep = {};
  if (!elem_of(g, prep.g) || !out) return FRAG_ERR_INVALID_ARG;
  const Plan q = make_plan(E, m, n);
  if (!workspace || workspace_bytes < q.bytes) return FRAG_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FRAG_ERR_ALIGN;
  prep.rows = m;
  prep.cols = n;
  prep.ldx = q.ldx;
  prep.eps = eps;
  const Elem o{out, 0, m * n, n, 1};
  return orthogonalise(prep, q, E, m, n, steps, coefficients, o, nullptr, 0.f, 0.f,
                       static_cast<unsigned char*>(workspace), reinterpret_cast<cudaStream_t>(stream));
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
  const Plan q = make_plan(E, m, n);
  if (!workspace || workspace_bytes < q.bytes) return FRAG_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FRAG_ERR_ALIGN;
  prep.mom_out = Elem{momentum_out, prep.mom.f32, m * n, n, 1};
  prep.has_mom = 1;
  prep.nesterov = nesterov;
  prep.mu = mu;
  prep.rows = m;
  prep.cols = n;
  prep.ldx = q.ldx;
  prep.eps = eps;
  const Elem o{param_out, par.f32, m * n, n, 1};
  return orthogonalise(prep, q, E, m, n, steps, coefficients, o, &par, 1.0f - lr * weight_decay, lr * scale,
                       static_cast<unsigned char*>(workspace), reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"

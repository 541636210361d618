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

constexpr float kXScale = 256.0f;  // X is kept times 2^8
constexpr float kAScale = 1024.0f;  // A and B times 2^10
constexpr int kT = 128;             // tile side
constexpr int kStages = 6;
constexpr int kStageBytes = 2 * kT * kTileK * 2;
constexpr int kThreads = 192;  // a loading warp, an issuing warp, four for the epilogue
constexpr int kSmem = kStages * kStageBytes + 1024;

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

struct ProductP {
  CUtensorMap mp, mq;  // operands: C[i, j] = sum_k P[i, k] Q[j, k]
  int I, J, K, E;
  int tall;
  // GRAM and POLY write A / B here, POLY reads A
  __half* c;
  const __half* a;
  int64_t ldc;      // row stride; a batch is I rows
  float2* diag;     // [E, s] B's diagonal in 32 bits and its rounding residual
  // STEP, LAST, UPDATE
  const __half* hi;
  __half* hi_out;
  __half* lo;
  int64_t ldx;
  float ca, cb, cc;   // the step's coefficients
  float lo_factor;    // 1 in the last two steps: the diagonal's product with lo
  Elem out, par;      // LAST, UPDATE; UPDATE also reads par
  float keep, rate;   // p' = keep p - rate O
  int* err;
};

__device__ __forceinline__ void unpack_h8(const uint4& v, float (&f)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack_h8(const float (&f)[8]) {
  uint4 v;
  __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  return v;
}

// Tile t of a batch: (row tile, column tile).  Symmetric products take the
// tiles on and below the diagonal.
template <bool SYM>
__device__ __forceinline__ void tile_at(int t, int tj_count, int& ti, int& tj) {
  if (SYM) {
    ti = static_cast<int>((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
    while (ti * (ti + 1) / 2 > t) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
  } else {
    ti = t / tj_count;
    tj = t - ti * tj_count;
  }
}

// Eight values of row i (< I) from column j on: what the tile's accumulator
// becomes.  Rows of the working buffers are padded to eight elements, so a
// group that is cut by the matrix's edge is still read and written whole.
template <int MODE>
__device__ __forceinline__ void finish8(const ProductP& p, int e, int i, int j, float (&v)[8], bool mirror) {
  if (MODE == GRAM || MODE == POLY) {
    const int64_t at = (static_cast<int64_t>(e) * p.I + i) * p.ldc + j;
    if (MODE == GRAM) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= kAScale / (kXScale * kXScale);
    } else {
      float a[8];
      unpack_h8(*reinterpret_cast<const uint4*>(p.a + at), a);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = p.cb * a[k] + (p.cc / kAScale) * v[k];
        if (j + k == i) p.diag[static_cast<int64_t>(e) * p.I + i] = make_float2(v[k], v[k] - __half2float(__float2half_rn(v[k])));
      }
    }
    *reinterpret_cast<uint4*>(p.c + at) = pack_h8(v);
    if (mirror) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (j + k < p.J) p.c[(static_cast<int64_t>(e) * p.I + j + k) * p.ldc + i] = __float2half_rn(v[k]);
    }
    return;
  }
  const int64_t at = (static_cast<int64_t>(e) * p.I + i) * p.ldx + j;
  float h[8], l[8];
  unpack_h8(*reinterpret_cast<const uint4*>(p.hi + at), h);
  unpack_h8(*reinterpret_cast<const uint4*>(p.lo + at), l);
  const float2* diag = p.diag + static_cast<int64_t>(e) * (p.tall ? p.J : p.I);
  const float2 dr = p.tall ? make_float2(0.f, 0.f) : diag[i];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 d = p.tall ? (j + k < p.J ? diag[j + k] : make_float2(0.f, 0.f)) : dr;
    v[k] = p.ca * (h[k] + l[k]) + (v[k] + d.y * h[k] + p.lo_factor * d.x * l[k]) * (1.0f / kAScale);
  }
  if (MODE == STEP) {
    *reinterpret_cast<uint4*>(p.hi_out + at) = pack_h8(v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] -= __half2float(__float2half_rn(v[k]));
    *reinterpret_cast<uint4*>(p.lo + at) = pack_h8(v);
    return;
  }
  const int64_t o = static_cast<int64_t>(e) * p.out.sb + i * p.out.sr + j;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (j + k >= p.J) break;
    float r = v[k] * (1.0f / kXScale);
    if (MODE == UPDATE)
      r = p.keep * load_elem(p.par, static_cast<int64_t>(e) * p.par.sb + i * p.par.sr + (j + k) * p.par.sc) - p.rate * r;
    store_elem(p.out, o + k, r);
  }
}

// C = P Q' tile by tile: one CTA per SM walks 128 x 128 tiles; a thread loads
// k-slices of both operands by TMA into a ring, a thread issues the matrix
// instructions into one of two accumulators, four warps finish the other.
template <bool P_MN, bool Q_MN, int MODE>
__global__ void __launch_bounds__(kThreads, 1) product(const __grid_constant__ ProductP p) {
  constexpr bool SYM = MODE == GRAM || MODE == POLY;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], done[2], freed[2], drain;
  __shared__ uint32_t tmem_slot;
  __shared__ int s_abort;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5;
  const int ti_count = (p.I + kT - 1) / kT, tj_count = (p.J + kT - 1) / kT;
  const int per = SYM ? ti_count * (ti_count + 1) / 2 : ti_count * tj_count;
  const int64_t tiles = static_cast<int64_t>(per) * p.E;
  const int ks = (p.K + kTileK - 1) / kTileK;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&done[i], 1);
      mbar_init(&freed[i], 4);
    }
    mbar_init(&drain, 1);
    mbar_init_fence();
    tma_prefetch_map(&p.mp);
    tma_prefetch_map(&p.mq);
  }
  if (warp == 1) tmem_alloc(&tmem_slot, 2 * kT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  volatile int* const abort_flag = &s_abort;

  if (warp == 0) {
    if (elect_one()) {
      int64_t n = 0;  // k-slices issued
      bool ok = true;
      for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int e = static_cast<int>(t / per);
        int ti, tj;
        tile_at<SYM>(static_cast<int>(t - static_cast<int64_t>(e) * per), tj_count, ti, tj);
        for (int k = 0; k < ks; ++k, ++n) {
          const int st = static_cast<int>(n % kStages);
          if (n >= kStages && !mbar_wait(&empty[st], static_cast<uint32_t>(n / kStages - 1) & 1, p.err)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          if (*abort_flag) {
            ok = false;
            break;
          }
          const uint32_t sp = smem + st * kStageBytes, sq = sp + kStageBytes / 2;
          mbar_arrive_expect_tx(&full[st], kStageBytes);
          if (P_MN) {
            tma_load_3d(sp, &p.mp, &full[st], ti * kT, k * kTileK, e);
            tma_load_3d(sp + 64 * kTileK * 2, &p.mp, &full[st], ti * kT + 64, k * kTileK, e);
          } else {
            tma_load_3d(sp, &p.mp, &full[st], k * kTileK, ti * kT, e);
          }
          if (Q_MN) {
            tma_load_3d(sq, &p.mq, &full[st], tj * kT, k * kTileK, e);
            tma_load_3d(sq + 64 * kTileK * 2, &p.mq, &full[st], tj * kT + 64, k * kTileK, e);
          } else {
            tma_load_3d(sq, &p.mq, &full[st], k * kTileK, tj * kT, e);
          }
        }
      }
      // every copy has landed before the block may end
      for (int64_t i = n > kStages ? n - kStages : 0; i < n; ++i)
        mbar_wait(&full[i % kStages], static_cast<uint32_t>(i / kStages) & 1, nullptr);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = instr_desc_f16(kT, kT, P_MN, Q_MN);
      int64_t n = 0, c = 0;  // k-slices, tiles
      bool ok = true;
      for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++c) {
        const int acc = static_cast<int>(c & 1);
        if (c >= 2 && !mbar_wait(&freed[acc], static_cast<uint32_t>(c / 2 - 1) & 1, p.err)) ok = false;
        tc_fence_after();
        const uint32_t d = tmem + acc * kT;
        for (int k = 0; k < ks && ok; ++k, ++n) {
          const int st = static_cast<int>(n % kStages);
          if (*abort_flag || !mbar_wait(&full[st], static_cast<uint32_t>(n / kStages) & 1, p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sp = smem + st * kStageBytes;
          const uint64_t da = smem_desc<P_MN>(sp), db = smem_desc<Q_MN>(sp + kStageBytes / 2);
#pragma unroll
          for (int kk = 0; kk < kTileK / 16; ++kk)
            mma_f16(d, da + kk * desc_k16<P_MN>(), db + kk * desc_k16<Q_MN>(), idesc, k > 0 || kk > 0);
          mma_commit(&empty[st]);
        }
        if (ok) mma_commit(&done[acc]);
      }
      if (!ok) *abort_flag = 1;
      mma_commit(&drain);  // nothing is in flight when the accumulators are freed
      mbar_wait(&drain, 0, p.err);
    }
  } else {
    const int quad = warp & 3, lane = threadIdx.x & 31;
    int64_t c = 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, ++c) {
      const int e = static_cast<int>(t / per);
      int ti, tj;
      tile_at<SYM>(static_cast<int>(t - static_cast<int64_t>(e) * per), tj_count, ti, tj);
      const int acc = static_cast<int>(c & 1);
      const bool ok = !*abort_flag && mbar_wait(&done[acc], static_cast<uint32_t>(c / 2) & 1, p.err);
      if (!__all_sync(0xffffffffu, ok)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const int i = ti * kT + quad * 32 + lane;
      for (int j0 = 0; j0 < kT; j0 += 32) {
        float v[32];
        tmem_load32(tmem + (static_cast<uint32_t>(quad * 32) << 16) + acc * kT + j0, v);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int j = tj * kT + j0 + 8 * g;
          float u[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) u[k] = v[8 * g + k];
          if (i < p.I && j < p.J) finish8<MODE>(p, e, i, j, u, SYM && tj < ti);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&freed[acc]);
    }
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free(tmem, 2 * kT);
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
  int64_t s, l, ldx, lds;
  size_t hi0, hi1, lo, a, b, diag, partials, bytes;
  int blocks;
};

Plan make_plan(int64_t E, int64_t m, int64_t n) {
  Plan q;
  q.s = std::min(m, n);
  q.l = std::max(m, n);
  q.ldx = ceil_div(n, 8) * 8;
  q.lds = ceil_div(q.s, 8) * 8;
  const size_t x = align_up(static_cast<size_t>(E) * m * q.ldx * 2, 256);
  const size_t a = align_up(static_cast<size_t>(E) * q.s * q.lds * 2, 256);
  q.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(1024, ceil_div(m * n, 4096))));
  q.hi0 = 0;
  q.hi1 = x;
  q.lo = 2 * x;
  q.a = 3 * x;
  q.b = q.a + a;
  q.diag = q.b + a;
  q.partials = q.diag + align_up(static_cast<size_t>(E) * q.s * sizeof(float2), 256);
  q.bytes = q.partials + align_up(static_cast<size_t>(E) * q.blocks * sizeof(float), 256);
  return q;
}

template <bool P_MN, bool Q_MN, int MODE>
int launch_product(const ProductP& p, cudaStream_t s) {
  auto kern = product<P_MN, Q_MN, MODE>;
  if (!allow_dynamic_smem(reinterpret_cast<const void*>(kern), kSmem)) return FRAG_ERR_CUDA;
  const int64_t ti = ceil_div(p.I, kT), tj = ceil_div(p.J, kT);
  const int64_t tiles = p.E * ((MODE == GRAM || MODE == POLY) ? ti * (ti + 1) / 2 : ti * tj);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(tiles, std::max(1, sm_count()))));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p));
}

int orthogonalise(const PrepP& prep, const Plan& q, int64_t E, int64_t m, int64_t n, int steps, const float* co,
                  Elem out, const Elem* par, float keep, float rate, unsigned char* ws, cudaStream_t s) {
  PrepP pp = prep;
  pp.hi = reinterpret_cast<__half*>(ws + q.hi0);
  pp.lo = reinterpret_cast<__half*>(ws + q.lo);
  pp.partials = reinterpret_cast<float*>(ws + q.partials);
  const dim3 grid(static_cast<unsigned>(q.blocks), static_cast<unsigned>(E));
  prep_norm<<<grid, 256, 0, s>>>(pp);
  prep_scale<<<grid, 256, 0, s>>>(pp, q.blocks);
  int st = check_launch();
  if (st != FRAG_OK) return st;

  const bool tall = m > n;
  __half* hi[2] = {reinterpret_cast<__half*>(ws + q.hi0), reinterpret_cast<__half*>(ws + q.hi1)};
  __half* A = reinterpret_cast<__half*>(ws + q.a);
  __half* B = reinterpret_cast<__half*>(ws + q.b);
  CUtensorMap xk[2], xm[2], ak, bk;  // X along its rows, X across them, A, B
  for (int i = 0; i < 2; ++i)
    if (!make_map_3d(&xk[i], hi[i], n, m, E, q.ldx, m * q.ldx, kTileK, kT) ||
        !make_map_3d(&xm[i], hi[i], n, m, E, q.ldx, m * q.ldx, 64, kTileK))
      return FRAG_ERR_CUDA;
  if (!make_map_3d(&ak, A, q.s, q.s, E, q.lds, q.s * q.lds, kTileK, kT) ||
      !make_map_3d(&bk, B, q.s, q.s, E, q.lds, q.s * q.lds, kTileK, kT))
    return FRAG_ERR_CUDA;

  ProductP p = {};
  p.E = static_cast<int>(E);
  p.tall = tall;
  p.ldc = q.lds;
  p.ldx = q.ldx;
  p.a = A;
  p.diag = reinterpret_cast<float2*>(ws + q.diag);
  p.lo = pp.lo;
  p.out = out;
  if (par) p.par = *par;
  p.keep = keep;
  p.rate = rate;
  p.err = device_error_word();
  for (int k = 0; k < steps; ++k) {
    const int cur = k & 1;
    p.ca = co[3 * k];
    p.cb = co[3 * k + 1];
    p.cc = co[3 * k + 2];
    p.lo_factor = k >= steps - 2 ? 1.0f : 0.0f;
    p.I = p.J = static_cast<int>(q.s);
    p.K = static_cast<int>(q.l);
    p.c = A;
    p.mp = p.mq = tall ? xm[cur] : xk[cur];
    st = tall ? launch_product<true, true, GRAM>(p, s) : launch_product<false, false, GRAM>(p, s);
    if (st != FRAG_OK) return st;
    p.K = static_cast<int>(q.s);
    p.c = B;
    p.mp = p.mq = ak;
    st = launch_product<false, false, POLY>(p, s);
    if (st != FRAG_OK) return st;
    p.I = static_cast<int>(m);
    p.J = static_cast<int>(n);
    p.hi = hi[cur];
    p.hi_out = hi[cur ^ 1];
    p.mp = tall ? xk[cur] : bk;
    p.mq = tall ? bk : xm[cur];
    const int mode = k + 1 < steps ? STEP : par ? UPDATE : LAST;
    if (tall)
      st = mode == STEP ? launch_product<false, false, STEP>(p, s)
           : mode == LAST ? launch_product<false, false, LAST>(p, s)
                          : launch_product<false, false, UPDATE>(p, s);
    else
      st = mode == STEP ? launch_product<false, true, STEP>(p, s)
           : mode == LAST ? launch_product<false, true, LAST>(p, s)
                          : launch_product<false, true, UPDATE>(p, s);
    if (st != FRAG_OK) return st;
  }
  return FRAG_OK;
}

int check_sizes(int64_t E, int64_t m, int64_t n, int steps, const float* co) {
  if (E < 0 || m < 0 || n < 0 || steps < 1 || !co) return FRAG_ERR_INVALID_ARG;
  if (m > (1 << 30) || n > (1 << 30) || E > 65535) return FRAG_ERR_SHAPE;
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

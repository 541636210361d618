// grad_norm.cu — the 2-norm of many tensors together and the factor that
// clips it:
//   norm = sqrt(sum of g^2),  scale = max_norm / max(norm, max_norm)
// and NaN for a norm that is not finite, which the weight update takes as the
// word to leave everything as it is.
//
// One pass over the data.  Block b of G owns the chunks [b C / G, (b + 1) C / G)
// of all tensors' C, so the order of the sums depends on sizes and alignment alone.
// A thread adds the 32 squares that it has of a chunk in 32 bits and everything
// beyond in 64 (a long run of equal gradients would round the same way every time);
// a second, one-block launch adds the blocks' sums and starts while the first ends.
//
// Bound: HBM.  218 million values in 9 tensors: 75 us in bf16 (5.8 TB/s; 67 at a
// copy's rate; 70 among other calls), 140 in fp32 (6.3), from addresses off 16 bytes too.  Tensors
// of a few thousand values are a chunk each, and the two launches' latency.
#include <algorithm>
#include <cmath>

#include "tensor_list.cuh"

namespace frag {
namespace {

constexpr int kThreads = 512;
constexpr int64_t kChunk = 16384;   // values
constexpr int kBlocksPerSm = 4;

template <int CAP>
struct NormList {
  const void* ptr[CAP];
  int64_t numel[CAP];
  uint32_t first[CAP + 1];
  uint8_t f32[CAP];
  int count;
  uint32_t chunks;
};

// Sum over the block in a fixed order, for thread 0.
__device__ __forceinline__ double block_sum_double(double a, double* slots) {
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = a;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x == 0)
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) t += slots[i];
  return t;
}

__device__ __forceinline__ float square8(const uint4& v, float a) {
  float2 s = make_float2(a, 0.f);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 f = bf16x2_to_f2(u4_word(v, q));
    s = __ffma2_rn(f, f, s);
  }
  return s.x + s.y;
}

// Sum of squares of n values from p on, by the whole block: what lies before
// the first and behind the last 16-byte boundary one by one.
template <class T>
__device__ __forceinline__ float chunk_squares(const T* p, int64_t n) {
  constexpr int E = 16 / sizeof(T);
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
  const int head = static_cast<int>(min(n, static_cast<int64_t>((E - off) % E)));
  const int64_t body = (n - head) / E;
  const int tail = static_cast<int>(n - head - body * E);
  float a = 0.f;
  const uint4* v = reinterpret_cast<const uint4*>(p + head);
  const int t = threadIdx.x;
#pragma unroll 4
  for (int64_t i = t; i < body; i += kThreads) {
    const uint4 u = ld_stream(v + i);
    if (sizeof(T) == 2) {
      a = square8(u, a);
    } else {
      const float4 f = *reinterpret_cast<const float4*>(&u);
      a = fmaf(f.x, f.x, a);
      a = fmaf(f.y, f.y, a);
      a = fmaf(f.z, f.z, a);
      a = fmaf(f.w, f.w, a);
    }
  }
  if (t < head + tail) {
    const T u = p[t < head ? t : head + body * E + (t - head)];
    const float f = sizeof(T) == 2 ? bf16_to_f(static_cast<uint16_t>(u)) : static_cast<float>(u);
    a = fmaf(f, f, a);
  }
  return a;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads) squares(const __grid_constant__ NormList<CAP> L, double* partials) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ double slots[32];
  const uint32_t G = gridDim.x;
  uint32_t c = static_cast<uint32_t>(static_cast<uint64_t>(L.chunks) * blockIdx.x / G);
  const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(L.chunks) * (blockIdx.x + 1) / G);
  double a = 0.0;
  int i = find_tensor(L.first, L.count, c);
  for (; c < end; ++c) {
    while (c >= L.first[i + 1]) ++i;
    // Chunks end at 16-byte boundaries: only a tensor's first and last have values
    // beside them.
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(L.ptr[i]) & 15u) >> (L.f32[i] ? 2 : 1));
    const int64_t at = static_cast<int64_t>(c - L.first[i]) * kChunk - off, from = max(at, static_cast<int64_t>(0));
    const int64_t n = (c + 1 == L.first[i + 1] ? L.numel[i] : at + kChunk) - from;
    a += L.f32[i] ? chunk_squares(static_cast<const float*>(L.ptr[i]) + from, n)
                  : chunk_squares(static_cast<const uint16_t*>(L.ptr[i]) + from, n);
  }
  a = block_sum_double(a, slots);
  if (threadIdx.x == 0) partials[blockIdx.x] = a;
}

__global__ void __launch_bounds__(1024) norm_finish(const double* partials, int count, float max_norm, float* norm,
                                                     float* scale) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ double slots[32];
  double t = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) t += partials[i];
  t = block_sum_double(t, slots);
  if (threadIdx.x != 0) return;
  const float n = static_cast<float>(sqrt(t));
  *norm = n;
  if (scale) *scale = isfinite(n) ? max_norm / fmaxf(n, max_norm) : __uint_as_float(0x7fffffffu);
}

int64_t list_chunks(const int64_t* numel, int64_t count) {
  int64_t c = 0;
  for (int64_t i = 0; i < count; ++i) c += ceil_div(numel[i], kChunk);
  return c;
}

int64_t list_blocks(int64_t chunks, int sms) {
  return std::min<int64_t>(chunks, static_cast<int64_t>(sms) * kBlocksPerSm);
}

template <int CAP>
int launch_squares(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int count, int64_t chunks,
                   int64_t blocks, double* partials, cudaStream_t s) {
  NormList<CAP> L;
  uint32_t c = 0;
  for (int i = 0; i < count; ++i) {
    L.ptr[i] = grads[i];
    L.numel[i] = numel[i];
    L.f32[i] = dtypes[i] == FRAG_DT_F32;
    L.first[i] = c;
    c += static_cast<uint32_t>(ceil_div(numel[i], kChunk));
  }
  L.first[count] = c;
  L.count = count;
  L.chunks = static_cast<uint32_t>(chunks);
  squares<CAP><<<dim3(static_cast<unsigned>(blocks)), kThreads, 0, s>>>(L, partials);
  return check_launch();
}

}  // namespace
}  // namespace frag

using namespace frag;

extern "C" {

size_t frag_grad_norm_workspace_bytes(int64_t count) {
  int sms = sm_count();
  if (sms <= 0) sms = 148;
  const int64_t launches = std::max<int64_t>(1, ceil_div(count, kListLarge));
  return align_up(static_cast<size_t>(launches) * sms * kBlocksPerSm * sizeof(double), 256);
}

int frag_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int64_t count,
                   float max_norm, float* norm, float* scale, void* workspace, size_t workspace_bytes,
                   frag_stream_t stream) {
  if (count < 0 || (count > 0 && (!grads || !numel || !dtypes)) || !norm) return FRAG_ERR_INVALID_ARG;
  if (scale && !(max_norm > 0.f && std::isfinite(max_norm))) return FRAG_ERR_INVALID_ARG;
  for (int64_t i = 0; i < count; ++i) {
    if (numel[i] < 0 || (numel[i] > 0 && !grads[i])) return FRAG_ERR_INVALID_ARG;
    if (dtypes[i] != FRAG_DT_BF16 && dtypes[i] != FRAG_DT_F32) return FRAG_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(grads[i]) % (dtypes[i] == FRAG_DT_F32 ? 4 : 2)) return FRAG_ERR_ALIGN;
    if (numel[i] > (1LL << 40)) return FRAG_ERR_SHAPE;
  }
  if (!workspace || workspace_bytes < frag_grad_norm_workspace_bytes(count)) return FRAG_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FRAG_ERR_ALIGN;
  const int sms = sm_count();
  if (sms <= 0) return FRAG_ERR_NO_DEVICE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  double* partials = static_cast<double*>(workspace);
  int64_t held = 0;
  for (int64_t i = 0; i < count; i += kListLarge) {
    const int n = static_cast<int>(std::min<int64_t>(kListLarge, count - i));
    const int64_t chunks = list_chunks(numel + i, n);
    if (chunks > 0xffffffffLL) return FRAG_ERR_SHAPE;
    if (chunks == 0) continue;
    const int64_t blocks = list_blocks(chunks, sms);
    const int st = n <= kListSmall
                       ? launch_squares<kListSmall>(grads + i, numel + i, dtypes + i, n, chunks, blocks,
                                                    partials + held, s)
                       : launch_squares<kListLarge>(grads + i, numel + i, dtypes + i, n, chunks, blocks,
                                                    partials + held, s);
    if (st != FRAG_OK) return st;
    held += blocks;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = held ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, norm_finish, static_cast<const double*>(partials),
                                        static_cast<int>(held), max_norm, norm, scale));
}

}  // extern "C"

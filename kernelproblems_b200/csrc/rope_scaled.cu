// rope_scaled.cu — rotary positions with given frequencies, on all or the
// first `rot` elements of each head, forward and gradient.
//
// Math, for pair j of a token at position p (f_j: turns per position, from
// the caller's plan; m: the plan's factor on the rotated values):
//   angle = 2 pi f_j p,  (a, b) -> m (a cos - b sin, b cos + a sin)
//   NEOX pairs (x[j], x[j + rot/2]); INTERLEAVED pairs (x[2j], x[2j+1])
// The gradient is the transpose: sin with the other sign, m unchanged.
// Elements rot..D of a head pass through (left alone when out is x itself).
//
// The angle: p f_j is taken in 64 bits and reduced to a fraction of a turn
// there, so a position deep in a long context loses nothing (the product in
// 32 bits is off by 4e-3 rad at p = 1e5); the sine and cosine of the reduced
// angle are then 32-bit (sincospif).  Rotated values are rounded once, to bf16.
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace frag {
namespace {

constexpr int kMaxPairs = 256;  // rot <= 512

struct ScaledT {
  const uint16_t* x;
  uint16_t* out;
  int H;
  int copy_rest;  // elements rot..D are copied (out is another buffer)
  int64_t xsb, xss, xsh, osb, oss, osh;
};

struct ScaledP {
  ScaledT t[2];
  int nt;
  int64_t B, S;
  int D, rot;
  const void* pos;
  int pos_dtype;
  int64_t psb, pss;
  float factor, sin_factor;  // m and +-m
  double turns[kMaxPairs];
};

__device__ __forceinline__ int64_t token_pos(const ScaledP& p, int64_t b, int64_t s) {
  if (p.pos_dtype == FRAG_POS_I32)
    return __ldg(static_cast<const int32_t*>(p.pos) + b * p.psb + s * p.pss);
  if (p.pos_dtype == FRAG_POS_I64)
    return __ldg(static_cast<const int64_t*>(p.pos) + b * p.psb + s * p.pss);
  return s;
}

// m cos and +-m sin of `turns` turns per position at position p.
__device__ __forceinline__ void turn(double turns, double p, const ScaledP& P, float& c, float& s) {
  double t = turns * p;
  t -= rint(t);  // exact: t and its nearest integer are within a factor of two or |t| < 1
  float sv, cv;
  sincospif(2.0f * static_cast<float>(t), &sv, &cv);
  c = cv * P.factor;
  s = sv * P.sin_factor;
}

// Any even rot, any strides: one CTA per token, one thread per pair or passed
// element, the token's sines and cosines in shared memory.
template <bool NEOX>
__global__ void __launch_bounds__(256) rope_scaled_any(const __grid_constant__ ScaledP p) {
  __shared__ float2 cs[kMaxPairs];
  const int half = p.rot >> 1, rest = p.D - p.rot;
  const int64_t tok = blockIdx.x;
  const int64_t b = tok / p.S, s = tok - b * p.S;
  const double pos = static_cast<double>(token_pos(p, b, s));
  for (int j = threadIdx.x; j < half; j += blockDim.x) turn(p.turns[j], pos, p, cs[j].x, cs[j].y);
  __syncthreads();
#pragma unroll
  for (int ti = 0; ti < 2; ++ti) {
    if (ti >= p.nt) break;
    const ScaledT& T = p.t[ti];
    const uint16_t* x = T.x + b * T.xsb + s * T.xss;
    uint16_t* out = T.out + b * T.osb + s * T.oss;
    const int per = half + (T.copy_rest ? rest : 0);
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(T.H) * per; i += blockDim.x) {
      const int h = static_cast<int>(i / per), j = static_cast<int>(i - static_cast<int64_t>(h) * per);
      if (j < half) {
        const int ia = NEOX ? j : 2 * j, ib = NEOX ? j + half : 2 * j + 1;
        const float a = bf16_to_f(x[h * T.xsh + ia]), c = bf16_to_f(x[h * T.xsh + ib]);
        out[h * T.osh + ia] = f_to_bf16(a * cs[j].x - c * cs[j].y);
        out[h * T.osh + ib] = f_to_bf16(c * cs[j].x + a * cs[j].y);
      } else {
        const int d = p.rot + j - half;
        out[h * T.osh + d] = x[h * T.xsh + d];
      }
    }
  }
}

}  // namespace
}  // namespace frag

using namespace frag;

extern "C" int frag_rope_scaled(const frag_rope_tensor* tensors, int num_tensors, int64_t B, int64_t S,
                                int64_t D, int64_t rot, const void* pos, int pos_dtype,
                                int64_t pos_stride_b, int64_t pos_stride_s, const double* turns,
                                float factor, int layout, int backward, frag_stream_t stream) {
  if (!tensors || num_tensors < 1 || num_tensors > 2 || !turns) return FRAG_ERR_INVALID_ARG;
  if (B < 0 || S < 0 || D < 0 || rot < 0) return FRAG_ERR_INVALID_ARG;
  if (layout != FRAG_ROPE_NEOX && layout != FRAG_ROPE_INTERLEAVED) return FRAG_ERR_INVALID_ARG;
  if (pos_dtype != FRAG_POS_NONE && pos_dtype != FRAG_POS_I32 && pos_dtype != FRAG_POS_I64)
    return FRAG_ERR_INVALID_ARG;
  if (pos_dtype != FRAG_POS_NONE && !pos) return FRAG_ERR_INVALID_ARG;
  if (B == 0 || S == 0) return FRAG_OK;
  if (rot == 0 || rot % 2 != 0 || rot > D || rot / 2 > kMaxPairs || D > 0x7fff) return FRAG_ERR_SHAPE;
  if (B > 0x7fffffffLL || S > 0x7fffffffLL || B * S > 0x7fffffffLL) return FRAG_ERR_SHAPE;
  ScaledP p;
  p.nt = num_tensors;
  p.B = B;
  p.S = S;
  p.D = static_cast<int>(D);
  p.rot = static_cast<int>(rot);
  p.pos = pos;
  p.pos_dtype = pos_dtype;
  p.psb = pos_stride_b;
  p.pss = pos_stride_s;
  p.factor = factor;
  p.sin_factor = backward ? -factor : factor;
  for (int j = 0; j < kMaxPairs; ++j) p.turns[j] = j < rot / 2 ? turns[j] : 0.0;
  p.t[1] = ScaledT{};
  bool any = false;
  for (int i = 0; i < num_tensors; ++i) {
    const frag_rope_tensor& t = tensors[i];
    if (t.H < 0 || t.H > 0x7fffffLL) return FRAG_ERR_SHAPE;
    if (t.H > 0 && (!t.x || !t.out)) return FRAG_ERR_INVALID_ARG;
    if (t.in_dtype != FRAG_ROPE_IN_BF16 || t.out_dtype != FRAG_ROPE_OUT_BF16) return FRAG_ERR_INVALID_ARG;
    const bool in_place = t.x == t.out;
    if (in_place && (t.x_stride_b != t.out_stride_b || t.x_stride_s != t.out_stride_s ||
                     t.x_stride_h != t.out_stride_h))
      return FRAG_ERR_INVALID_ARG;
    p.t[i] = ScaledT{static_cast<const uint16_t*>(t.x), static_cast<uint16_t*>(t.out), static_cast<int>(t.H),
                     in_place ? 0 : 1, t.x_stride_b, t.x_stride_s, t.x_stride_h, t.out_stride_b,
                     t.out_stride_s, t.out_stride_h};
    any = any || t.H > 0;
  }
  if (!any) return FRAG_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(B * S);
  if (layout == FRAG_ROPE_NEOX) rope_scaled_any<true><<<grid, 256, 0, s>>>(p);
  else rope_scaled_any<false><<<grid, 256, 0, s>>>(p);
  return check_launch();
}

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

// CH bf16 values that one access moves.
template <int CH> struct Chunk;
template <> struct Chunk<8> { typedef uint4 T; };
template <> struct Chunk<4> { typedef uint2 T; };
template <> struct Chunk<2> { typedef uint32_t T; };

template <int CH>
__device__ __forceinline__ void widen(const typename Chunk<CH>::T& v, float (&f)[CH]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < CH / 2; ++i) {
    f[2 * i] = bf16lo(w[i]);
    f[2 * i + 1] = bf16hi(w[i]);
  }
}
template <int CH>
__device__ __forceinline__ typename Chunk<CH>::T narrow(const float (&f)[CH]) {
  typename Chunk<CH>::T v;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < CH / 2; ++i) w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  return v;
}

// rot a multiple of 2 CH, heads and strides of CH elements.  A warp takes one
// token and a run of `span` head groups, q's and then k's; L = rot / (2 CH)
// lanes share a head, and lane j of it owns the chunks at CH j and rot/2 + CH j:
// whole pairs in either layout, the same frequencies in every head.  The warp
// makes the token's sines and cosines once, a lane a pair, and shares them.  The
// passed elements follow, chunk by chunk.
//
// Bound: HBM.  8 x 4096 tokens of 32 + 8 heads of 128: 110 us, 6.1 TB/s (93% of
// the measured copy).  Two head groups in flight and four warps a block
// measured best: 120 us for four groups and eight warps, 145 for one group at
// twice the occupancy; loading the next groups ahead 115 to 119; sines made by
// every head's lanes 112; stores without the streaming hint 2 us more.
constexpr int kWarps = 4;

template <int CH, bool NEOX>
__global__ void __launch_bounds__(32 * kWarps, 7) rope_scaled_vec(const __grid_constant__ ScaledP p, int splits, int span) {
  typedef typename Chunk<CH>::T V;
  constexpr int UNR = 2;
  __shared__ float2 shared_turns[kWarps][kMaxPairs];
  __shared__ double per_position[kMaxPairs];  // (a lane's own entry of a kernel argument would be 32 loads)
  float2* const turns = shared_turns[threadIdx.x >> 5];
  const int half = p.rot >> 1;
  for (int i = threadIdx.x; i < half; i += blockDim.x) per_position[i] = p.turns[i];
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t tok = w / splits;
  if (tok >= p.B * p.S) return;
  const int first = static_cast<int>(w - tok * splits) * span;
  const int64_t b = tok / p.S, s = tok - b * p.S;
  const double pos = static_cast<double>(token_pos(p, b, s));
  const int L = half / CH, HPG = 32 / L;  // lanes of a head, heads of a group
  const int j = lane % L, hs = lane / L;
  for (int f = lane; f < half; f += 32) turn(per_position[f], pos, p, turns[f].x, turns[f].y);
  __syncwarp();
  float cs[CH], sn[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int f = NEOX ? CH * j + i : (i < CH / 2 ? CH / 2 * j + i : (half >> 1) + CH / 2 * j + i - CH / 2);
    if (f < half) {
      cs[i] = turns[f].x;
      sn[i] = turns[f].y;
    }
  }
  const int rest = (p.D - p.rot) / CH;
  const int gq = (p.t[0].H + HPG - 1) / HPG;
  int base = 0;  // the tensor's first head group
#pragma unroll
  for (int ti = 0; ti < 2; ++ti) {
    if (ti >= p.nt) break;
    const ScaledT& T = p.t[ti];
    const int groups = ti == 0 ? gq : (T.H + HPG - 1) / HPG;
    const int g0 = max(first - base, 0), g1 = min(first + span - base, groups);
    base += groups;
    if (g0 >= g1) continue;
    const uint16_t* x = T.x + b * T.xsb + s * T.xss;
    uint16_t* out = T.out + b * T.osb + s * T.oss;
    const int h1 = min(T.H, g1 * HPG);
    for (int h0 = g0 * HPG + hs; hs < HPG && h0 < h1; h0 += HPG * UNR) {
      V va[UNR], vb[UNR];
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        const int h = h0 + u * HPG;
        if (h < h1) {
          va[u] = *reinterpret_cast<const V*>(x + h * T.xsh + CH * j);
          vb[u] = *reinterpret_cast<const V*>(x + h * T.xsh + half + CH * j);
        }
      }
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        const int h = h0 + u * HPG;
        if (h < h1) {
          float fa[CH], fb[CH], ra[CH], rb[CH];
          widen<CH>(va[u], fa);
          widen<CH>(vb[u], fb);
          if (NEOX) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
              ra[i] = fa[i] * cs[i] - fb[i] * sn[i];
              rb[i] = fb[i] * cs[i] + fa[i] * sn[i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) {
              ra[2 * i] = fa[2 * i] * cs[i] - fa[2 * i + 1] * sn[i];
              ra[2 * i + 1] = fa[2 * i + 1] * cs[i] + fa[2 * i] * sn[i];
              rb[2 * i] = fb[2 * i] * cs[CH / 2 + i] - fb[2 * i + 1] * sn[CH / 2 + i];
              rb[2 * i + 1] = fb[2 * i + 1] * cs[CH / 2 + i] + fb[2 * i] * sn[CH / 2 + i];
            }
          }
          __stcs(reinterpret_cast<V*>(out + h * T.osh + CH * j), narrow<CH>(ra));
          __stcs(reinterpret_cast<V*>(out + h * T.osh + half + CH * j), narrow<CH>(rb));
        }
      }
    }
    if (T.copy_rest && rest > 0) {
      const int hf = g0 * HPG, n = (h1 - hf) * rest;
      for (int i0 = lane; i0 < n; i0 += 32 * UNR) {
        V v[UNR];
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
          const int i = i0 + 32 * u, h = i / rest;
          if (i < n) v[u] = *reinterpret_cast<const V*>(x + (hf + h) * T.xsh + p.rot + CH * (i - h * rest));
        }
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
          const int i = i0 + 32 * u, h = i / rest;
          if (i < n) __stcs(reinterpret_cast<V*>(out + (hf + h) * T.osh + p.rot + CH * (i - h * rest)), v[u]);
        }
      }
    }
  }
}

// Whether every head of the call divides into chunks of CH elements.
bool fits(const ScaledP& p, int CH) {
  if (p.rot % (2 * CH) != 0 || p.D % CH != 0 || p.rot / (2 * CH) > 32) return false;
  for (int i = 0; i < p.nt; ++i) {
    const ScaledT& t = p.t[i];
    const int64_t st[6] = {t.xsb, t.xss, t.xsh, t.osb, t.oss, t.osh};
    for (int64_t v : st)
      if (v % CH != 0) return false;
    if ((reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.out)) % (2 * CH) != 0) return false;
  }
  return true;
}

template <int CH>
int launch_vec(const ScaledP& p, bool neox, cudaStream_t s) {
  const int HPG = 32 / (p.rot / (2 * CH));
  int64_t groups = 0;
  for (int i = 0; i < p.nt; ++i) groups += ceil_div(p.t[i].H, HPG);
  const int64_t tokens = p.B * p.S;
  int sms = sm_count();
  if (sms <= 0) sms = 148;
  // A token's sines cost as much as a few head groups, so a warp takes the
  // whole token while there are enough of them to fill the machine (16 warps
  // an SM), and the heads are split over more warps when there are not.
  const int64_t splits = std::max<int64_t>(1, std::min(groups, ceil_div(16LL * sms, tokens)));
  const int64_t span = ceil_div(groups, splits);
  const int64_t warps = tokens * ceil_div(groups, span);
  const int per = warps >= 8LL * sms ? kWarps : 2;  // warps of a block
  const int64_t grid = ceil_div(warps, per);
  if (grid > 0x7fffffffLL) return FRAG_ERR_SHAPE;
  auto kern = neox ? rope_scaled_vec<CH, true> : rope_scaled_vec<CH, false>;
  kern<<<static_cast<unsigned>(grid), 32 * per, 0, s>>>(p, static_cast<int>(ceil_div(groups, span)),
                                                        static_cast<int>(span));
  return check_launch();
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
    ScaledT& o = p.t[i];
    o = ScaledT{static_cast<const uint16_t*>(t.x), static_cast<uint16_t*>(t.out), static_cast<int>(t.H),
                in_place ? 0 : 1, t.x_stride_b, t.x_stride_s, t.x_stride_h, t.out_stride_b,
                t.out_stride_s, t.out_stride_h};
    // a dimension of one element has no stride to respect
    if (B == 1) o.xsb = o.osb = 0;
    if (S == 1) o.xss = o.oss = 0;
    if (t.H == 1) o.xsh = o.osh = 0;
    if (in_place && (o.xsb != o.osb || o.xss != o.oss || o.xsh != o.osh)) return FRAG_ERR_INVALID_ARG;
    any = any || t.H > 0;
  }
  if (!any) return FRAG_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool neox = layout == FRAG_ROPE_NEOX;
  if (fits(p, 8)) return launch_vec<8>(p, neox, s);
  if (fits(p, 4)) return launch_vec<4>(p, neox, s);
  if (fits(p, 2)) return launch_vec<2>(p, neox, s);
  const unsigned grid = static_cast<unsigned>(B * S);
  if (neox) rope_scaled_any<true><<<grid, 256, 0, s>>>(p);
  else rope_scaled_any<false><<<grid, 256, 0, s>>>(p);
  return check_launch();
}

// Norm of every query and key head and the rotation of its pairs by the token's position, in one pass, and its gradient.
//
//   y = x / sqrt(mean(x^2) + eps) * w;   (y_a, y_b) -> (y_a cos t - y_b sin t, y_a sin t + y_b cos t),  t = pos base^(-2i/D)
//   backward: u = the gradient turned back by t;  dw = sum u x r;  dx = r (u w - x r^2 mean(u w x)),  r = 1/sqrt(...)
//
// Bound by HBM: every element is read once and written once.  A group of lanes holds one head, each lane two vectors
// of its pairs, so norm, rotation and both sums stay in registers; a warp keeps the sines of its token for all its heads.
// Angles: base^(-2i/D) / 2 pi is a 64-bit fraction of a turn, and position times fraction wraps modulo one turn exactly,
// so far positions are as exact as near ones; only the angle within the turn is rounded to fp32.
#include <math.h>

#include "../api/chb.h"
#include "common.cuh"

namespace chb {
namespace {

constexpr int kMaxPairs = 128;      // D <= 256
constexpr int kThreads = 256, kWarps = kThreads / 32;

struct RopeArgs {
  const void* x[2];          // queries, keys
  const void* dy[2];         // backward: gradients of the outputs
  void* y[2];                // outputs, or gradients of x (contiguous)
  long long xt[2], xh[2];    // strides of a token and of a head, in elements
  long long dt[2], dh[2];
  int heads[2];
  const void* w[2];          // null: no norm
  int w_f32;
  const void* pos;           // null: 0, 1, 2, ...
  int pos64;
  int T, D, lanes, group;    // lanes of a head, and the power of two that holds them
  int iters[2], slices;      // turns of a warp over the heads of a token, and how many warps share them
  int interleaved;
  float eps;
  float* part;               // backward: sums of dw of each CTA, [CTA][2][D]
};
struct Turns { unsigned long long f[kMaxPairs]; };

template <typename T> __device__ __forceinline__ float2 two(uint32_t v);
template <> __device__ __forceinline__ float2 two<__nv_bfloat16>(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 two<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <typename T> __device__ __forceinline__ uint32_t from_two(float a, float b);
template <> __device__ __forceinline__ uint32_t from_two<__nv_bfloat16>(float a, float b) { const __nv_bfloat162 v = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&v); }
template <> __device__ __forceinline__ uint32_t from_two<__half>(float a, float b) { const __half2 v = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&v); }

// V neighbouring elements (8 or 16 bytes of 16-bit elements, 16 bytes of fp32) as fp32
template <typename T, int V> struct Vec {
  uint32_t r[V * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) == 16) {
      const uint4 a = __ldcg(reinterpret_cast<const uint4*>(p));
      r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
    } else {
      const uint2 a = __ldcg(reinterpret_cast<const uint2*>(p));
      r[0] = a.x; r[1] = a.y;
    }
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(r[i]);
      } else {
        const float2 v = two<T>(r[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) {
      if constexpr (sizeof(T) == 4) r[i] = __float_as_uint(f[i]);
      else r[i] = from_two<T>(f[2 * i], f[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_weights(const RopeArgs& a, int which, int e0, int e1, float* w) {
  if (a.w_f32) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[i] = reinterpret_cast<const float*>(a.w[which])[e0 + i];
      w[V + i] = reinterpret_cast<const float*>(a.w[which])[e1 + i];
    }
  } else {
    Vec<T, V> p, q;
    p.load(reinterpret_cast<const T*>(a.w[which]) + e0);
    q.load(reinterpret_cast<const T*>(a.w[which]) + e1);
    p.get(w);
    q.get(w + V);
  }
}

// f[0..V) and f[V..2V) are the lane's two vectors.  Interleaved: 2V neighbours, pairs (2i, 2i + 1); else the i-th of the
// first vector and the i-th of the second.
template <int V, bool BACK>
__device__ __forceinline__ void turn(float* f, const float* c, const float* s, bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = f[2 * i], y = f[2 * i + 1], sn = BACK ? -s[i] : s[i];
      f[2 * i] = x * c[i] - y * sn;
      f[2 * i + 1] = x * sn + y * c[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = f[i], y = f[V + i], sn = BACK ? -s[i] : s[i];
      f[i] = x * c[i] - y * sn;
      f[V + i] = x * sn + y * c[i];
    }
  }
}

template <typename T, int V, bool NORM, bool BACK>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeArgs a, const Turns turns) {
  __shared__ float sums[BACK && NORM ? kWarps * 2 * 256 : 1];
  dependent_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & (a.group - 1), per = 32 / a.group, mine = lane / a.group;
  const bool live = sub < a.lanes;
  const int e0 = a.interleaved ? sub * 2 * V : sub * V, e1 = a.interleaved ? e0 + V : a.D / 2 + sub * V;
  const float inv_d = 1.f / (float)a.D;
  float dw[2][BACK && NORM ? 2 * V : 1];
  if constexpr (BACK && NORM) {
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) dw[0][i] = dw[1][i] = 0.f;
  }
  const int total = a.iters[0] + a.iters[1];
  const long long items = (long long)a.T * a.slices;
  for (long long it = (long long)blockIdx.x * kWarps + warp; it < items; it += (long long)gridDim.x * kWarps) {
    const long long t = it / a.slices;
    const int slice = (int)(it - t * a.slices);
    const int i0 = (int)((long long)total * slice / a.slices), i1 = (int)((long long)total * (slice + 1) / a.slices);
    const long long pos = !a.pos ? t : a.pos64 ? reinterpret_cast<const long long*>(a.pos)[t] : (long long)reinterpret_cast<const int*>(a.pos)[t];
    float c[V], s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const unsigned long long ph = (unsigned long long)pos * turns.f[live ? sub * V + i : 0];
      sincospif((float)(int)(ph >> 32) * 4.656612873077392578125e-10f, &s[i], &c[i]);      // (2^-31: in half turns)
    }
#pragma unroll 2
    for (int i = i0; i < i1; ++i) {
      const int which = i >= a.iters[0];
      const int head = (which ? i - a.iters[0] : i) * per + mine;
      const bool on = live && head < a.heads[which];
      const T* x = reinterpret_cast<const T*>(a.x[which]) + t * a.xt[which] + head * a.xh[which];
      T* y = reinterpret_cast<T*>(a.y[which]) + (t * a.heads[which] + head) * a.D;
      Vec<T, V> p, q, dp, dq;
      float f[2 * V], g[2 * V], w[2 * V];
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) f[j] = g[j] = 0.f;
      if (on && (NORM || !BACK)) { p.load(x + e0); q.load(x + e1); }
      if (BACK && on) {
        const T* d = reinterpret_cast<const T*>(a.dy[which]) + t * a.dt[which] + head * a.dh[which];
        dp.load(d + e0);
        dq.load(d + e1);
      }
      if (NORM && on) load_weights<T, V>(a, which, e0, e1, w);
      if (on && (NORM || !BACK)) { p.get(f); q.get(f + V); }
      if (BACK && on) {
        dp.get(g);
        dq.get(g + V);
        turn<V, true>(g, c, s, a.interleaved);
      }
      if constexpr (NORM) {
        float ss = 0.f, dot = 0.f;
        if (on) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            ss = fmaf(f[j], f[j], ss);
            if (BACK) dot = fmaf(g[j] * w[j], f[j], dot);
          }
        }
        for (int o = a.group >> 1; o; o >>= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, o);
          if (BACK) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        const float r = rsqrtf(fmaf(ss, inv_d, a.eps));
        if (on) {
          if (BACK) {
            const float k = r * r * dot * inv_d;
            if (which) {
#pragma unroll
              for (int j = 0; j < 2 * V; ++j) dw[1][j] = fmaf(g[j], f[j] * r, dw[1][j]);
            } else {
#pragma unroll
              for (int j = 0; j < 2 * V; ++j) dw[0][j] = fmaf(g[j], f[j] * r, dw[0][j]);
            }
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) f[j] = r * (g[j] * w[j] - f[j] * k);
          } else {
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) f[j] = f[j] * r * w[j];
          }
        }
      } else if (BACK) {
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) f[j] = g[j];
      }
      if (!BACK) turn<V, false>(f, c, s, a.interleaved);
      if (on) {
        p.set(f);
        q.set(f + V);
        p.store(y + e0);
        q.store(y + e1);
      }
    }
  }
  if constexpr (BACK && NORM) {
    if (!a.part) return;
    // the groups of a warp, then the warps in order
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) {
        float v = dw[k][j];
        for (int o = a.group; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (live && mine == 0) sums[(warp * 2 + k) * a.D + (j < V ? e0 + j : e1 + j - V)] = v;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += kThreads) {
      float v = 0.f;
      for (int w = 0; w < kWarps; ++w) v += sums[w * 2 * a.D + i];
      a.part[(long long)blockIdx.x * 2 * a.D + i] = v;
    }
  }
}

// dw[which][e] = the CTAs' sums, in their order (eight warps take every eighth, 32 elements a CTA)
__global__ void __launch_bounds__(256) rope_weight_grad(const float* part, int ctas, int D, void* dq, void* dk, int dtype) {
  __shared__ float sm[8][32];
  dependent_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (e < 2 * D)
    for (int c = warp; c < ctas; c += 8) v += part[(long long)c * 2 * D + e];
  sm[warp][lane] = v;
  __syncthreads();
  if (warp || e >= 2 * D) return;
  for (int w = 1; w < 8; ++w) v += sm[w][lane];
  void* out = e < D ? dq : dk;
  const int i = e < D ? e : e - D;
  if (!out) return;
  if (dtype == CHB_F32) static_cast<float*>(out)[i] = v;
  else if (dtype == CHB_BF16) static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16(v);
  else static_cast<__half*>(out)[i] = __float2half(v);
}

template <typename T, int V>
cudaError_t launch(const RopeArgs& a, const Turns& t, bool back, int ctas, cudaStream_t s) {
  const dim3 g((unsigned)ctas), b(kThreads);
  if (a.w[0]) return back ? launch_overlapped(rope_kernel<T, V, true, true>, g, b, s, a, t) : launch_overlapped(rope_kernel<T, V, true, false>, g, b, s, a, t);
  return back ? launch_overlapped(rope_kernel<T, V, false, true>, g, b, s, a, t) : launch_overlapped(rope_kernel<T, V, false, false>, g, b, s, a, t);
}

int warps_and_ctas(RopeArgs* a, int sms) {
  const int per = 32 / a->group;
  a->iters[0] = (a->heads[0] + per - 1) / per;
  a->iters[1] = (a->heads[1] + per - 1) / per;
  // a token's heads are shared out where the tokens alone would not give every SM sixteen warps
  const int total = a->iters[0] + a->iters[1];
  long long slices = (16ll * sms + a->T - 1) / a->T;
  a->slices = (int)(slices < 1 ? 1 : slices > total ? total : slices);
  const long long ctas = ((long long)a->T * a->slices + kWarps - 1) / kWarps;
  return (int)(ctas < 4ll * sms ? ctas : 4ll * sms);
}

}  // namespace
}  // namespace chb

using namespace chb;

extern "C" {

// Most CTAs of a launch on the current device (the partial sums of the backward pass: that many times 2 D floats).
int chb_head_rope_ctas(int* out) {
  int dev = 0, sms = 0;
  if (!out) return CHB_ERR_ARG;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return CHB_ERR_CUDA;
  *out = 4 * sms;
  return CHB_SUCCESS;
}

// x[2], dy[2], y[2]: queries and keys; strides[8]: token and head stride of x[0], x[1], dy[0], dy[1], in elements, multiples of
// 16 bytes.  dy null: forward.  w null: no norm.  part: chb_head_rope_ctas() * 2 * D floats, or null where dw is not wanted.
int chb_head_rope(int dtype, const void* const* x, const void* const* dy, void* const* y, const long long* strides, long long T,
                  int heads_q, int heads_k, int D, const void* const* w, int w_dtype, const void* pos, int pos64, float eps,
                  double base, int interleaved, float* part, void* const* dw, cudaStream_t stream) {
  if (!x || !y || !strides || T < 1 || T >= (1ll << 31) || heads_q < 1 || heads_k < 1 || D < 8 || D % 8 || D > 2 * kMaxPairs) return CHB_ERR_ARG;
  if ((dtype != CHB_F32 && dtype != CHB_BF16 && dtype != CHB_F16) || !(base > 0.0)) return CHB_ERR_ARG;
  if (w && w_dtype != dtype && w_dtype != CHB_F32) return CHB_ERR_ARG;
  const bool half = dtype != CHB_F32;
  const int V = half && D % 16 == 0 ? 8 : 4, size = half ? 2 : 4;
  RopeArgs a{};
  uintptr_t low = 0;
  for (int i = 0; i < 2; ++i) {
    a.x[i] = x[i];
    a.dy[i] = dy ? dy[i] : nullptr;
    a.y[i] = y[i];
    a.xt[i] = strides[2 * i];
    a.xh[i] = strides[2 * i + 1];
    a.dt[i] = strides[4 + 2 * i];
    a.dh[i] = strides[4 + 2 * i + 1];
    a.w[i] = w ? w[i] : nullptr;
    if (!y[i] || (!dy && !x[i]) || (dy && !dy[i]) || (w && (!w[i] || !x[i]))) return CHB_ERR_ARG;
    low |= reinterpret_cast<uintptr_t>(x[i]) | reinterpret_cast<uintptr_t>(a.dy[i]) | reinterpret_cast<uintptr_t>(y[i]) | reinterpret_cast<uintptr_t>(a.w[i]);
    low |= (uintptr_t)((a.xt[i] | a.xh[i] | (dy ? a.dt[i] | a.dh[i] : 0)) * size);
  }
  if (low & 15u) return CHB_ERR_ARG;
  a.heads[0] = heads_q;
  a.heads[1] = heads_k;
  a.w_f32 = half && w && w_dtype == CHB_F32;
  a.pos = pos;
  a.pos64 = pos64;
  a.T = (int)T;
  a.D = D;
  a.lanes = D / (2 * V);
  a.group = 1;
  while (a.group < a.lanes) a.group *= 2;
  a.interleaved = interleaved != 0;
  a.eps = eps;
  a.part = dy && w ? part : nullptr;
  Turns t{};
  for (int i = 0; i < D / 2; ++i) {
    const long double f = powl((long double)base, -2.0L * i / D) / 6.283185307179586476925286766559L;
    t.f[i] = (unsigned long long)ldexpl(f - floorl(f), 64);
  }
  int sms = 0;
  if (chb_head_rope_ctas(&sms) != CHB_SUCCESS) return CHB_ERR_CUDA;
  const int ctas = warps_and_ctas(&a, sms / 4);
  const bool back = dy != nullptr;
  const cudaError_t e = dtype == CHB_F32 ? launch<float, 4>(a, t, back, ctas, stream)
                        : dtype == CHB_BF16 ? (V == 8 ? launch<__nv_bfloat16, 8>(a, t, back, ctas, stream) : launch<__nv_bfloat16, 4>(a, t, back, ctas, stream))
                                            : (V == 8 ? launch<__half, 8>(a, t, back, ctas, stream) : launch<__half, 4>(a, t, back, ctas, stream));
  if (e != cudaSuccess) return CHB_ERR_CUDA;
  if (a.part && dw && launch_overlapped(rope_weight_grad, dim3((unsigned)((2 * D + 31) / 32)), dim3(256), stream, (const float*)part, ctas, D,
                                        dw[0], dw[1], w_dtype) != cudaSuccess) return CHB_ERR_CUDA;
  return CHB_SUCCESS;
}

}  // extern "C"

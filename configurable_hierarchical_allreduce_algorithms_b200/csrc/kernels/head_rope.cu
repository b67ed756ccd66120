// Norm of every query and key head and the rotation of its pairs by the token's position, in one pass, and its gradient.
//
//   y = x / sqrt(mean(x^2) + eps) * w;   (y_a, y_b) -> (y_a cos t - y_b sin t, y_a sin t + y_b cos t),  t = pos base^(-2i/D)
//   backward: u = the gradient turned back by t;  dw = sum u x r;  dx = r (u w - x r^2 mean(u w x)),  r = 1/sqrt(...)
//
// Bound by HBM: every element is read once and written once.  A group of lanes holds one head, each lane two vectors
// of its pairs, so norm, rotation and both sums stay in registers; a warp keeps the sines of its token for all its heads and
// has the next heads' loads in flight while it works on these (the compiler may not move them ahead of the stores itself).
// 8192 tokens, 16 + 16 heads of 128, bf16: forward 33 us (134 MB, 4.1 TB/s), backward with dw 47 us (201 MB, 4.3 TB/s); latency
// and the registers that the loads ahead take are what is between that and a copy's 6.5 TB/s.
// A CTA has queries or keys only, so that a thread sums one weight's gradient.
// Angles: base^(-2i/D) / 2 pi is a 64-bit fraction of a turn, and position times fraction wraps modulo one turn exactly; only the
// angle within the turn is rounded to fp32.  The fraction is cut at 2^-64, so positions up to about 2^38 are as exact as near ones;
// each doubling beyond costs a bit.
#include <math.h>

#include <mutex>

#include "../api/chb.h"
#include "common.cuh"
#include "tc.cuh"

namespace chb {
namespace {

constexpr int kMaxPairs = 128;      // D <= 256
constexpr int kThreads = 256, kWarps = kThreads / 32;

struct RopeSide {            // queries or keys
  const void* x;
  const void* dy;            // backward: gradient of the output
  void* y;                   // output, or gradient of x (contiguous)
  long long xt, xh, dt, dh;  // strides of a token and of a head, in elements
  const void* w;             // null: no norm
  int heads, slices;         // slices: shares of a token's heads, each a warp's
};
struct RopeArgs {
  RopeSide side[2];
  int w_f32;
  const void* pos;           // null: 0, 1, 2, ...
  int pos64;
  int T, D, lanes, group;    // lanes of a head, and the power of two that holds them
  int turns_each;
  float eps;
  float* part;               // backward: sums of dw of each CTA, [CTA][D]
};
struct Turns { unsigned long long f[kMaxPairs]; };

// V neighbouring elements (8 or 16 bytes of 16-bit elements, 16 bytes of fp32)
template <typename T, int V> struct Vec {
  static constexpr int kWords = V * sizeof(T) / 4;
  uint32_t r[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords == 4) {
      const uint4 a = __ldcg(reinterpret_cast<const uint4*>(p));
      r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
    } else {
      const uint2 a = __ldcg(reinterpret_cast<const uint2*>(p));
      r[0] = a.x; r[1] = a.y;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kWords == 4) *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
  }
};

// A lane's V pairs as fp32, first and second members apart, two to a 64-bit register pair (packed arithmetic).  Interleaved
// heads: the lane has 2 V neighbours, pairs (2i, 2i + 1); else V neighbours of the head's first half and as many of its second.
template <int V> struct Pairs {
  uint64_t x[V / 2], y[V / 2];
};
template <typename T, int V, bool INTER>
__device__ __forceinline__ void unpack(const Vec<T, V>& p, const Vec<T, V>& q, Pairs<V>& f) {
  float e[2 * V];
#pragma unroll
  for (int i = 0; i < Vec<T, V>::kWords; ++i) {
    if constexpr (sizeof(T) == 4) {
      e[i] = __uint_as_float(p.r[i]);
      e[V + i] = __uint_as_float(q.r[i]);
    } else {
      const float2 a = tc::unpack2<T>(p.r[i]), b = tc::unpack2<T>(q.r[i]);
      e[2 * i] = a.x; e[2 * i + 1] = a.y;
      e[V + 2 * i] = b.x; e[V + 2 * i + 1] = b.y;
    }
  }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    f.x[i] = INTER ? tc::pair(e[4 * i], e[4 * i + 2]) : tc::pair(e[2 * i], e[2 * i + 1]);
    f.y[i] = INTER ? tc::pair(e[4 * i + 1], e[4 * i + 3]) : tc::pair(e[V + 2 * i], e[V + 2 * i + 1]);
  }
}
template <typename T, int V, bool INTER>
__device__ __forceinline__ void pack(const Pairs<V>& f, Vec<T, V>& p, Vec<T, V>& q) {
  float e[2 * V];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 a = tc::unpair(f.x[i]), b = tc::unpair(f.y[i]);
    if (INTER) {
      e[4 * i] = a.x; e[4 * i + 1] = b.x; e[4 * i + 2] = a.y; e[4 * i + 3] = b.y;
    } else {
      e[2 * i] = a.x; e[2 * i + 1] = a.y; e[V + 2 * i] = b.x; e[V + 2 * i + 1] = b.y;
    }
  }
#pragma unroll
  for (int i = 0; i < Vec<T, V>::kWords; ++i) {
    if constexpr (sizeof(T) == 4) {
      p.r[i] = __float_as_uint(e[i]);
      q.r[i] = __float_as_uint(e[V + i]);
    } else {
      p.r[i] = tc::pack2<T>(e[2 * i], e[2 * i + 1]);
      q.r[i] = tc::pack2<T>(e[V + 2 * i], e[V + 2 * i + 1]);
    }
  }
}

template <typename T, int V, bool INTER>
__device__ __forceinline__ void load_weights(const void* from, bool f32, int e0, int e1, Pairs<V>& w) {
  if (f32) {
    Vec<float, 4> a[V / 4], b[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      a[i].load(reinterpret_cast<const float*>(from) + e0 + 4 * i);
      b[i].load(reinterpret_cast<const float*>(from) + e1 + 4 * i);
    }
    float e[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      e[i] = __uint_as_float(a[i / 4].r[i % 4]);
      e[V + i] = __uint_as_float(b[i / 4].r[i % 4]);
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      w.x[i] = INTER ? tc::pair(e[4 * i], e[4 * i + 2]) : tc::pair(e[2 * i], e[2 * i + 1]);
      w.y[i] = INTER ? tc::pair(e[4 * i + 1], e[4 * i + 3]) : tc::pair(e[V + 2 * i], e[V + 2 * i + 1]);
    }
  } else {
    Vec<T, V> p, q;
    p.load(reinterpret_cast<const T*>(from) + e0);
    q.load(reinterpret_cast<const T*>(from) + e1);
    unpack<T, V, INTER>(p, q, w);
  }
}

// Sine and cosine of a fraction of a turn.  fp32 heads get them correctly to a unit or two; 16-bit ones from the special
// function unit, whose 2^-21 is far below their own rounding (a tenth of the instructions).
template <typename T>
__device__ __forceinline__ void sincos_turn(unsigned long long phase, float* s, float* c) {
  const float half_turns = (float)(int)(phase >> 32) * 4.656612873077392578125e-10f;      // (2^-31)
  if constexpr (sizeof(T) == 4) {
    sincospif(half_turns, s, c);
  } else {
    const float a = half_turns * 3.14159265358979f;
    *s = __sinf(a);
    *c = __cosf(a);
  }
}

// Warp: a token and a share of its heads (blockIdx.y: which, first the queries' shares, then the keys'), `turns_each` turns of
// as many heads as a warp holds.  The loads of the next turn are in flight while one is worked on, those of the first ahead of
// the position's sines.  Forward: one token a warp.  Backward: a warp walks tokens, as its sums of dw stay in registers.
template <typename T, int V, bool NORM, bool BACK, bool INTER>
__global__ void __launch_bounds__(kThreads, BACK ? 2 : 3) rope_kernel(const RopeArgs a, const Turns turns) {
  __shared__ float sums[BACK && NORM ? kWarps * 256 : 1];
  using namespace tc;
  dependent_launch();
  const int which = (int)blockIdx.y >= a.side[0].slices;
  const RopeSide& sd = a.side[which];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & (a.group - 1), per = 32 / a.group, heads = sd.heads, D = a.D;
  const bool live = sub < a.lanes;
  const int first = ((int)blockIdx.y - (which ? a.side[0].slices : 0)) * a.turns_each * per + lane / a.group;
  const int e0 = INTER ? sub * 2 * V : sub * V, e1 = INTER ? e0 + V : D / 2 + sub * V;
  const float inv_d = 1.f / (float)D;
  Pairs<V> w, dw;
  if constexpr (BACK && NORM) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) dw.x[i] = dw.y[i] = 0ull;
  }
  const int stride = (int)gridDim.x * kWarps;
  for (int t = (int)blockIdx.x * kWarps + warp; t < a.T; t = BACK && t < a.T - stride ? t + stride : a.T) {
    const long long pos = !a.pos ? t : a.pos64 ? reinterpret_cast<const long long*>(a.pos)[t] : (long long)reinterpret_cast<const int*>(a.pos)[t];
    const T* x = reinterpret_cast<const T*>(sd.x) + t * sd.xt;
    const T* d = reinterpret_cast<const T*>(sd.dy) + t * sd.dt;
    T* y = reinterpret_cast<T*>(sd.y) + (long long)t * heads * D;
    Vec<T, V> nx[2], nd[2];
    const auto fetch = [&](int head) {
      if (!live || head >= heads) return;
      if constexpr (NORM || !BACK) {
        nx[0].load(x + head * sd.xh + e0);
        nx[1].load(x + head * sd.xh + e1);
      }
      if constexpr (BACK) {
        nd[0].load(d + head * sd.dh + e0);
        nd[1].load(d + head * sd.dh + e1);
      }
    };
    fetch(first);
    if constexpr (NORM) {
      // (read again for every token: the registers are worth more)
      if (live) load_weights<T, V, INTER>(sd.w, a.w_f32, e0, e1, w);
    }
    uint64_t c[V / 2], s[V / 2], ns[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float sn[2], cs[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) sincos_turn<T>((unsigned long long)pos * turns.f[live ? sub * V + 2 * i + j : 0], &sn[j], &cs[j]);
      c[i] = pair(cs[0], cs[1]);
      s[i] = BACK ? pair(-sn[0], -sn[1]) : pair(sn[0], sn[1]);
      ns[i] = BACK ? pair(sn[0], sn[1]) : pair(-sn[0], -sn[1]);
    }
    const auto turn = [&](Pairs<V>& f) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const uint64_t u = fma2(f.x[i], c[i], mul2(f.y[i], ns[i]));
        f.y[i] = fma2(f.x[i], s[i], mul2(f.y[i], c[i]));
        f.x[i] = u;
      }
    };
#pragma unroll 1
    for (int k = 0, head = first; k < a.turns_each; ++k, head += per) {
      const bool on = live && head < heads;
      Pairs<V> f, g;
      if constexpr (NORM || !BACK) unpack<T, V, INTER>(nx[0], nx[1], f);
      if constexpr (BACK) {
        unpack<T, V, INTER>(nd[0], nd[1], g);
        turn(g);
      }
      if (k + 1 < a.turns_each) fetch(head + per);
      if constexpr (NORM) {
        uint64_t ss2 = 0ull, dot2 = 0ull;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          ss2 = fma2(f.x[i], f.x[i], fma2(f.y[i], f.y[i], ss2));
          if constexpr (BACK) dot2 = fma2(mul2(g.x[i], w.x[i]), f.x[i], fma2(mul2(g.y[i], w.y[i]), f.y[i], dot2));
        }
        const float2 sp = unpair(ss2), dp = unpair(dot2);
        float ss = on ? sp.x + sp.y : 0.f, dot = on && BACK ? dp.x + dp.y : 0.f;      // (lanes without elements)
        for (int o = a.group >> 1; o; o >>= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, o);
          if (BACK) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        const float r = rsqrtf(fmaf(ss, inv_d, a.eps));
        const uint64_t r2 = pair(r, r);
        if constexpr (BACK) {
          const float q = -r * (r * r * dot * inv_d);
          const uint64_t q2 = pair(q, q);
          if (on) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              dw.x[i] = fma2(g.x[i], mul2(f.x[i], r2), dw.x[i]);
              dw.y[i] = fma2(g.y[i], mul2(f.y[i], r2), dw.y[i]);
              f.x[i] = fma2(f.x[i], q2, mul2(mul2(g.x[i], w.x[i]), r2));
              f.y[i] = fma2(f.y[i], q2, mul2(mul2(g.y[i], w.y[i]), r2));
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            f.x[i] = mul2(mul2(f.x[i], r2), w.x[i]);
            f.y[i] = mul2(mul2(f.y[i], r2), w.y[i]);
          }
        }
      }
      if constexpr (!BACK) turn(f);
      if (on) {
        Vec<T, V> p, q;
        if constexpr (BACK && !NORM) pack<T, V, INTER>(g, p, q);
        else pack<T, V, INTER>(f, p, q);
        p.store(y + head * D + e0);
        q.store(y + head * D + e1);
      }
    }
  }
  if constexpr (BACK && NORM) {
    if (!a.part) return;
    // the groups of a warp, then the warps in order
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) {
      const int i = j % V;
      const float2 v2 = unpair(j < V ? dw.x[i / 2] : dw.y[i / 2]);
      float v = i & 1 ? v2.y : v2.x;
      for (int o = a.group; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      const int e = INTER ? 2 * (sub * V + i) + (j >= V) : sub * V + i + (j >= V ? D / 2 : 0);
      if (live && lane < a.group) sums[warp * D + e] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kThreads) {
      float v = 0.f;
      for (int k = 0; k < kWarps; ++k) v += sums[k * D + i];
      a.part[((long long)blockIdx.y * gridDim.x + blockIdx.x) * D + i] = v;
    }
  }
}

// dw = the CTAs' sums, in their order (eight warps take every eighth, 32 elements a CTA; y: queries or keys)
__global__ void __launch_bounds__(256) rope_weight_grad(const float* part, int ctas_q, int ctas_k, int D, void* dq, void* dk, int dtype) {
  __shared__ float sm[8][32];
  dependent_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  const int c0 = blockIdx.y ? ctas_q : 0, c1 = blockIdx.y ? ctas_q + ctas_k : ctas_q;
  float v = 0.f;
  if (e < D) {
#pragma unroll 8
    for (int c = c0 + warp; c < c1; c += 8) v += part[(long long)c * D + e];
  }
  sm[warp][lane] = v;
  __syncthreads();
  void* out = blockIdx.y ? dk : dq;
  if (warp || e >= D || !out) return;
  for (int k = 1; k < 8; ++k) v += sm[k][lane];
  if (dtype == CHB_F32) static_cast<float*>(out)[e] = v;
  else if (dtype == CHB_BF16) static_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16(v);
  else static_cast<__half*>(out)[e] = __float2half(v);
}

// Backward launches have two CTAs an SM (as many as fit) in all, or one for every share of a token's heads if those are more.
int tokens_across(const RopeArgs& a, int sms) {
  const int all = a.side[0].slices + a.side[1].slices, ctas = (a.T + kWarps - 1) / kWarps;
  const int most = 2 * sms / all < 1 ? 1 : 2 * sms / all;
  return ctas < most ? ctas : most;
}

// A warp takes four turns (for as many, a token's sines cost little), fewer where the tokens alone would not give every SM
// sixteen warps.
void share_out(RopeArgs* a, int sms) {
  const int per = 32 / a->group;
  const int iq = (a->side[0].heads + per - 1) / per, ik = (a->side[1].heads + per - 1) / per;
  a->turns_each = 4;
  while (a->turns_each > 1 && (long long)a->T * ((iq + a->turns_each - 1) / a->turns_each + (ik + a->turns_each - 1) / a->turns_each) < 16ll * sms) --a->turns_each;
  a->side[0].slices = (iq + a->turns_each - 1) / a->turns_each;
  a->side[1].slices = (ik + a->turns_each - 1) / a->turns_each;
}

template <typename T, int V, bool INTER>
cudaError_t launch_order(const RopeArgs& a, const Turns& t, bool back, int sms, cudaStream_t s) {
  const dim3 g((unsigned)(back ? tokens_across(a, sms) : (a.T + kWarps - 1) / kWarps), (unsigned)(a.side[0].slices + a.side[1].slices)), b(kThreads);
  if (a.side[0].w) return back ? launch_overlapped(rope_kernel<T, V, true, true, INTER>, g, b, s, a, t) : launch_overlapped(rope_kernel<T, V, true, false, INTER>, g, b, s, a, t);
  return back ? launch_overlapped(rope_kernel<T, V, false, true, INTER>, g, b, s, a, t) : launch_overlapped(rope_kernel<T, V, false, false, INTER>, g, b, s, a, t);
}
template <typename T, int V>
cudaError_t launch(const RopeArgs& a, const Turns& t, bool interleaved, bool back, int sms, cudaStream_t s) {
  return interleaved ? launch_order<T, V, true>(a, t, back, sms, s) : launch_order<T, V, false>(a, t, back, sms, s);
}

// The fractions of a turn for one base and D, kept from call to call (as a program keeps its tables): the last eight that were
// made, as a base may change with every call.  A copy, as the entry may be overwritten by the next call.
Turns turns_of(double base, int D) {
  constexpr unsigned kKept = 8;
  struct Entry { double base; int D; Turns t; };
  static std::mutex mu;
  static Entry known[kKept];
  static unsigned made = 0;
  std::lock_guard<std::mutex> g(mu);
  for (unsigned i = 0; i < kKept && i < made; ++i)
    if (known[i].base == base && known[i].D == D) return known[i].t;
  Entry& e = known[made % kKept];
  made = made + 1 < 2 * kKept ? made + 1 : kKept;      // (a number of the same remainder: it never wraps)
  e.base = base;
  e.D = D;
  for (int i = 0; i < D / 2; ++i) {
    const long double f = powl((long double)base, -2.0L * i / D) / 6.283185307179586476925286766559L;
    e.t.f[i] = (unsigned long long)ldexpl(f - floorl(f), 64);
  }
  return e.t;
}

}  // namespace
}  // namespace chb

using namespace chb;

extern "C" {

// Most rows of partial sums of a backward launch on the current device (of D floats each).
int chb_head_rope_rows(int heads_q, int heads_k, int* out) {
  const int sms = tc::sm_count();
  if (!out || heads_q < 1 || heads_k < 1) return CHB_ERR_ARG;
  if (!sms) return CHB_ERR_CUDA;
  // (a share is a head at least, so there are no more shares than heads)
  *out = 2 * sms > heads_q + heads_k ? 2 * sms : heads_q + heads_k;
  return CHB_SUCCESS;
}

// x[2], dy[2], y[2]: queries and keys; strides[8]: token and head stride of x[0], x[1], dy[0], dy[1], in elements, multiples of
// 16 bytes.  dy null: forward.  w null: no norm.  part: chb_head_rope_rows() * D floats, or null where dw is not wanted.
int chb_head_rope(int dtype, const void* const* x, const void* const* dy, void* const* y, const long long* strides, long long T,
                  int heads_q, int heads_k, int D, const void* const* w, int w_dtype, const void* pos, int pos64, float eps,
                  double base, int interleaved, float* part, void* const* dw, cudaStream_t stream) try {
  if (!x || !y || !strides || T < 1 || T >= (1ll << 31) || heads_q < 1 || heads_k < 1 || D < 8 || D % 8 || D > 2 * kMaxPairs) return CHB_ERR_ARG;
  if ((dtype != CHB_F32 && dtype != CHB_BF16 && dtype != CHB_F16) || !(base > 0.0)) return CHB_ERR_ARG;
  if (w && w_dtype != dtype && w_dtype != CHB_F32) return CHB_ERR_ARG;
  const bool half = dtype != CHB_F32;
  const int V = half && D % 16 == 0 ? 8 : 4, size = half ? 2 : 4;
  RopeArgs a{};
  uintptr_t low = 0;
  for (int i = 0; i < 2; ++i) {
    RopeSide& d = a.side[i];
    d.x = x[i];
    d.dy = dy ? dy[i] : nullptr;
    d.y = y[i];
    d.xt = strides[2 * i];
    d.xh = strides[2 * i + 1];
    d.dt = strides[4 + 2 * i];
    d.dh = strides[4 + 2 * i + 1];
    d.w = w ? w[i] : nullptr;
    d.heads = i ? heads_k : heads_q;
    if (!y[i] || (!dy && !x[i]) || (dy && !dy[i]) || (w && (!w[i] || !x[i]))) return CHB_ERR_ARG;
    low |= reinterpret_cast<uintptr_t>(x[i]) | reinterpret_cast<uintptr_t>(d.dy) | reinterpret_cast<uintptr_t>(y[i]) | reinterpret_cast<uintptr_t>(d.w);
    low |= (uintptr_t)((d.xt | d.xh | (dy ? d.dt | d.dh : 0)) * size);
  }
  if (low & 15u) return CHB_ERR_ARG;
  if (!tc::on_boundary(pos64 ? 8 : 4, static_cast<const char*>(pos)) || !tc::on_boundary(4, part)) return CHB_ERR_ARG;
  if (dw && !tc::on_boundary(w_dtype == CHB_F32 ? 4 : 2, static_cast<const char*>(dw[0]), static_cast<const char*>(dw[1]))) return CHB_ERR_ARG;
  a.w_f32 = half && w && w_dtype == CHB_F32;
  a.pos = pos;
  a.pos64 = pos64;
  a.T = (int)T;
  a.D = D;
  a.lanes = D / (2 * V);
  a.group = 1;
  while (a.group < a.lanes) a.group *= 2;
  a.eps = eps;
  a.part = dy && w ? part : nullptr;
  const int sms = tc::sm_count();
  if (!sms) return CHB_ERR_CUDA;
  const bool back = dy != nullptr, in = interleaved != 0;
  share_out(&a, sms);
  const int shares = a.side[0].slices + a.side[1].slices;
  if (shares > 65535) return CHB_ERR_UNSUPPORTED;
  const Turns t = turns_of(base, D);
  const cudaError_t e = dtype == CHB_F32 ? launch<float, 4>(a, t, in, back, sms, stream)
                        : dtype == CHB_BF16 ? (V == 8 ? launch<__nv_bfloat16, 8>(a, t, in, back, sms, stream) : launch<__nv_bfloat16, 4>(a, t, in, back, sms, stream))
                                            : (V == 8 ? launch<__half, 8>(a, t, in, back, sms, stream) : launch<__half, 4>(a, t, in, back, sms, stream));
  if (e != cudaSuccess) return CHB_ERR_CUDA;
  if (a.part && dw) {
    const int across = tokens_across(a, sms);
    if (launch_overlapped(rope_weight_grad, dim3((unsigned)((D + 31) / 32), 2), dim3(256), stream, (const float*)part, across * a.side[0].slices,
                          across * a.side[1].slices, D, dw[0], dw[1], w_dtype) != cudaSuccess) return CHB_ERR_CUDA;
  }
  return CHB_SUCCESS;
} catch (...) {
  return CHB_ERR_OTHER;      // (the lock of the table of angles)
}

}  // extern "C"

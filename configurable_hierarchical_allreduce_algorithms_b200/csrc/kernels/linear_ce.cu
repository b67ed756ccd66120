// Softmax cross entropy of a linear output layer, logits = x W^T, without the logits: they exist as accumulators of one
// tile at a time, and for the gradient as one piece of the vocabulary in 16 bits.
//
//   loss_r = log sum_v exp(l_rv) - l_r,t(r)          G_rv = (exp(l_rv - lse_r) - [v = t(r)]) g_r
//   dx = G W                                          dW = G^T x
//
// Forward: rows with a label are gathered (a row without one costs nothing, and whatever its x holds, infinities
// included, reaches neither the loss nor dW); one product whose epilogue keeps maximum and sum of exponentials of 256
// columns; a small kernel joins them.  Backward, for each piece of the vocabulary: the product again with an epilogue
// that writes G, then dW (complete for the piece) and dx (summed over the pieces in fp32) from G.
//
// Sums are fp32.  G is rounded to the operands' type, as the tensor cores need it; an fp16 G is kept 2^14 times larger
// and relative to the largest |g_r|, or softmax tails would fall below fp16's range.
#include "../api/chb.h"
#include "common.cuh"
#include "tc.cuh"

namespace chb {
namespace {

using namespace tc;

constexpr int BM = 128, BN = 256, BK = 64, kStages = 4;
constexpr int kBox = 64 * 128;                               // bytes of one load: 64 rows of 64 elements
constexpr int kStageBytes = (BM + BN) * BK * 2;
constexpr int kGemmSmem = kStages * kStageBytes + 1024;      // (1024: the swizzle's alignment)
constexpr float kLog2e = 1.4426950408889634f;

enum Mode { LSE, GRAD, DX, DW };

// Kept from forward to backward.
struct Saved {
  int* head;       // [0] rows with a label, [1] CTAs of the joining kernel that are done
  int* idx;        // row of x of every gathered row
  int* pos;        // gathered row of every row of x, -1: none
  int* tgt;        // label of every gathered row, -1: not in the vocabulary
  float* lse2;     // log2 of the sum of exponentials
  char* xc;        // gathered rows
};

struct GemmArgs {
  const int* count;
  int N, V, v0, vn;          // rows of x at most; vocabulary, first column and width of the piece
  int D;
  int K;                     // extent of the summed axis (0: the rows)
  // LSE
  float2* part;
  float* tlogit;
  const int* tgt;
  int rows_pad;
  // GRAD
  const float* lse2;
  const float* gs;
  char* g;
  long long ldg;
  // DX / DW
  float* acc;
  int first, last;
  const float* coef;
  const int* idx;
  char* out;
  unsigned* status;
};

__device__ __forceinline__ void st256(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

template <typename T> struct GScale { static constexpr float up = 1.f, down = 1.f; };
template <> struct GScale<__half> { static constexpr float up = 16384.f, down = 1.f / 16384.f; };

// One persistent CTA per SM; warp 0 loads, warp 1 issues the products, warps 4 to 7 finish a tile (thread = row) while the
// next one is summed in the other half of tensor memory.
template <typename T, int MODE>
__global__ void __launch_bounds__(256, 1)
ce_gemm(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const GemmArgs p) {
  constexpr bool a_mn = MODE == DW, b_mn = MODE == DX || MODE == DW;
  extern __shared__ char smem_raw[];
  __shared__ __align__(8) unsigned long long full_[kStages], empty_[kStages], done_[2], free_[2];
  __shared__ uint32_t tmem_;
  __shared__ Fault fault;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full = smem_u32(full_), empty = smem_u32(empty_), done = smem_u32(done_), free_b = smem_u32(free_);
  if (threadIdx.x == 0) {
    fault.raised = 0;
    fault.status = p.status;
    for (int i = 0; i < kStages; ++i) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { bar_init(done + 8 * i, 1); bar_init(free_b + 8 * i, 128); }
    bar_init_done();
    prefetch_map(&ma);
    prefetch_map(&mb);
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_), 512);
  fence_before();
  __syncthreads();
  fence_after();
  dependent_launch();
  const uint32_t tmem = tmem_;
  const int count = *(volatile const int*)p.count;
  const int mt = MODE == DW ? (p.vn + BM - 1) / BM : (count + BM - 1) / BM;
  const int ncols = MODE == LSE || MODE == GRAD ? p.vn : p.D;
  const int nt = (ncols + BN - 1) / BN;
  const int nk = ((MODE == DW ? count : p.K) + BK - 1) / BK;
  const int tiles = mt * nt;
  // neighbouring CTAs share the operand that is read from HBM: the rows of W (LSE, GRAD) or of G (DX, DW)
  auto m_of = [&](int t) { return MODE == LSE || MODE == GRAD ? t % mt : t / nt; };
  auto n_of = [&](int t) { return MODE == LSE || MODE == GRAD ? t / mt : t % nt; };

  if (warp == 0) {
    const bool one = elect();
    int s = 0;
    unsigned ph = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const int m0 = m_of(t) * BM, n0 = n_of(t) * BN;
      for (int k = 0; k < nk; ++k) {
        if (!(ok = bar_wait_warp(empty + 8 * s, ph ^ 1u, &fault))) break;
        const uint32_t bar = full + 8 * s, a = smem + s * kStageBytes, b = a + BM * BK * 2;
        if (one) {
          bar_expect(bar, kStageBytes);
#pragma unroll
          for (int j = 0; j < BM / 64; ++j) {
            if (a_mn) load2(a + j * kBox, &ma, m0 + 64 * j, k * BK, bar);
            else load2(a + j * kBox, &ma, k * BK, m0 + 64 * j, bar);
          }
#pragma unroll
          for (int j = 0; j < BN / 64; ++j) {
            if (MODE == DX) load2(b + j * kBox, &mb, n0 + 64 * j, p.v0 + k * BK, bar);
            else if (MODE == DW) load2(b + j * kBox, &mb, n0 + 64 * j, k * BK, bar);
            else load2(b + j * kBox, &mb, k * BK, p.v0 + n0 + 64 * j, bar);
          }
        }
        __syncwarp();
        if (++s == kStages) { s = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t desc = product_desc<T>(BM, BN, a_mn, b_mn);
    const bool one = elect();
    int s = 0, buf = 0;
    unsigned ph = 0, bph = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok && nk; t += gridDim.x) {
      if (!(ok = bar_wait_warp(free_b + 8 * buf, bph ^ 1u, &fault))) break;
      fence_after();
      for (int k = 0; k < nk; ++k) {
        if (!(ok = bar_wait_warp(full + 8 * s, ph, &fault))) break;
        fence_after();
        const uint32_t a = smem + s * kStageBytes, b = a + BM * BK * 2;
        const uint64_t da = operand(a, a_mn ? kBox : 16), db = operand(b, b_mn ? kBox : 16);
        if (one) {
#pragma unroll
          for (int i = 0; i < BK / 16; ++i)
            mma_ss(tmem + buf * BN, da + i * (a_mn ? 128 : 2), db + i * (b_mn ? 128 : 2), desc, k > 0 || i > 0);
          commit(empty + 8 * s);
        }
        __syncwarp();
        if (++s == kStages) { s = 0; ph ^= 1u; }
      }
      if (!ok) break;
      if (one) commit(done + 8 * buf);
      __syncwarp();
      if (++buf == 2) { buf = 0; bph ^= 1u; }
    }
  } else if (warp >= 4) {
    int buf = 0;
    unsigned bph = 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      const int m0 = m_of(t) * BM, n0 = n_of(t) * BN;
      const int row = m0 + (warp & 3) * 32 + lane;
      if (nk && !bar_wait_warp(done + 8 * buf, bph, &fault)) break;
      fence_after();
      const uint32_t src = tmem + buf * BN + lanes;
      if (MODE == LSE || MODE == GRAD) {
        const bool in = row < count;
        const int tg = in ? p.tgt[row] - p.v0 - n0 : -1;
        const int cols = min(BN, p.V - p.v0 - n0);
        float m = -INFINITY, sum = 0.f;
        float lse = 0.f, gs = 0.f;
        if (MODE == GRAD && in) { lse = p.lse2[row]; gs = p.gs[row] * GScale<T>::up; }
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          uint32_t r[32];
          __syncwarp();
          ld32(src + c, r);
          wait_ld(r);
          if (MODE == LSE) {
            if (c + 32 > cols) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c + j >= cols) r[j] = __float_as_uint(-INFINITY);
            }
            float cm = m;
#pragma unroll
            for (int j = 0; j < 32; ++j) cm = fmaxf(cm, __uint_as_float(r[j]));
            const float ref = cm == -INFINITY ? 0.f : cm * kLog2e;
            float add = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) add += ex2(fmaf(__uint_as_float(r[j]), kLog2e, -ref));
            sum = fmaf(sum, ex2(fmaf(m, kLog2e, -ref)), add);
            m = cm;
            if ((unsigned)(tg - c) < 32u) {
              float x = 0.f;
#pragma unroll
              for (int j = 0; j < 32; ++j) x = tg - c == j ? __uint_as_float(r[j]) : x;
              p.tlogit[row] = x;
            }
          } else {
            uint32_t o[16];
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = ex2(fmaf(__uint_as_float(r[j]), kLog2e, -lse));
            if ((unsigned)(tg - c) < 32u) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] -= tg - c == j ? 1.f : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= gs;
            if (!in || c + 32 > cols) {      // (selected, not multiplied: these values may be anything)
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = in && c + j < cols ? v[j] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
            char* d = p.g + ((long long)row * p.ldg + n0 + c) * 2;
            st256(d, o);
            st256(d + 32, o + 8);
          }
        }
        if (MODE == LSE && in) p.part[(long long)(n0 / BN) * p.rows_pad + row] = make_float2(m, sum);
      } else {
        const bool in = row < (MODE == DX ? count : min(p.vn, p.V - p.v0));
        const float coef = *p.coef * GScale<T>::down;
        const bool fin = MODE == DW || p.last;
        long long orow = 0;
        if (in) orow = MODE == DX ? (long long)p.idx[row] * p.D : (long long)(p.v0 + row) * p.D;
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          uint32_t r[32];
          __syncwarp();
          ld32(src + c, r);
          wait_ld(r);
          if (!nk) {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0;
          }
          if (!in) continue;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int col = n0 + c + 8 * q;
            if (col >= p.D) break;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[8 * q + j]);
            float4* ac = reinterpret_cast<float4*>(p.acc + (long long)row * p.D + col);
            if (MODE == DX && !p.first) {
              const float4 x = ac[0], y = ac[1];
              v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
              v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
            }
            if (fin) {
              uint4 o;
              o.x = pack2<T>(v[0] * coef, v[1] * coef);
              o.y = pack2<T>(v[2] * coef, v[3] * coef);
              o.z = pack2<T>(v[4] * coef, v[5] * coef);
              o.w = pack2<T>(v[6] * coef, v[7] * coef);
              *reinterpret_cast<uint4*>(p.out + (orow + col) * 2) = o;
            } else {
              ac[0] = make_float4(v[0], v[1], v[2], v[3]);
              ac[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
          }
        }
      }
      fence_before();
      if (nk) bar_arrive(free_b + 8 * buf);
      if (++buf == 2) { buf = 0; bph ^= 1u; }
    }
  }
  __syncthreads();
  if (fault.raised) drain_after_abort();
  __syncthreads();
  if (warp == 1) tmem_free(tmem, 512);
}

// Which rows have a label: positions among them by a scan (one CTA; thread = a run of neighbouring rows).
__global__ void __launch_bounds__(1024) ce_rows(const long long* targets, int N, int V, long long ignore, Saved sv) {
  __shared__ int sums[32];
  dependent_launch();
  const int per = (N + 1023) / 1024, tid = threadIdx.x;
  const int r0 = min(N, tid * per), r1 = min(N, r0 + per);
  int n = 0;
  for (int r = r0; r < r1; ++r) n += targets[r] != ignore;
  int inc = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, d);
    if ((tid & 31) >= d) inc += v;
  }
  if ((tid & 31) == 31) sums[tid >> 5] = inc;
  __syncthreads();
  if (tid < 32) {
    int v = sums[tid];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, d);
      if (tid >= d) v += u;
    }
    sums[tid] = v;
  }
  __syncthreads();
  int at = inc - n + (tid >= 32 ? sums[(tid >> 5) - 1] : 0);
  for (int r = r0; r < r1; ++r) {
    const long long t = targets[r];
    const bool in = t != ignore;
    sv.pos[r] = in ? at : -1;
    if (in) {
      sv.idx[at] = r;
      sv.tgt[at] = t >= 0 && t < V ? (int)t : -1;
      ++at;
    }
  }
  if (tid == 1023) { sv.head[0] = at; sv.head[1] = 0; }
}

// Gathers the rows of x (warp = row of 16-byte words); zeros behind the last one up to a full tile.  Rows without a label
// have a loss of zero.
__global__ void __launch_bounds__(256) ce_gather(const char* x, long long ldx, int N, int D, Saved sv, float* loss_rows) {
  dependent_launch();
  const int words = D / 8, lane = threadIdx.x & 31;
  const int count = *(volatile const int*)sv.head;
  const int pad = min((N + BM - 1) / BM * BM, (count + BM - 1) / BM * BM);
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r < N) {
    const int at = sv.pos[r];
    if (at >= 0) {
      const uint4* s = reinterpret_cast<const uint4*>(x + (long long)r * ldx * 2);
      uint4* d = reinterpret_cast<uint4*>(sv.xc + (long long)at * D * 2);
      for (int i = lane; i < words; i += 32) d[i] = s[i];
    } else if (loss_rows && lane == 0) {
      loss_rows[r] = 0.f;
    }
  }
  if (r >= count && r < pad) {
    uint4* d = reinterpret_cast<uint4*>(sv.xc + (long long)r * D * 2);
    for (int i = lane; i < words; i += 32) d[i] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// Joins the column tiles of 32 rows (lane = row, the eight warps take every eighth tile) and, in the last CTA to come, the
// sum over the rows: CTA sums in the order of the rows, whichever CTA is last.
__global__ void __launch_bounds__(256)
ce_join(const float2* part, const float* tlogit, int nt, int rows_pad, int reduction, Saved sv, double* sums, float* loss) {
  __shared__ float sm[8][32], ss[8][32];
  __shared__ int is_last;
  dependent_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int count = *(volatile const int*)sv.head;
  const int row = blockIdx.x * 32 + lane;
  const bool in = row < count;
  float m = -INFINITY, s = 0.f;
  if (in) {
#pragma unroll 4
    for (int t = warp; t < nt; t += 8) {
      const float2 v = part[(long long)t * rows_pad + row];
      const float nm = fmaxf(m, v.x), ref = nm == -INFINITY ? 0.f : nm;
      s = s * ex2((m - ref) * kLog2e) + v.y * ex2((v.x - ref) * kLog2e);
      m = nm;
    }
  }
  sm[warp][lane] = m;
  ss[warp][lane] = s;
  __syncthreads();
  if (warp == 0) {
    float loss_r = 0.f;
    if (in) {
      float M = m;
#pragma unroll
      for (int w = 1; w < 8; ++w) M = fmaxf(M, sm[w][lane]);
      const float ref = M == -INFINITY ? 0.f : M;
      float S = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) S += ss[w][lane] * ex2((sm[w][lane] - ref) * kLog2e);
      const bool known = sv.tgt[row] >= 0;
      loss_r = known ? logf(S) + (M - tlogit[row]) : __int_as_float(0x7fffffff);      // (no such label: NaN)
      sv.lse2[row] = known ? fmaf(M, kLog2e, log2f(S)) : __int_as_float(0x7fffffff);
      if (reduction == 0) loss[sv.idx[row]] = loss_r;
    }
    if (reduction != 0) {
      double d = loss_r;
#pragma unroll
      for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
      if (lane == 0) sums[blockIdx.x] = d;
    }
  }
  if (reduction == 0) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    is_last = atomicAdd(&sv.head[1], 1) == (int)gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!is_last || warp) return;
  double d = 0.;
  for (int i = lane; i < (int)gridDim.x; i += 32) d += *(volatile double*)(sums + i);
#pragma unroll
  for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if (lane == 0) *loss = (float)(reduction == 1 ? d / count : d);
}

// Before the backward products: every row's weight relative to the largest, that largest, and zeros in dx where a row has
// no label.  Every CTA finds the largest for itself (the gradients of the rows are few bytes and in L2).
__global__ void __launch_bounds__(256)
ce_weights(const float* grad, int reduction, int N, int D, Saved sv, float* gs, float* coef, char* dx) {
  __shared__ float mx[8];
  dependent_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int count = *(volatile const int*)sv.head;
  float top;
  if (reduction == 0) {
    float m = 0.f;
    for (int i = threadIdx.x; i < count; i += 256) {
      const float a = fabsf(grad[sv.idx[i]]);
      m = a > m || !(a == a) ? a : m;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float a = __shfl_xor_sync(0xffffffffu, m, o);
      m = a > m || !(a == a) ? a : m;
    }
    if (lane == 0) mx[warp] = m;
    __syncthreads();
    top = mx[0];
    for (int w = 1; w < 8; ++w) top = mx[w] > top || !(mx[w] == mx[w]) ? mx[w] : top;
  } else {
    top = fabsf(*grad) / (reduction == 1 ? (float)count : 1.f);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *coef = count ? top : 0.f;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256) {
    const float g = reduction == 0 ? grad[sv.idx[i]] / top : *grad < 0.f ? -1.f : 1.f;
    gs[i] = top == 0.f ? 0.f : g;
  }
  if (!dx) return;
  for (int r = blockIdx.x * 8 + warp; r < N; r += gridDim.x * 8) {
    if (sv.pos[r] >= 0) continue;
    uint4* d = reinterpret_cast<uint4*>(dx + (long long)r * D * 2);
    for (int i = lane; i < D / 8; i += 32) d[i] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// ------------------------------------------------------------------ host side
constexpr long long kPieceBytes = 96ll << 20;

long long up(long long v, long long to) { return (v + to - 1) / to * to; }

struct Carve {      // consecutive parts of a workspace, 256-byte aligned
  char* base;
  long long at = 0;
  template <typename P> P* take(long long bytes) {
    P* r = reinterpret_cast<P*>(base ? base + at : nullptr);
    at += up(bytes, 256);
    return r;
  }
};

long long saved_layout(char* base, long long N, int D, Saved* sv) {
  Carve c{base};
  const long long pad = up(N, BM);
  sv->head = c.take<int>(64);
  sv->idx = c.take<int>(pad * 4);
  sv->pos = c.take<int>(pad * 4);
  sv->tgt = c.take<int>(pad * 4);
  sv->lse2 = c.take<float>(pad * 4);
  sv->xc = c.take<char>(pad * D * 2);
  return c.at;
}

struct Fwd { float2* part; float* tlogit; double* sums; };
long long fwd_layout(char* base, long long N, int V, Fwd* w) {
  Carve c{base};
  const long long pad = up(N, BM);
  w->part = c.take<float2>(pad * 8 * ((V + BN - 1) / BN));
  w->tlogit = c.take<float>(pad * 4);
  w->sums = c.take<double>(pad / 32 * 8);
  return c.at;
}

// Width of a piece of the vocabulary: its G takes kPieceBytes at most (it stays in L2 from the kernel that writes it to
// those that read it), and the pieces are even.
int piece_width(long long N, int V) {
  const long long pad = up(N, BM), most = kPieceBytes / (pad * 2) / BN * BN;
  const long long one = most < BN ? BN : most;
  const long long pieces = (V + one - 1) / one;
  return (int)up((V + pieces - 1) / pieces, BN);
}

struct Bwd { float* gs; float* coef; float* acc; char* g; };
long long bwd_layout(char* base, long long N, int D, int V, Bwd* w) {
  Carve c{base};
  const long long pad = up(N, BM);
  w->gs = c.take<float>(pad * 4);
  w->coef = c.take<float>(4);
  w->acc = c.take<float>(pad * D * 4);
  w->g = c.take<char>(pad * piece_width(N, V) * 2);
  return c.at;
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

template <typename T, int MODE>
cudaError_t gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmArgs& p, long long tiles, int sms, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(ce_gemm<T, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)(tiles < sms ? tiles : sms));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = kGemmSmem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, ce_gemm<T, MODE>, a, b, p);
}

bool map2(CUtensorMap* m, int dtype, const void* base, long long inner, long long rows, long long ld) {
  const unsigned long long d[2] = {(unsigned long long)inner, (unsigned long long)rows}, s[1] = {(unsigned long long)ld};
  return make_map(m, dtype, base, 2, d, s, 64);
}

bool sizes_ok(int dtype, long long N, int D, int V, int reduction) {
  return (dtype == CHB_BF16 || dtype == CHB_F16) && N >= 1 && N < (1ll << 31) - 256 && D >= 8 && D % 8 == 0 && V >= 1 &&
         V < (1 << 30) && reduction >= 0 && reduction <= 2;
}

template <typename T>
int backward(int dtype, const char* w, int N, int D, int V, const Saved& sv, const Bwd& b, char* dx, char* dw, int sms,
             cudaStream_t stream) {
  const long long pad = up(N, BM);
  const int width = piece_width(N, V);
  CUtensorMap mx, mw, mg;
  if (!map2(&mx, dtype, sv.xc, D, pad, D) || !map2(&mw, dtype, w, D, V, D) || !map2(&mg, dtype, b.g, width, pad, width)) return CHB_ERR_CUDA;
  GemmArgs p{};
  p.count = sv.head;
  p.N = N; p.V = V; p.D = D;
  p.tgt = sv.tgt; p.lse2 = sv.lse2; p.gs = b.gs; p.g = b.g; p.ldg = width;
  p.acc = b.acc; p.coef = b.coef; p.idx = sv.idx;
  p.status = status_word();
  if (!p.status) return CHB_ERR_CUDA;
  const long long mt = pad / BM, dt = (D + BN - 1) / BN;
  for (int v0 = 0; v0 < V; v0 += width) {
    p.v0 = v0;
    p.vn = V - v0 < width ? V - v0 : width;
    p.first = v0 == 0;
    p.last = v0 + width >= V;
    p.K = D;
    if (gemm<T, GRAD>(mx, mw, p, mt * ((p.vn + BN - 1) / BN), sms, stream) != cudaSuccess) return CHB_ERR_CUDA;
    if (dw) {
      p.out = dw;
      if (gemm<T, DW>(mg, mx, p, (p.vn + BM - 1) / BM * dt, sms, stream) != cudaSuccess) return CHB_ERR_CUDA;
    }
    if (dx) {
      p.out = dx;
      p.K = p.vn;
      if (gemm<T, DX>(mg, mw, p, mt * dt, sms, stream) != cudaSuccess) return CHB_ERR_CUDA;
    }
  }
  return CHB_SUCCESS;
}

}  // namespace
}  // namespace chb

using namespace chb;

extern "C" {

int chb_linear_ce_bytes(long long N, int D, int V, long long* saved, long long* forward, long long* backward) {
  if (!sizes_ok(CHB_BF16, N, D, V, 0) || !saved || !forward || !backward) return CHB_ERR_ARG;
  Saved sv;
  Fwd f;
  Bwd b;
  *saved = saved_layout(nullptr, N, D, &sv);
  *forward = fwd_layout(nullptr, N, V, &f);
  *backward = bwd_layout(nullptr, N, D, V, &b);
  return CHB_SUCCESS;
}

int chb_linear_ce_forward(int dtype, const void* x, long long ldx, const void* w, const long long* targets, long long N, int D,
                          int V, long long ignore_index, int reduction, float* loss, void* saved, void* work, cudaStream_t stream) {
  if (!sizes_ok(dtype, N, D, V, reduction) || !x || !w || !targets || !loss || !saved || !work || ldx % 8) return CHB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15u) return CHB_ERR_ARG;
  Saved sv;
  Fwd f;
  saved_layout(static_cast<char*>(saved), N, D, &sv);
  fwd_layout(static_cast<char*>(work), N, V, &f);
  const long long pad = up(N, BM);
  const int sms = sm_count(), nt = (V + BN - 1) / BN, n = (int)N;
  CUtensorMap mx, mw;
  if (!sms || !map2(&mx, dtype, sv.xc, D, pad, D) || !map2(&mw, dtype, w, D, V, D)) return CHB_ERR_CUDA;
  if (launch_overlapped(ce_rows, dim3(1), dim3(1024), stream, targets, n, V, ignore_index, sv) != cudaSuccess) return CHB_ERR_CUDA;
  if (launch_overlapped(ce_gather, dim3((unsigned)(pad / 8)), dim3(256), stream, (const char*)x, ldx, n, D, sv,
                        reduction == 0 ? loss : nullptr) != cudaSuccess) return CHB_ERR_CUDA;
  GemmArgs p{};
  p.count = sv.head;
  p.N = n; p.V = V; p.D = D; p.K = D; p.vn = V;
  p.part = f.part; p.tlogit = f.tlogit; p.tgt = sv.tgt; p.rows_pad = (int)pad;
  p.status = status_word();
  if (!p.status) return CHB_ERR_CUDA;
  const long long tiles = pad / BM * nt;
  const cudaError_t e = dtype == CHB_F16 ? gemm<__half, LSE>(mx, mw, p, tiles, sms, stream)
                                         : gemm<__nv_bfloat16, LSE>(mx, mw, p, tiles, sms, stream);
  if (e != cudaSuccess) return CHB_ERR_CUDA;
  if (launch_overlapped(ce_join, dim3((unsigned)(pad / 32)), dim3(256), stream, (const float2*)f.part, (const float*)f.tlogit, nt, (int)pad,
                        reduction, sv, f.sums, loss) != cudaSuccess) return CHB_ERR_CUDA;
  return CHB_SUCCESS;
}

int chb_linear_ce_backward(int dtype, const void* w, const float* grad, long long N, int D, int V, int reduction, const void* saved,
                           void* work, void* dx, void* dw, cudaStream_t stream) {
  if (!sizes_ok(dtype, N, D, V, reduction) || !w || !grad || !saved || !work || (reinterpret_cast<uintptr_t>(w) & 15u)) return CHB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw)) & 15u) return CHB_ERR_ARG;
  if (!dx && !dw) return CHB_SUCCESS;
  Saved sv;
  Bwd b;
  saved_layout(static_cast<char*>(const_cast<void*>(saved)), N, D, &sv);
  bwd_layout(static_cast<char*>(work), N, D, V, &b);
  const int sms = sm_count();
  if (!sms) return CHB_ERR_CUDA;
  const long long rows8 = (N + 7) / 8;
  if (launch_overlapped(ce_weights, dim3((unsigned)(rows8 < 2 * sms ? rows8 : 2 * sms)), dim3(256), stream, grad, reduction, (int)N, D,
                        sv, b.gs, b.coef, static_cast<char*>(dx)) != cudaSuccess) return CHB_ERR_CUDA;
  char *x = static_cast<char*>(dx), *v = static_cast<char*>(dw);
  const char* ww = static_cast<const char*>(w);
  return dtype == CHB_F16 ? backward<__half>(dtype, ww, (int)N, D, V, sv, b, x, v, sms, stream)
                          : backward<__nv_bfloat16>(dtype, ww, (int)N, D, V, sv, b, x, v, sms, stream);
}

}  // extern "C"

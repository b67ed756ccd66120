// Softmax cross entropy of a linear output layer, logits = x W^T, without the logits: they exist as accumulators of one
// tile at a time, and for the gradient as one piece of the vocabulary in 16 bits.
//
//   loss_r = log sum_v exp(l_rv) - l_r,t(r)          G_rv = (exp(l_rv - lse_r) - [v = t(r)]) g_r
//   dx = G W                                          dW = G^T x
//
// Forward: rows with a label are gathered (a row without one costs nothing, and whatever its x holds, infinities
// included, reaches neither the loss nor dW); one product whose epilogue keeps maximum and sum of exponentials of 256
// columns; a small kernel joins them.  Backward, for each piece of the vocabulary: the product again with an epilogue
// that writes G, then one launch for dW (complete for the piece) and dx (summed over the pieces in fp32) from G.
//
// Sums are fp32.  G is rounded to the operands' type, as the tensor cores need it; an fp16 G is kept 2^14 times larger
// and relative to the largest |g_r|, or softmax tails would fall below fp16's range.
#include "../api/chb.h"
#include "common.cuh"
#include "tc.cuh"

namespace chb {
namespace {

using namespace tc;

constexpr int BM = 128, BN = 256, BK = 64, kStages = 4;      // (BN: a tile's columns at most)
constexpr int kBox = 64 * 128;                               // bytes of 64 rows of 64 elements
constexpr int kStageBytes = (BM + BN) * BK * 2;
constexpr int kGemmSmem = kStages * kStageBytes + 1024;      // (1024: the swizzle's alignment)
constexpr float kLog2e = 1.4426950408889634f;

enum Mode { LSE, GRAD, BOTH };      // BOTH: dW and dx of a piece in one launch

// Kept from forward to backward.
struct Saved {
  int* head;       // [0] rows with a label, [1] CTAs of the joining kernel that are done
  int* idx;        // row of x of every gathered row
  int* pos;        // gathered row of every row of x, -1: none
  int* tgt;        // label of every gathered row, -1: not in the vocabulary
  float2* norm;    // largest logit, and log2 of the sum of the exponentials relative to it (one number for both would round by the
                   // size of the logits: a factor of 2^(1/16) at 2^20, infinity from 2^32 on)
  char* xc;        // gathered rows
};

struct GemmArgs {
  const int* count;
  int V, v0, vn;             // vocabulary, first column and width of the piece
  int D;
  int a_rows;                // LSE and GRAD: rows of x that a tile loads (all 128, or all there are: the others' results go nowhere)
  int bn;                    // columns of a tile: a multiple of 32 (GRAD and BOTH: of 64)
  // LSE
  float2* part;
  float* tlogit;
  const int* tgt;
  int rows_pad;
  // GRAD
  const float2* norm;
  const float* gs;
  char* g;
  long long ldg;
  // BOTH
  int split_w, split_x;      // shares of the summed axis; more than one: fp32 sums in slabs, joined by ce_finish
  float* slab_w;             // [split_w][vn][D]
  float* slab_x;             // [split_x][rows_pad][D], summed over the pieces
  int first, last;
  const float* coef;
  const int* idx;
  char *dx, *dw;             // null: not wanted
  unsigned* status;
};

__device__ __forceinline__ void st256(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

template <typename T> struct GScale { static constexpr float up = 1.f, down = 1.f; };
template <> struct GScale<__half> { static constexpr float up = 16384.f, down = 1.f / 16384.f; };

// 32 columns of a finished fp32 row, to the 16-bit row `out` or, added to what is there if `add`, to the fp32 row `sum`
template <typename T>
__device__ __forceinline__ void finish_cols(const uint32_t* r, int col, int D, float* sum, bool add, char* out, float coef) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = col + 8 * q;
    if (c >= D) break;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[8 * q + j]);
    if (add) {
      const float4 x = reinterpret_cast<const float4*>(sum + c)[0], y = reinterpret_cast<const float4*>(sum + c)[1];
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    if (out) {
      uint4 o;
      o.x = pack2<T>(v[0] * coef, v[1] * coef);
      o.y = pack2<T>(v[2] * coef, v[3] * coef);
      o.z = pack2<T>(v[4] * coef, v[5] * coef);
      o.w = pack2<T>(v[6] * coef, v[7] * coef);
      *reinterpret_cast<uint4*>(out + c * 2) = o;
    } else {
      reinterpret_cast<float4*>(sum + c)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(sum + c)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
}

// One tile of a launch: its rows, columns and summed range (in steps of BK)
struct TilePlace {
  bool w;                    // BOTH: a tile of dW (else of dx)
  int m0, n0, k0, k1, split;
};

// One persistent CTA per SM; warp 0 loads, warp 1 issues the products, warps 4 to 7 finish a tile (thread = row) while the
// next one is summed in the other half of tensor memory.  Bound by the tensor cores where there are many rows (8192 x 1024 x
// 50257: LSE 516 us, a piece of 12288 columns GRAD 133 and BOTH 262 us, 1.55 to 1.63 PFLOP/s alone, less once the power limit
// holds the clock), by the streaming of W where there are few (33 rows: 103 MB in 20 us from L2, 28 us from HBM).
// Maps: gathered rows and W (LSE and GRAD: boxes of a tile's rows and columns, else of 64), and BOTH: G.
template <typename T, int MODE>
__global__ void __launch_bounds__(256, 1)
ce_gemm(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mg, const GemmArgs p) {
  constexpr int STAGES = kStages, STAGE = kStageBytes;
  extern __shared__ char smem_raw[];
  __shared__ __align__(8) unsigned long long full_[STAGES], empty_[STAGES], done_[2], free_[2];
  __shared__ uint32_t tmem_;
  __shared__ Fault fault;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full = smem_u32(full_), empty = smem_u32(empty_), done = smem_u32(done_), free_b = smem_u32(free_);
  if (threadIdx.x == 0) {
    fault.raised = 0;
    fault.status = p.status;
    for (int i = 0; i < STAGES; ++i) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { bar_init(done + 8 * i, 1); bar_init(free_b + 8 * i, 128); }
    bar_init_done();
    prefetch_map(&mx);
    prefetch_map(&mw);
    if (MODE == BOTH) prefetch_map(&mg);
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_), 2 * BN);
  fence_before();
  __syncthreads();
  fence_after();
  dependent_launch();
  const uint32_t tmem = tmem_;
  const int count = *(volatile const int*)p.count;
  const int bn = p.bn, rows_t = (count + BM - 1) / BM, nt = ((MODE == BOTH ? p.D : p.vn) + bn - 1) / bn;
  const int voc_t = (p.vn + BM - 1) / BM;
  const int kd = (p.D + BK - 1) / BK, kw = (count + BK - 1) / BK, kx = (p.vn + BK - 1) / BK;
  const int tiles_w = MODE == BOTH && p.dw ? voc_t * nt * p.split_w : 0;
  const int tiles = MODE == BOTH ? tiles_w + (p.dx ? rows_t * nt * p.split_x : 0) : rows_t * nt;
  // neighbouring CTAs share the operand that is read from HBM: the rows of W (LSE, GRAD) or of G (BOTH, the longer sums first)
  const auto place = [&](int t) {
    TilePlace q{};
    if (MODE != BOTH) {
      q.m0 = t % rows_t * BM;
      q.n0 = t / rows_t * bn;
      q.k1 = kd;
      return q;
    }
    q.w = t < tiles_w;
    if (!q.w) t -= tiles_w;
    const int per = (q.w ? voc_t : rows_t) * nt, k = q.w ? kw : kx, splits = q.w ? p.split_w : p.split_x;
    q.split = t / per;
    t -= q.split * per;
    q.m0 = t / nt * BM;
    q.n0 = t % nt * bn;
    q.k0 = (int)((long long)k * q.split / splits);
    q.k1 = (int)((long long)k * (q.split + 1) / splits);
    return q;
  };

  if (warp == 0) {
    const bool one = elect();
    int s = 0;
    unsigned ph = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const TilePlace q = place(t);
      for (int k = q.k0; k < q.k1; ++k) {
        if (!(ok = bar_wait_warp(empty + 8 * s, ph ^ 1u, &fault))) break;
        const uint32_t bar = full + 8 * s, a = smem + s * STAGE, b = a + BM * BK * 2;
        if (one) {
          bar_expect(bar, ((MODE == BOTH ? BM : p.a_rows) + bn) * BK * 2);
          if (MODE != BOTH) {
            load2(a, &mx, k * BK, q.m0, bar);
            load2(b, &mw, k * BK, p.v0 + q.n0, bar);
          } else if (q.w) {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) load2(a + j * kBox, &mg, q.m0 + 64 * j, k * BK, bar);
            for (int j = 0; j < bn / 64; ++j) load2(b + j * kBox, &mx, q.n0 + 64 * j, k * BK, bar);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) load2(a + j * kBox, &mg, k * BK, q.m0 + 64 * j, bar);
            for (int j = 0; j < bn / 64; ++j) load2(b + j * kBox, &mw, q.n0 + 64 * j, p.v0 + k * BK, bar);
          }
        }
        __syncwarp();
        if (++s == STAGES) { s = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    const bool one = elect();
    int s = 0, buf = 0;
    unsigned ph = 0, bph = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const TilePlace q = place(t);
      if (q.k0 == q.k1) continue;
      const bool a_mn = MODE == BOTH && q.w;
      constexpr bool b_mn = MODE == BOTH;
      const uint32_t desc = product_desc<T>(BM, bn, a_mn, b_mn);
      const uint32_t a_step = a_mn ? 128 : 2;
      if (!(ok = bar_wait_warp(free_b + 8 * buf, bph ^ 1u, &fault))) break;
      fence_after();
      for (int k = q.k0; k < q.k1; ++k) {
        if (!(ok = bar_wait_warp(full + 8 * s, ph, &fault))) break;
        fence_after();
        const uint32_t a = smem + s * STAGE, b = a + BM * BK * 2;
        const uint64_t da = operand(a, a_mn ? kBox : 16), db = operand(b, b_mn ? kBox : 16);
        if (one) {
#pragma unroll
          for (int i = 0; i < BK / 16; ++i) mma_ss(tmem + buf * BN, da + i * a_step, db + i * (b_mn ? 128 : 2), desc, k > q.k0 || i > 0);
          commit(empty + 8 * s);
        }
        __syncwarp();
        if (++s == STAGES) { s = 0; ph ^= 1u; }
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
      const TilePlace q = place(t);
      const bool nothing = q.k0 == q.k1;      // (no row has a label: zeros)
      const int row = q.m0 + (warp & 3) * 32 + lane, n0 = q.n0;
      if (!nothing && !bar_wait_warp(done + 8 * buf, bph, &fault)) break;
      fence_after();
      const uint32_t src = tmem + buf * BN + lanes;
      if (MODE != BOTH) {
        const bool in = row < count;
        const int tg = in ? p.tgt[row] - p.v0 - n0 : -1;
        const int cols = min(bn, p.V - p.v0 - n0);
        float m = -INFINITY, sum = 0.f;
        float2 norm = make_float2(0.f, 0.f);
        float gs = 0.f;
        if (MODE == GRAD && in) { norm = p.norm[row]; gs = p.gs[row] * GScale<T>::up; }
#pragma unroll 1
        for (int c = 0; c < bn; c += 32) {
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
            // (subtracted ahead of the factor: exact where it matters, whatever the logits' size)
            const float ref = cm == -INFINITY ? 0.f : cm;
            float add = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) add += ex2((__uint_as_float(r[j]) - ref) * kLog2e);
            sum = fmaf(sum, ex2((m - ref) * kLog2e), add);
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
            for (int j = 0; j < 32; ++j) v[j] = ex2(fmaf(__uint_as_float(r[j]) - norm.x, kLog2e, -norm.y));
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
            if (n0 + c < p.ldg) {      // (a piece is as wide as its G: its last tile may be wider)
              char* d = p.g + ((long long)row * p.ldg + n0 + c) * 2;
              st256(d, o);
              st256(d + 32, o + 8);
            }
          }
        }
        if (MODE == LSE && in) p.part[(long long)(n0 / bn) * p.rows_pad + row] = make_float2(m, sum);
      } else {
        const bool in = row < (q.w ? min(p.vn, p.V - p.v0) : count);
        const float coef = *p.coef * GScale<T>::down;
        float* sum = nullptr;
        char* out = nullptr;
        bool add = false;
        if (q.w) {
          if (p.split_w > 1) sum = p.slab_w + ((long long)q.split * p.vn + row) * p.D;
          else out = p.dw + (long long)(p.v0 + row) * p.D * 2;
        } else {
          sum = p.slab_x + ((long long)q.split * p.rows_pad + row) * p.D;
          add = !p.first;
          if (in && p.last && p.split_x == 1) out = p.dx + (long long)p.idx[row] * p.D * 2;
        }
#pragma unroll 1
        for (int c = 0; c < bn; c += 32) {
          uint32_t r[32];
          __syncwarp();
          ld32(src + c, r);
          wait_ld(r);
          if (nothing) {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0;
          }
          if (in) finish_cols<T>(r, n0 + c, p.D, sum, add, out, coef);
        }
      }
      fence_before();
      if (nothing) continue;
      bar_arrive(free_b + 8 * buf);
      if (++buf == 2) { buf = 0; bph ^= 1u; }
    }
  }
  __syncthreads();
  if (fault.raised) drain_after_abort();
  __syncthreads();
  if (warp == 1) tmem_free(tmem, 2 * BN);
}

// Joins the slabs of a split sum, in their order: rows of dx go where they came from, rows of dW stay (blockIdx.y).
template <typename T>
__global__ void __launch_bounds__(256) ce_finish(const GemmArgs p) {
  dependent_launch();
  const bool w = blockIdx.y == 0;
  const int splits = w ? p.split_w : p.split_x;
  if (splits < 2 || !(w ? p.dw : p.dx)) return;
  const int count = *(volatile const int*)p.count;
  const float coef = *p.coef * GScale<T>::down;
  const long long words = p.D / 8, rows = w ? p.vn : count, apart = (long long)(w ? p.vn : p.rows_pad) * p.D;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * words; i += (long long)gridDim.x * 256) {
    const long long row = i / words;
    const float* f = (w ? p.slab_w : p.slab_x) + i * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(f + k * apart)), y = __ldcg(reinterpret_cast<const float4*>(f + k * apart) + 1);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    uint4 o;
    o.x = pack2<T>(v[0] * coef, v[1] * coef);
    o.y = pack2<T>(v[2] * coef, v[3] * coef);
    o.z = pack2<T>(v[4] * coef, v[5] * coef);
    o.w = pack2<T>(v[6] * coef, v[7] * coef);
    char* out = w ? p.dw + i * 16 : p.dx + ((long long)p.idx[row] * words + i % words) * 16;
    *reinterpret_cast<uint4*>(out) = o;
  }
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

// Both in one launch for few rows: every CTA counts the labels ahead of its own eight rows for itself (and all of them, for the
// zeros behind the last).
constexpr int kCountedRows = 4096;
__global__ void __launch_bounds__(256)
ce_gather_few(const long long* targets, const char* x, long long ldx, int N, int D, int V, long long ignore, Saved sv, float* loss_rows) {
  __shared__ int before_[8], all_[8];
  dependent_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r0 = blockIdx.x * 8;
  int before = 0, all = 0;
  for (int r = threadIdx.x; r < N; r += 256) {
    const int in = targets[r] != ignore;
    all += in;
    before += r < r0 ? in : 0;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if (lane == 0) {
    before_[warp] = before;
    all_[warp] = all;
  }
  __syncthreads();
  before = all = 0;
  for (int k = 0; k < 8; ++k) {
    before += before_[k];
    all += all_[k];
  }
  const int r = r0 + warp;
  const long long mine = lane < 8 && r0 + lane < N ? targets[r0 + lane] : ignore;
  const unsigned in = __ballot_sync(0xffffffffu, mine != ignore);
  const int at = before + __popc(in & ((1u << warp) - 1u)), words = D / 8;
  const long long t = __shfl_sync(0xffffffffu, mine, warp);
  if (r < N) {
    const bool has = (in >> warp) & 1u;
    if (lane == 0) {
      sv.pos[r] = has ? at : -1;
      if (has) {
        sv.idx[at] = r;
        sv.tgt[at] = t >= 0 && t < V ? (int)t : -1;
      } else if (loss_rows) {
        loss_rows[r] = 0.f;
      }
    }
    if (has) {
      const uint4* s = reinterpret_cast<const uint4*>(x + (long long)r * ldx * 2);
      uint4* d = reinterpret_cast<uint4*>(sv.xc + (long long)at * D * 2);
      for (int i = lane; i < words; i += 32) d[i] = s[i];
    }
  }
  if (r >= all && r < (all + BM - 1) / BM * BM) {
    uint4* d = reinterpret_cast<uint4*>(sv.xc + (long long)r * D * 2);
    for (int i = lane; i < words; i += 32) d[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    sv.head[0] = all;
    sv.head[1] = 0;
  }
}

// Joins the column tiles of 32 rows (lane = row, the 32 warps take every 32nd tile, eight loads at a time: the kernel is a
// chain of latencies, 15.2 us with eight warps and four loads at a time, 4.0 us so, 33 rows of 50257 columns) and, in the last
// CTA to come, the sum over the rows: CTA sums in the order of the rows, whichever CTA is last.
constexpr int kJoinWarps = 32, kJoinLoads = 8;

__global__ void __launch_bounds__(kJoinWarps * 32)
ce_join(const float2* part, const float* tlogit, int nt, int rows_pad, int reduction, Saved sv, double* sums, float* loss) {
  __shared__ float sm[kJoinWarps][32], ss[kJoinWarps][32];
  __shared__ int is_last;
  dependent_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int count = *(volatile const int*)sv.head;
  const int row = blockIdx.x * 32 + lane;
  const bool in = row < count;
  int label = -1;
  float target = 0.f;
  if (in && warp == 0) label = sv.tgt[row], target = tlogit[row];
  float m = -INFINITY, s = 0.f;
  if (in) {
    for (int t0 = warp; t0 < nt; t0 += kJoinWarps * kJoinLoads) {
      float2 v[kJoinLoads];
#pragma unroll
      for (int i = 0; i < kJoinLoads; ++i) {
        const int t = t0 + i * kJoinWarps;
        v[i] = t < nt ? part[(long long)t * rows_pad + row] : make_float2(-INFINITY, 0.f);
      }
      float nm = m;
#pragma unroll
      for (int i = 0; i < kJoinLoads; ++i) nm = fmaxf(nm, v[i].x);
      const float ref = nm == -INFINITY ? 0.f : nm;
      s *= ex2((m - ref) * kLog2e);
#pragma unroll
      for (int i = 0; i < kJoinLoads; ++i) s += v[i].y * ex2((v[i].x - ref) * kLog2e);
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
      for (int w = 1; w < kJoinWarps; ++w) M = fmaxf(M, sm[w][lane]);
      const float ref = M == -INFINITY ? 0.f : M;
      float S = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) S += ss[w][lane] * ex2((sm[w][lane] - ref) * kLog2e);
      const bool known = label >= 0;
      loss_r = known ? logf(S) + (M - target) : __int_as_float(0x7fffffff);      // (no such label: NaN)
      sv.norm[row] = make_float2(known ? M : __int_as_float(0x7fffffff), log2f(S));
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

// Before the backward products: every row's weight relative to the largest finite one, that largest, and zeros in dx where a row
// has no label.  Every CTA finds the largest for itself (the gradients of the rows are few bytes and in L2).  A row whose gradient
// is infinite or NaN keeps that as its weight, so it reaches its own dx (and dW, which sums over all rows) and no other row's.
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
      m = a > m && a < INFINITY ? a : m;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) mx[warp] = m;
    __syncthreads();
    top = mx[0];
    for (int w = 1; w < 8; ++w) top = fmaxf(top, mx[w]);
    if (top == 0.f) top = 1.f;      // (zeros, infinities and NaN only: they stay what they are)
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
// Bytes of G at most, as long as that leaves a piece 256 columns: above 393216 rows a piece has 256, and G 512 bytes a row.
// A launch costs about ten microseconds of its own, so fewer pieces are faster though less of G is in L2
// when it is read (8192 x 1024 x 50257: 48 MiB 3209 us, 96 MiB 2770, 192 MiB 2612, 384 MiB 2598).
constexpr long long kPieceBytes = 192ll << 20;

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
  sv->norm = c.take<float2>(pad * 8);
  sv->xc = c.take<char>(pad * D * 2);
  return c.at;
}

struct Fwd { float2* part; float* tlogit; double* sums; };
long long fwd_layout(char* base, long long N, int V, int bn, Fwd* w) {
  Carve c{base};
  const long long pad = up(N, BM);
  w->part = c.take<float2>(pad * 8 * ((V + bn - 1) / bn));
  w->tlogit = c.take<float>(pad * 4);
  w->sums = c.take<double>(pad / 32 * 8);
  return c.at;
}

// Columns of a tile of rows times W: 256 where there are many tiles, else the width at which the SMs' last round is fullest (33
// rows, 50257 columns: 148 SMs have two tiles of 192 each instead of one or two of 256).
int tile_columns(long long rows_t, long long columns, int sms, int unit) {
  int best = BN;
  long long least = -1;
  for (long long rounds = 1; rounds <= 8; ++rounds) {
    const long long across = rounds * sms / rows_t;      // column tiles that so many rounds have room for
    if (!across) continue;
    const long long bn = up((columns + across - 1) / across, unit);
    if (bn > BN) continue;
    const long long cost = rounds * ((bn < 128 ? 128 : bn) + 16);
    if (least < 0 || cost < least) {
      least = cost;
      best = (int)bn;
    }
  }
  return best;
}

// With few rows the way from L2 to the SMs is the limit, and a tile's 128 rows of x would take a third of it.
int rows_loaded(long long N) { return N < BM ? (int)up(N, 8) : BM; }

// How the backward pass is cut for N rows: the width of a piece of the vocabulary (its G takes kPieceBytes at most), and into
// how many shares the sums of dW and dx are split where there are too few tiles for the SMs.
struct Plan { int width, pieces, split_w, split_x, bn_g, bn_d; };

// The longest CTA of a launch in which CTA c takes the tiles c, c + sms, ...: `first` tiles of length `a`, then `second` of length
// `b`.  What a CTA has changes only at the remainders of the two counts.
long long longest(long long first, long long a, long long second, long long b, int sms) {
  long long most = 0;
  for (const long long c : {0ll, first % sms, (first + second) % sms}) {
    const long long n = (first + second - c + sms - 1) / sms, n1 = (first - c + sms - 1) / sms;
    const long long l = n1 * a + (n - n1) * b;
    if (l > most) most = l;
  }
  return most;
}

Plan make_plan(long long N, int D, int V, int sms) {
  const long long pad = up(N, BM), rows_t = pad / BM, kw = (N + BK - 1) / BK;
  Plan q{};
  const long long nt = (D + BN - 1) / BN;
  q.bn_d = (int)up((D + nt - 1) / nt, 64);
  long long most = kPieceBytes / (pad * 2) / BM * BM;
  if (most < 256) most = 256;
  if (most > up(V, BM)) most = up(V, BM);
  // the width at which the launches' last rounds waste least: products of G in tiles, then dW and dx together
  long long best = -1;
  const long long step = up(most / 64, BM);
  for (long long width = most; width >= 256 && width * 2 > most; width -= step) {
    const long long pieces = (V + width - 1) / width, g = (rows_t * ((width + 255) / 256) + sms - 1) / sms * ((D + BK - 1) / BK) * 2;
    const long long d = longest(width / BM * nt, kw, rows_t * nt, width / BK, sms) * q.bn_d / 128;
    const long long cost = pieces * (g + d + 8);      // (8: a launch's first loads and last stores, in steps)
    if (best < 0 || cost < best) {
      best = cost;
      q.width = (int)width;
    }
  }
  if (best < 0) q.width = (int)most;
  q.pieces = (V + q.width - 1) / q.width;
  const long long voc_t = (q.width + BM - 1) / BM, kx = q.width / BK;
  long long target = (voc_t * nt * kw + rows_t * nt * kx + sms - 1) / sms;
  if (target < 8) target = 8;
  const auto split = [&](long long k) { const long long n = 2 * k > 3 * target ? (k + target - 1) / target : 1; return (int)(n > 32 ? 32 : n); };
  q.split_x = split(kx);
  q.split_w = q.pieces == 1 ? split(kw) : 1;
  q.bn_g = tile_columns(rows_t, q.width, sms, 64);      // (dx sums over G in steps of 64: all of them have to be written)
  return q;
}

struct Bwd { float* gs; float* coef; float* slab_x; float* slab_w; char* g; };
long long bwd_layout(char* base, long long N, int D, int V, const Plan& q, Bwd* w) {
  Carve c{base};
  const long long pad = up(N, BM);
  w->gs = c.take<float>(pad * 4);
  w->coef = c.take<float>(4);
  w->slab_x = c.take<float>(pad * D * 4 * q.split_x);
  w->slab_w = c.take<float>(q.split_w > 1 ? (long long)q.width * D * 4 * q.split_w : 0);
  w->g = c.take<char>(pad * q.width * 2);
  return c.at;
}

template <typename T, int MODE>
cudaError_t gemm(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& g, const GemmArgs& p, long long tiles, int sms, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  return launch_big(ce_gemm<T, MODE>, kGemmSmem, (unsigned)(tiles < sms ? tiles : sms), 256, stream, done, x, w, g, p);
}

bool map2(CUtensorMap* m, int dtype, const void* base, long long inner, long long rows, long long ld, int box_rows = 64) {
  const unsigned long long d[2] = {(unsigned long long)inner, (unsigned long long)rows}, s[1] = {(unsigned long long)ld};
  return make_map(m, dtype, base, 2, d, s, (unsigned)box_rows);
}

bool sizes_ok(int dtype, long long N, int D, int V, int reduction) {
  return (dtype == CHB_BF16 || dtype == CHB_F16) && N >= 1 && N < (1ll << 31) - 256 && D >= 8 && D % 8 == 0 && V >= 1 &&
         V < (1 << 30) && reduction >= 0 && reduction <= 2;
}

template <typename T>
int backward(int dtype, const char* w, int N, int D, int V, const Saved& sv, const Bwd& b, const Plan& q, char* dx, char* dw, int sms,
             cudaStream_t stream) {
  const long long pad = up(N, BM);
  CUtensorMap ma, mx, mw, mt, mg;
  if (!map2(&ma, dtype, sv.xc, D, pad, D, rows_loaded(N)) || !map2(&mx, dtype, sv.xc, D, pad, D) || !map2(&mw, dtype, w, D, V, D) || !map2(&mt, dtype, w, D, V, D, q.bn_g) ||
      !map2(&mg, dtype, b.g, q.width, pad, q.width)) return CHB_ERR_CUDA;
  GemmArgs p{};
  p.count = sv.head;
  p.V = V; p.D = D;
  p.tgt = sv.tgt; p.norm = sv.norm; p.gs = b.gs; p.g = b.g; p.ldg = q.width;
  p.slab_x = b.slab_x; p.slab_w = b.slab_w; p.split_x = q.split_x; p.split_w = q.split_w;
  p.rows_pad = (int)pad;
  p.a_rows = rows_loaded(N);
  p.coef = b.coef; p.idx = sv.idx; p.dx = dx; p.dw = dw;
  p.status = status_word();
  if (!p.status) return CHB_ERR_CUDA;
  const long long rows_t = pad / BM, nt = (D + q.bn_d - 1) / q.bn_d;
  for (int v0 = 0; v0 < V; v0 += q.width) {
    p.v0 = v0;
    p.vn = V - v0 < q.width ? V - v0 : q.width;
    p.first = v0 == 0;
    p.last = v0 + q.width >= V;
    p.bn = q.bn_g;
    if (gemm<T, GRAD>(ma, mt, mg, p, rows_t * ((p.vn + p.bn - 1) / p.bn), sms, stream) != cudaSuccess) return CHB_ERR_CUDA;
    const long long tiles = (dw ? (p.vn + BM - 1) / BM * nt * q.split_w : 0) + (dx ? rows_t * nt * q.split_x : 0);
    p.bn = q.bn_d;
    if (gemm<T, BOTH>(mx, mw, mg, p, tiles, sms, stream) != cudaSuccess) return CHB_ERR_CUDA;
  }
  if (q.split_x > 1 || q.split_w > 1) {
    if (launch_overlapped(ce_finish<T>, dim3((unsigned)(2 * sms), 2), dim3(256), stream, p) != cudaSuccess) return CHB_ERR_CUDA;
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
  const int sms = sm_count();
  if (!sms) return CHB_ERR_CUDA;
  *forward = fwd_layout(nullptr, N, V, tile_columns(up(N, BM) / BM, V, sms, 32), &f);
  *backward = bwd_layout(nullptr, N, D, V, make_plan(N, D, V, sms), &b);
  return CHB_SUCCESS;
}

int chb_linear_ce_forward(int dtype, const void* x, long long ldx, const void* w, const long long* targets, long long N, int D,
                          int V, long long ignore_index, int reduction, float* loss, void* saved, void* work, cudaStream_t stream) {
  if (!sizes_ok(dtype, N, D, V, reduction) || !x || !w || !targets || !loss || !saved || !work || ldx % 8) return CHB_ERR_ARG;
  if (!on_boundary(16, x, w, saved, work) || !on_boundary(8, targets) || !on_boundary(4, loss)) return CHB_ERR_ARG;
  Saved sv;
  Fwd f;
  const long long pad = up(N, BM);
  const int sms = sm_count(), n = (int)N;
  if (!sms) return CHB_ERR_CUDA;
  const int bn = tile_columns(pad / BM, V, sms, 32), nt = (V + bn - 1) / bn;
  saved_layout(static_cast<char*>(saved), N, D, &sv);
  fwd_layout(static_cast<char*>(work), N, V, bn, &f);
  CUtensorMap mx, mw;
  if (!map2(&mx, dtype, sv.xc, D, pad, D, rows_loaded(n)) || !map2(&mw, dtype, w, D, V, D, bn)) return CHB_ERR_CUDA;
  float* const loss_rows = reduction == 0 ? loss : nullptr;
  const char* const xs = static_cast<const char*>(x);
  if (n <= kCountedRows) {
    if (launch_overlapped(ce_gather_few, dim3((unsigned)(pad / 8)), dim3(256), stream, targets, xs, ldx, n, D, V, ignore_index, sv, loss_rows) != cudaSuccess) return CHB_ERR_CUDA;
  } else if (launch_overlapped(ce_rows, dim3(1), dim3(1024), stream, targets, n, V, ignore_index, sv) != cudaSuccess ||
             launch_overlapped(ce_gather, dim3((unsigned)(pad / 8)), dim3(256), stream, xs, ldx, n, D, sv, loss_rows) != cudaSuccess) {
    return CHB_ERR_CUDA;
  }
  GemmArgs p{};
  p.count = sv.head;
  p.V = V; p.D = D; p.vn = V; p.bn = bn; p.a_rows = rows_loaded(n);
  p.part = f.part; p.tlogit = f.tlogit; p.tgt = sv.tgt; p.rows_pad = (int)pad;
  p.status = status_word();
  if (!p.status) return CHB_ERR_CUDA;
  const long long tiles = pad / BM * nt;
  const cudaError_t e = dtype == CHB_F16 ? gemm<__half, LSE>(mx, mw, mw, p, tiles, sms, stream)
                                         : gemm<__nv_bfloat16, LSE>(mx, mw, mw, p, tiles, sms, stream);
  if (e != cudaSuccess) return CHB_ERR_CUDA;
  if (launch_overlapped(ce_join, dim3((unsigned)(pad / 32)), dim3(kJoinWarps * 32), stream, (const float2*)f.part, (const float*)f.tlogit, nt, (int)pad,
                        reduction, sv, f.sums, loss) != cudaSuccess) return CHB_ERR_CUDA;
  return CHB_SUCCESS;
}

int chb_linear_ce_backward(int dtype, const void* w, const float* grad, long long N, int D, int V, int reduction, const void* saved,
                           void* work, void* dx, void* dw, cudaStream_t stream) {
  if (!sizes_ok(dtype, N, D, V, reduction) || !w || !grad || !saved || !work) return CHB_ERR_ARG;
  // (G is stored in words of 32 bytes, at a multiple of 256 in `work`)
  if (!on_boundary(32, work) || !on_boundary(16, w, saved, dx, dw) || !on_boundary(4, grad)) return CHB_ERR_ARG;
  if (!dx && !dw) return CHB_SUCCESS;
  const int sms = sm_count();
  if (!sms) return CHB_ERR_CUDA;
  Saved sv;
  Bwd b;
  const Plan q = make_plan(N, D, V, sms);
  saved_layout(static_cast<char*>(const_cast<void*>(saved)), N, D, &sv);
  bwd_layout(static_cast<char*>(work), N, D, V, q, &b);
  const long long rows8 = (N + 7) / 8;
  if (launch_overlapped(ce_weights, dim3((unsigned)(rows8 < 2 * sms ? rows8 : 2 * sms)), dim3(256), stream, grad, reduction, (int)N, D,
                        sv, b.gs, b.coef, static_cast<char*>(dx)) != cudaSuccess) return CHB_ERR_CUDA;
  char *x = static_cast<char*>(dx), *v = static_cast<char*>(dw);
  const char* ww = static_cast<const char*>(w);
  return dtype == CHB_F16 ? backward<__half>(dtype, ww, (int)N, D, V, sv, b, q, x, v, sms, stream)
                          : backward<__nv_bfloat16>(dtype, ww, (int)N, D, V, sv, b, q, x, v, sms, stream);
}

}  // extern "C"

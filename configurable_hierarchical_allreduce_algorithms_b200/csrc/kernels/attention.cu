// Causal attention over packed sequences with grouped heads, and its gradients, on the tensor cores.
//
//   S = Q K^T;  P_ij = exp(scale S_ij - lse_i) for j <= i of the same sequence, else 0;  O = P V
//   D_i = dO_i . O_i;  dS = P (dO V^T - D);  dQ = scale dS K;  dK = scale dS^T Q;  dV = P^T dO
//
// A tile is 128 rows of 128 keys (or of 128 queries); a thread owns a row, so maxima and sums need no exchange.  Scores are
// accumulators in tensor memory; P and dS go back there in 16 bits as the left operand of the second product, over the
// scores that they came from, and never to shared or global memory.  Every operand tile is loaded once and serves as K-major
// operand of a score product and as MN-major operand of an output product.  Three kernels:
//
//   forward  a CTA has two tiles of queries at a time (neighbouring in (tile, head of the group) order, so that two heads share
//            the keys and values where there are groups): the products of one run while the other's exponentials are taken.
//            One pass with a running maximum; the sums are rescaled only when a maximum grows by more than 2^8.
//   dq       a CTA has a tile of queries and walks its keys; also finds D.
//   dkv      a CTA has a tile of keys of one key head and walks the queries of all heads of the group that see it, so
//            gradients of shared heads are summed in the accumulators, in one order: no atomics on results anywhere.  Where
//            there are few tiles for the SMs the group's heads are shared out; the last share to end adds all, in their order.
//
// Each has one CTA an SM that takes one piece of work after the other: the loads and first products of the next run under the
// end of this one (8 x 1024 tokens, 16 heads of 64, forward: a CTA for each piece 53 us).  A first small kernel lists the
// pieces, the longest first, and CTAs take them in turns forth and back, so that all end at about the same time.
//
// Sequences: the rows [cu[s], cu[s+1]); the list is made from the bounds on the device, so no length is needed on the host.
// Rows outside all sequences get zeros.  A tile that reaches past its sequence holds the next one's rows: those are overwritten with zeros
// where they would be summed over (a product 0 * infinity would carry them across).
//
// P and dS are rounded to the operands' type (as the tensor cores need them); maxima, sums, lse and D are fp32.  An fp16 dS is kept
// 2^k times larger, with k from the sizes of the dO and V that go into it (Range below): dO may be near either end of fp16's range
// (scaled losses, gradients of a mean over many tokens), where dS would be infinite or zero and dQ and dK, which sum it, are not.
#include "../api/chb.h"
#include "common.cuh"
#include "tc.cuh"

namespace chb {
namespace {

using namespace tc;

constexpr int TILE = 128;
constexpr int kAtom = TILE * 128;        // bytes of a tile's 64 elements: 128 rows of 128 bytes

struct AttnArgs {
  const int4* list;       // pieces of work: pairs (forward) or tiles
  const int* listed;      // how many
  int T, heads, kv_heads, group, D;
  float scale, scale_log2;
  char* o;                // [T, heads, D] (written by forward, read by dq)
  float* lse;             // [heads, T], in units of log2
  float* delta;           // [heads, T]
  float2* sizes;          // fp16: [kv_heads, T], at the first row of every tile the largest |dO_i| (of the group) and |V_j| there
  const char* v;          // for the sizes
  long long v_t, v_h;
  const char* dout;       // strides in elements
  long long dout_t, dout_h;
  char *dq, *dk, *dv;     // contiguous
  int split;              // dkv: shares of a group's heads, each a piece of its own
  float* sums;            // split > 1: [piece][share][dV, dK][column][row]
  int* arrived;           // shares of a piece that are there (dq clears them)
  int pieces;
  unsigned* status;
};

// Piece number `unit` of the rows [start, start + len): a tile, or a pair of (tile, head of the group), counted so that cost
// falls with the number; nothing: rows outside all sequences.
struct Work { int start, len, unit, nothing; };

// The pieces that this CTA takes: of the list times the heads, a row of them at a time, forth and back.  Little of it stays in
// registers: the list is read again where a warp needs a piece's place once more.
struct Walk {
  unsigned row = ~0u;
  __device__ __forceinline__ unsigned at() const { return row * gridDim.x + (row & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x); }      // number of the piece
  __device__ __forceinline__ bool next(int total) {
    for (++row; row * gridDim.x < (unsigned)total; ++row)
      if (at() < (unsigned)total) return true;
    return false;
  }
  __device__ __forceinline__ Work work(const AttnArgs& p, int heads) const {
    const int4 e = p.list[at() / heads];
    return Work{e.x, e.y, e.z, e.w};
  }
  __device__ __forceinline__ int head(int heads) const { return (int)(at() % heads); }
};

// Lists the pieces of all sequences by falling cost (tiles of keys to walk), by counting: one CTA.  Up to 1024 costs are kept
// apart, more share a place.  plan: [0] pairs, [1] tiles, then from the fourth int4 on both lists, `most[]` entries each.
// Sequences outside [0, T] or overlapping are clamped; what does not fit the lists is left out.
constexpr int kPlanHead = 4, kCosts = 1024;
__global__ void __launch_bounds__(1024) attn_plan(const int* cu, int seqs, int T, int group, int most_pairs, int most_tiles, int4* plan) {
  __shared__ int at[2][kCosts], warps[2][32], longest_;
  dependent_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = cu ? seqs + 2 : 1;      // (with the rows before the first and behind the last)
  const auto segment = [&](int s, int& a) {
    int b = T;
    a = 0;
    if (cu) {
      a = s == 0 ? 0 : min(max(cu[s - 1], 0), T);
      b = s == n - 1 ? T : min(max(cu[s], 0), T);
    }
    return max(b - a, 0);
  };
  at[0][tid] = at[1][tid] = 0;
  if (tid == 0) longest_ = 1;
  __syncthreads();
  for (int s = tid; s < n; s += 1024) {
    int a;
    const int len = segment(s, a);
    if (len > TILE) atomicMax(&longest_, (len + TILE - 1) / TILE);
  }
  __syncthreads();
  const int longest = longest_;
  const auto place = [&](int cost) { return longest <= kCosts ? longest - cost : (int)((long long)(longest - cost) * kCosts / longest); };
  // few sequences: a warp walks the pieces of one; many: a thread
  const auto walk = [&](auto&& each) {
    const bool few = n <= 64;
    for (int s = few ? warp : tid; s < n; s += few ? 32 : 1024) {
      int a;
      const int len = segment(s, a), tiles = (len + TILE - 1) / TILE, nothing = cu && (s == 0 || s == n - 1);
      for (int u = few ? lane : 0; u < tiles; u += few ? 32 : 1) each(1, a, len, u, nothing, nothing ? 1 : tiles - u);
      for (int u = few ? lane : 0; u < (tiles * group + 1) / 2; u += few ? 32 : 1) each(0, a, len, u, nothing, nothing ? 1 : tiles - 2 * u / group);
    }
  };
  walk([&](int l, int, int, int, int, int cost) { atomicAdd(&at[l][place(cost)], 1); });
  __syncthreads();
  int inc[2];
#pragma unroll
  for (int l = 0; l < 2; ++l) {
    inc[l] = at[l][tid];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc[l], d);
      if (lane >= d) inc[l] += v;
    }
    if (lane == 31) warps[l][warp] = inc[l];
  }
  __syncthreads();
  if (warp < 2) {
    int v = warps[warp][lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += u;
    }
    warps[warp][lane] = v;
  }
  __syncthreads();
#pragma unroll
  for (int l = 0; l < 2; ++l) {
    const int before = warp ? warps[l][warp - 1] : 0;
    at[l][tid] = before + inc[l] - at[l][tid];
    if (tid == 1023) reinterpret_cast<int*>(plan)[l] = min(before + inc[l], l ? most_tiles : most_pairs);
  }
  __syncthreads();
  walk([&](int l, int a, int len, int u, int nothing, int cost) {
    // (pieces of the same cost in any order: who works on a piece has no influence on its result)
    const int i = atomicAdd(&at[l][place(cost)], 1);
    if (i < (l ? most_tiles : most_pairs)) plan[kPlanHead + (l ? most_pairs : 0) + i] = make_int4(a, len, u, nothing);
  });
}

// rows [from, 128) of a tile of `atoms` x 64 elements become zero (by one warp)
__device__ __forceinline__ void zero_rows(char* tile, int atoms, int from) {
  const int lane = threadIdx.x & 31;
  for (int a = 0; a < atoms; ++a)
    for (int i = from * 8 + lane; i < TILE * 8; i += 32) reinterpret_cast<uint4*>(tile + a * kAtom)[i] = make_uint4(0u, 0u, 0u, 0u);
  fence_async_proxy();
  __syncwarp();
}

// A K-major tile as operand of the k-th 16 summed elements; and an MN-major one
__device__ __forceinline__ uint64_t along(uint64_t tile, int k) { return tile + (uint64_t)((k >> 2) * (kAtom >> 4) + (k & 3) * 2); }
__device__ __forceinline__ uint64_t across(uint64_t tile, int k) { return tile + (uint64_t)(k * 128); }

// A warp's 32 rows of `cols` columns of an accumulator, times a factor, to 16-bit rows in global memory: by way of 2 KB of shared
// memory of the warp's own, so that a store covers 64 bytes of eight rows and not one 16-byte word of 32 (an epilogue at D = 128:
// 5000 -> 1400 clocks).  `rows`: how many of the 32 exist, `pitch`: bytes between rows.
// fetch(c, r): the lane's row of columns c to c + 31.
template <typename T, typename F>
__device__ __forceinline__ void store_rows(F&& fetch, int cols, float f, char* stage, char* out, long long pitch, int rows, int col0, int D) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int c = 0; c < cols; c += 32) {
    uint32_t r[32];
    __syncwarp();
    fetch(c, r);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint4 o;
      o.x = pack2<T>(__uint_as_float(r[8 * q]) * f, __uint_as_float(r[8 * q + 1]) * f);
      o.y = pack2<T>(__uint_as_float(r[8 * q + 2]) * f, __uint_as_float(r[8 * q + 3]) * f);
      o.z = pack2<T>(__uint_as_float(r[8 * q + 4]) * f, __uint_as_float(r[8 * q + 5]) * f);
      o.w = pack2<T>(__uint_as_float(r[8 * q + 6]) * f, __uint_as_float(r[8 * q + 7]) * f);
      reinterpret_cast<uint4*>(stage)[lane * 4 + (q ^ (lane / 2 & 3))] = o;      // (words of neighbouring rows in different banks)
    }
    __syncwarp();
    const int col = col0 + c + lane % 4 * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 8 + lane / 4;
      const uint4 o = reinterpret_cast<const uint4*>(stage)[row * 4 + ((lane % 4) ^ (row / 2 & 3))];
      if (row < rows && col < D) *reinterpret_cast<uint4*>(out + row * pitch + col * 2) = o;
    }
  }
  __syncwarp();
}
// (from an accumulator)
struct FromTmem {
  uint32_t acc;
  __device__ __forceinline__ void operator()(int c, uint32_t (&r)[32]) const {
    ld32(acc + c, r);
    wait_ld(r);
  }
};

// (by the first `threads` threads of the CTA)
__device__ __forceinline__ void zero_out(char* base, long long first, int rows, int heads, int head, int D, int threads) {
  const int words = D / 8;
  for (int i = threadIdx.x; i < rows * words; i += threads)
    *reinterpret_cast<uint4*>(base + (((first + i / words) * heads + head) * D + i % words * 8) * 2) = make_uint4(0u, 0u, 0u, 0u);
}

// ------------------------------------------------------------------ forward
// Warps 0-7 and 8-15: rows of the two tiles, each row twice, half of the 128 columns a thread; 16: loads; 17 and 18: products
// of the two tiles; 19: zeros.
// What bounds the kernel is the chain scores -> softmax -> product of one tile (per tile of 128 x 128: 1024 clocks of products
// at D = 128, 1024 of the special function unit, and latencies between them), so each tile has a warp of its own for its
// products, and four warps a scheduler hide the latencies in a softmax (16384 tokens, 16 / 4 heads of 128: 858 us; with two
// warps a scheduler 1066 us, or 917 us with tile 1 held back by half a turn).  That is 1.28 PFLOP/s, the best of replayed passes;
// calls in a row, under the power limit, run at 1.1 (1000 us).  Short sequences pay for the ends of their pieces: 4 x 2048 tokens,
// 16 heads of 128, 85 us, 0.81 PFLOP/s; 8 x 1024, 16 of 64, 47 us.
constexpr int kFwdThreads = 640;

// Whether any of a tile's 256 threads wants it; barrier 1 + tile
__device__ __forceinline__ bool any_of_tile(int tile, bool want) {
  unsigned r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 256, p;\n selp.u32 %0, 1, 0, q;\n}"
               : "=r"(r) : "r"((unsigned)want), "r"(1 + tile) : "memory");
  return r != 0;
}
__device__ __forceinline__ void sync_tile(int tile) { asm volatile("barrier.cta.sync %0, 256;" ::"r"(1 + tile) : "memory"); }

// What a forward CTA makes of a piece: two of the sequence's (tile, head of the group), the second the same tile of the next head
// or the tile before.  (Members of one of the two are computed when asked for; arrays would go to local memory.)
struct Pair {
  int nt, unit, group, head0, len;
  __device__ __forceinline__ Pair(const Work& w, int kvh, int group_) : nt((w.len + TILE - 1) / TILE), unit(w.unit), group(group_), head0(kvh * group_), len(w.len) {}
  __device__ __forceinline__ int n(int u) const { return max(nt - (2 * unit + u) / group, 0); }      // tiles of keys; the tile is the last
  __device__ __forceinline__ int head(int u) const { return head0 + (2 * unit + u) % group; }
  __device__ __forceinline__ bool ragged() const { return n(0) * TILE > len; }      // the last tile of keys reaches past the sequence
};

template <typename T, int DP>
__global__ void __launch_bounds__(kFwdThreads, 1)
attn_forward(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
             const AttnArgs p) {
  constexpr int ATOMS = DP / 64, TB = ATOMS * kAtom;
  // At DP = 64 tensor memory has room for P beside the scores, and the next scores are made as soon as these are read.
  constexpr bool kApart = DP == 64;
  extern __shared__ char smem_raw[];
  __shared__ __align__(8) unsigned long long bars[22];
  __shared__ uint32_t tmem_;
  __shared__ Fault fault;
  char* const smem_p = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem = smem_u32(smem_p), bar0 = smem_u32(bars);
  // (two of each.  Turns go on counting from one piece of work to the next: a barrier's phase is its count of turns)
  const uint32_t qfull = bar0, qempty = bar0 + 16, kfull = bar0 + 32, kempty = bar0 + 48, vfull = bar0 + 64, vempty = bar0 + 80, sfull = bar0 + 96,
                 pfull = bar0 + 112, vready = bar0 + 128, sread = bar0 + 144, odone = bar0 + 160;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 17) tmem_alloc(smem_u32(&tmem_), 512);
  if (warp == 0) {
    if (lane == 31) {
      fault.raised = 0;
      fault.status = p.status;
    }
    const int kind = lane >> 1;      // (a lane a barrier)
    if (kind < 11) bar_init(bar0 + 8 * lane, kind == 3 ? 2 : kind == 5 ? 3 : kind == 7 || kind == 9 ? 256 : 1);
    bar_init_done();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_;
  dependent_launch();
  const int total = *(volatile const int*)p.listed * p.kv_heads;
  const uint32_t sq = smem, sk = smem + 2 * TB, sv = smem + 4 * TB;
  char* const stage = smem_p + 6 * TB;      // 2 KB a softmax warp

  if (warp == 16) {
    const bool one = elect();
    const auto load_tile = [&](uint32_t dst, const CUtensorMap* m, int row, int h, uint32_t bar) {
      if (one) {
        bar_expect(bar, TB);
#pragma unroll
        for (int a = 0; a < ATOMS; ++a) load3(dst + a * kAtom, m, 64 * a, row, h, bar);
      }
      __syncwarp();
    };
    bool ok = true;
    int g = 0, qn0 = 0, qn1 = 0;
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, p.kv_heads);
      const int kvh = it.head(p.kv_heads);
      if (w.nothing) continue;
      const Pair x(w, kvh, p.group);
      const int n0 = x.n(0), n1 = x.n(1);
      if (!(ok = bar_wait_warp(qempty, (qn0++ & 1) ^ 1, &fault))) break;
      load_tile(sq, &mq, w.start + (n0 - 1) * TILE, x.head(0), qfull);
      for (int i = 0; i < n0; ++i, ++g) {
        const int s = g & 1;
        const unsigned ph = ((g >> 1) & 1) ^ 1u;
        if (!(ok = bar_wait_warp(kempty + 8 * s, ph, &fault))) break;
        load_tile(sk + s * TB, &mk, w.start + i * TILE, kvh, kfull + 8 * s);
        if (i == 0 && n1) {
          if (!(ok = bar_wait_warp(qempty + 8, (qn1++ & 1) ^ 1, &fault))) break;
          load_tile(sq + TB, &mq, w.start + (n1 - 1) * TILE, x.head(1), qfull + 8);
        }
        if (!(ok = bar_wait_warp(vempty + 8 * s, ph, &fault))) break;
        load_tile(sv + s * TB, &mv, w.start + i * TILE, kvh, vfull + 8 * s);
      }
    }
  } else if (warp == 19) {
    // every tile of values goes through this warp's hands, which overwrites the rows behind the sequence (it keeps its place in
    // the ring so); only pieces with such rows wait for it
    bool ok = true;
    int g = 0;
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, p.kv_heads);
      const int kvh = it.head(p.kv_heads);
      if (w.nothing) continue;
      const Pair x(w, kvh, p.group);
      const int n0 = x.n(0);
      const bool ragged = x.ragged();
      for (int i = 0; i < n0; ++i, ++g) {
        const int s = g & 1;
        if (!(ok = bar_wait_warp(vfull + 8 * s, (g >> 1) & 1, &fault))) break;
        if (ragged && i == n0 - 1) zero_rows(smem_p + 4 * TB + s * TB, ATOMS, w.len - i * TILE);
        if (lane == 0) {
          bar_arrive(vready + 8 * s);
          bar_arrive(vempty + 8 * s);
        }
      }
    }
  } else if (warp >= 17) {
    const int u = warp - 17, ksteps = (p.D + 15) / 16;
    const bool one = elect();
    const uint32_t dscore = product_desc<T>(TILE, TILE, false, false);
    const uint32_t dout = product_desc<T>(TILE, ksteps * 16, false, true);
    const uint32_t ts = tmem + u * TILE, to = tmem + 2 * TILE + u * DP, tp = kApart ? tmem + 3 * TILE + u * 64 : ts;
    constexpr int kHalf = kApart ? 32 : 64;      // columns from one half of P to the other
    const uint64_t a = operand(sq + u * TB), k0 = operand(sk), v0 = operand(sv, kAtom);
    const auto scores = [&](int s, bool last) {
      const uint64_t b = k0 + (uint64_t)(s * (TB >> 4));
      if (one) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          if (k < ksteps) mma_ss(ts, along(a, k), along(b, k), dscore, k > 0);
        commit(sfull + 8 * u);
        commit(kempty + 8 * s);
        if (last) commit(qempty + 8 * u);
      }
      __syncwarp();
    };
    bool ok = true;
    int g = 0, t = 0, qn = 0;      // tiles of keys, own turns, own pieces
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, p.kv_heads);
      const int kvh = it.head(p.kv_heads);
      if (w.nothing) continue;
      const Pair x(w, kvh, p.group);
      const int n0 = x.n(0), nu = x.n(u);
      const bool ragged = x.ragged();
      if (nu) {
        if (!(ok = bar_wait_warp(qfull + 8 * u, qn++ & 1, &fault) && bar_wait_warp(kfull + 8 * (g & 1), (g >> 1) & 1, &fault))) break;
        scores(g & 1, nu == 1);
      }
#pragma unroll 1
      for (int i = 0; i < nu; ++i, ++g, ++t) {
        const int s = g & 1;
        const uint64_t b = v0 + (uint64_t)(s * (TB >> 4));
        if (i + 1 < nu && !(ok = bar_wait_warp(kfull + 8 * (s ^ 1), ((g + 1) >> 1) & 1, &fault))) break;
        if (kApart && i + 1 < nu) {
          if (!(ok = bar_wait_warp(sread + 8 * u, t & 1, &fault))) break;
          fence_after();
          scores(s ^ 1, i + 2 == nu);
        }
        // (the load first, even where the zeros count: the load comes behind the zeros' warp's last turn in this slot, so the phase
        // of vready that is asked for cannot be taken for the one before the last)
        if (!(ok = bar_wait_warp(vfull + 8 * s, (g >> 1) & 1, &fault) && (!ragged || bar_wait_warp(vready + 8 * s, (g >> 1) & 1, &fault)))) break;
        if (!(ok = bar_wait_warp(pfull + 8 * u, t & 1, &fault))) break;
        fence_after();
        if (one) {
#pragma unroll
          for (int k = 0; k < 8; ++k) mma_ts(to, tp + (k >> 2) * kHalf + (k & 3) * 8, across(b, k), dout, i > 0 || k > 0);
          if (kApart || i + 1 == nu) commit(odone + 8 * u);
        }
        __syncwarp();
        // the next scores go over P, behind the products that read it
        if (!kApart && i + 1 < nu) scores(s ^ 1, i + 2 == nu);
        if (one) commit(vempty + 8 * s);
        __syncwarp();
      }
      // tiles that only tile 0 sees: this one's arrivals
      for (int i = nu; i < n0 && ok; ++i, ++g) {
        const int s = g & 1;
        if (!(ok = bar_wait_warp(kfull + 8 * s, (g >> 1) & 1, &fault))) break;
        if (one) bar_arrive(kempty + 8 * s);
        if (!(ok = bar_wait_warp(vfull + 8 * s, (g >> 1) & 1, &fault))) break;
        if (one) bar_arrive(vempty + 8 * s);
        __syncwarp();
      }
    }
  } else {
    const int u = warp >> 3, half = (warp >> 2) & 1, r0 = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + u * TILE + half * 64 + lanes, tp = kApart ? tmem + 3 * TILE + u * 64 + half * 32 + lanes : ts,
                   to = tmem + 2 * TILE + u * DP + half * (DP / 2) + lanes;
    float* const joint = reinterpret_cast<float*>(stage + u * 8 * 2048);      // [half][row]; the outputs' way later
    const float sl = p.scale_log2;
    const uint64_t sl2 = pair(sl, sl);
    unsigned turn = 0, piece = 0;      // parities of the turns and of the pieces so far
    for (Walk it; it.next(total);) {
      const Work w = it.work(p, p.kv_heads);
      const Pair x(w, it.head(p.kv_heads), p.group);
      if (w.nothing) {
        for (int v = 0; v < 2; ++v)
          if (x.n(v)) zero_out(p.o, w.start + (x.n(v) - 1) * TILE, min(TILE, w.len - (x.n(v) - 1) * TILE), p.heads, x.head(v), p.D, 512);
        continue;
      }
      const int nu = x.n(u);
      if (!nu) continue;
      // The maximum that the sums are relative to, times scale log2 e.  Rows behind the sequence's end hold the next one's queries:
      // at infinity they never ask for the tile's maxima to be moved (which would change this sequence's rounding).
      float ref = (nu - 1) * TILE + r0 < x.len ? 0.f : INFINITY;
      uint64_t sum2[2] = {0ull, 0ull};       // (two zeros each)
      // The warps of a tile meet at barriers that cannot give up, so none of them leaves the loops: once a wait ran out all
      // waits end at once, and the turns that are left go over whatever the scores hold.
#pragma unroll 1
      for (int left = nu; left > 0; --left) {
        bar_wait_warp(sfull + 8 * u, turn, &fault);
        fence_after();
        uint32_t r[64];
        ld32(ts, r);
        ld32(ts + 32, r + 32);
        wait_ld(r);
        if (kApart) {
          fence_before();
          bar_arrive(sread + 8 * u);
        }
        if (left == 1) {
          const int last = r0 - half * 64;
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (c > last) r[c] = __float_as_uint(-INFINITY);
        }
        float m4[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) m4[c] = fmaxf(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]));
#pragma unroll
        for (int c = 4; c < 32; ++c) m4[c & 3] = max3(m4[c & 3], __uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]));
        const float top = max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]) * sl;
        const bool grows = any_of_tile(u, left == nu || top > ref + 8.f);
        if (kApart && left < nu) bar_wait_warp(odone + 8 * u, turn ^ 1, &fault);
        if (grows) {
          joint[half * TILE + r0] = top;
          sync_tile(u);
          const float both = fmaxf(top, joint[(half ^ 1) * TILE + r0]);
          sync_tile(u);
          if (left == nu) {
            // (no key with a weight yet: so low that any score moves it, and finite, as infinities have no difference)
            if (ref == 0.f) ref = both == -INFINITY ? -1.7e38f : both;
          } else {
            // (the output rests: the products of the tile before are done, as the scores' commit came behind them or odone says so)
            fence_after();
            const float next = fmaxf(ref, both), f = ex2(ref - next);
            const uint64_t f2 = pair(f, f);
            ref = next;
            sum2[0] = mul2(sum2[0], f2);
            sum2[1] = mul2(sum2[1], f2);
#pragma unroll 1
            for (int c = 0; c < DP / 2; c += 16) {
              uint32_t o[16];
              ld16(to + c, o);
              wait_ld(o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              st16(to + c, o);
            }
            wait_st();
          }
        }
        const uint64_t nref2 = pair(-ref, -ref);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float2 e = ex2_pair(fma2(pair(r[32 * h + 2 * c], r[32 * h + 2 * c + 1]), sl2, nref2));
            sum2[c & 1] = add2(sum2[c & 1], pair(e.x, e.y));
            pk[c] = pack2<T>(e.x, e.y);
          }
          st16(tp + 16 * h, pk);
        }
        wait_st();
        fence_before();
        bar_arrive(pfull + 8 * u);
        turn ^= 1;
      }
      const float2 a = unpair(add2(sum2[0], sum2[1]));
      joint[half * TILE + r0] = a.x + a.y;
      sync_tile(u);
      const float sum = joint[r0] + joint[TILE + r0], f = 1.f / sum;
      sync_tile(u);
      bar_wait_warp(odone + 8 * u, kApart ? turn ^ 1 : piece, &fault);
      fence_after();
      piece ^= 1;
      const Work w2 = it.work(p, p.kv_heads);
      const Pair x2(w2, it.head(p.kv_heads), p.group);
      const int head = x2.head(u), first = (nu - 1) * TILE + (warp & 3) * 32;      // the warp's first row
      if (half == 0 && first + lane < w2.len) p.lse[(long long)head * p.T + w2.start + first + lane] = ref + log2f(sum);
      store_rows<T>(FromTmem{to}, DP / 2, f, stage + warp * 2048, p.o + ((long long)(w2.start + first) * p.heads + head) * p.D * 2,
                    (long long)p.heads * p.D * 2, w2.len - first, half * (DP / 2), p.D);
      fence_before();      // (the accumulators are read: the next piece's products come behind its first P)
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (fault.raised) drain_after_abort();
  if (warp == 17) tmem_free(tmem, 512);
}

// The kernel below fills the shared memory of an SM to the last kilobyte: what aligning the tiles leaves is checked.
__device__ __forceinline__ bool fits(const char* end, const char* dynamic) {
  unsigned size;
  asm("mov.u32 %0, %dynamic_smem_size;" : "=r"(size));
  return end <= dynamic + size;
}

// ------------------------------------------------------------------ backward
// Both kernels: warps 0-15 hold the tile's rows four times, each a quarter of the 128 columns (P and dS of a quarter go over the
// first half of its scores' columns, so no thread writes where another reads; with eight warps and halves
// 8 x 1024 tokens, 16 heads of 64, take 166 us forward and backward for 161); warp 16 loads, warp 17 issues the products, warp 18
// writes the zeros.  Shared memory: the CTA's own two tiles, three slots of the operand that is used by two products and two of
// the other.  P is made in both (seven products for five): one kernel for all three gradients would add dq with atomics, in an
// order that changes from run to run.  What bounds them is the chain of two products, exponentials and a third product, and the
// ends of the pieces (16 heads of 128, 8192 tokens in sequences of 1024 to 8192: 1.2 us a tile and 39 us in dq, 1.8 us a tile and
// 27 us in dkv; 4 x 2048: dq 110 us, 0.94 PFLOP/s; dkv 124 us, 1.11 PFLOP/s).
constexpr int kRowWarps = 16, kRowThreads = kRowWarps * 32, kBwdThreads = kRowThreads + 96;

// 32 scores of a row: P = exp2(scale S - lse)
__device__ __forceinline__ void probabilities(uint32_t* r, uint64_t sl2, uint64_t nlse2) {
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const float2 e = ex2_pair(fma2(pair(r[2 * c], r[2 * c + 1]), sl2, nlse2));
    r[2 * c] = __float_as_uint(e.x);
    r[2 * c + 1] = __float_as_uint(e.y);
  }
}

// The range of dS.  |P (dP - D)| is at most 2 max|dO_i| max|V_j| (lengths of rows; D is a mean of dP), over the rows that a piece
// multiplies; 2^k brings that bound to 2^14 to 2^15.  A bound by rows' lengths is about sqrt(D) above what dP reaches, which leaves
// 13 bits of normal numbers below a dS of 1/2048 of the largest dP.  Sequences have ranges of their own.  Exact: the power is
// taken out again from fp32 sums.  Only fp16 has it (bf16 has the exponents of fp32).
template <typename T> constexpr bool kRanged = false;
template <> constexpr bool kRanged<__half> = true;
// dkv's own P, the left operand of dV, is kept 2^14 times larger there: a key that many queries give less than 2^-14 each would
// lose bits of its dV (the sums run over up to T such weights).
template <typename T> constexpr int kUp = kRanged<T> ? 14 : 0;

struct Range {
  float o = 0.f, v = 0.f;
  // sizes of tile `u` of the sequence at `at`
  __device__ __forceinline__ void take(const float2* at, int u, bool queries, bool keys) {
    const float2 s = __ldcg(at + (long long)u * TILE);
    if (queries) o = fmaxf(o, s.x);
    if (keys) v = fmaxf(v, s.y);
  }
  // k, from all lanes' tiles
  __device__ __forceinline__ int power() const {
    const float a = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(o)));
    const float b = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
    const float most = 2.f * a * b;
    return most > 0.f ? 14 + 127 - (int)(__float_as_uint(most) >> 23) : 0;
  }
};
__device__ __forceinline__ float power_of_two(int k) { return __uint_as_float((unsigned)(127 + k) << 23); }      // |k| < 127
// dP - D, of the range; nd: -D, of the range already
template <typename T>
__device__ __forceinline__ uint64_t less(uint64_t dp, uint64_t nd, float power) {
  return kRanged<T> ? fma2(dp, pair(power, power), nd) : add2(dp, nd);
}

// The sizes: CTA = a listed tile and a key head, 8 or 16 lanes a row, rows of V behind those of the group's dO.  Rows that hold
// infinities or NaN have no size: what they make of their own dS needs no range.  Reads dO and V once: 8191 tokens, 16 / 4 heads
// of 128, 42 MB; the pass costs that case 18 us of 286 on the device (as much with eight loads in flight, or 1024 threads).
constexpr int kSizesThreads = 512, kSizesLoads = 4;
__global__ void __launch_bounds__(kSizesThreads) attn_sizes(const AttnArgs p) {
  __shared__ float most[2][kSizesThreads / 32];
  dependent_launch();
  if ((int)blockIdx.x >= *(volatile const int*)p.listed * p.kv_heads) return;
  const int4 e = p.list[blockIdx.x / p.kv_heads];
  const int kvh = blockIdx.x % p.kv_heads, first = e.x + e.z * TILE, rows = min(TILE, e.y - e.z * TILE), each = p.group + 1;
  if (e.w) return;
  const int lanes = p.D <= 64 ? 8 : 16, sub = threadIdx.x / lanes, per = kSizesThreads / lanes, col = threadIdx.x % lanes * 8;
  float o = 0.f, v = 0.f;
  for (int i0 = sub; i0 - sub < rows * each; i0 += per * kSizesLoads) {
    uint4 x[kSizesLoads];
#pragma unroll
    for (int j = 0; j < kSizesLoads; ++j) {
      const int i = i0 + j * per, row = i / each, head = i - row * each;
      x[j] = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows && col < p.D) {
        const long long at = head < p.group ? (first + row) * p.dout_t + (kvh * p.group + head) * p.dout_h : (first + row) * p.v_t + kvh * p.v_h;
        x[j] = __ldcg(reinterpret_cast<const uint4*>((head < p.group ? p.dout : p.v) + (at + col) * 2));
      }
    }
#pragma unroll
    for (int j = 0; j < kSizesLoads; ++j) {
      const uint32_t r[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2<__half>(r[k]);
        s = fmaf(f.x, f.x, fmaf(f.y, f.y, s));
      }
      for (int d = lanes / 2; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (s < INFINITY) {
        if ((i0 + j * per) % each < p.group) o = fmaxf(o, s);
        else v = fmaxf(v, s);
      }
    }
  }
  o = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(o)));
  v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
  if (threadIdx.x % 32 == 0) {
    most[0][threadIdx.x / 32] = o;
    most[1][threadIdx.x / 32] = v;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < kSizesThreads / 32; ++i) {
    o = fmaxf(o, most[0][i]);
    v = fmaxf(v, most[1][i]);
  }
  p.sizes[(long long)kvh * p.T + first] = make_float2(sqrtf(o), sqrtf(v));
}

// At DP = 64 there is room for the outputs' way out beside the tiles; else it leads through the second own tile (dO or V), whose
// next load waits; the first one's (Q or K) does not.
template <int DP> constexpr bool kRoom = DP == 64;

// A tile of queries against its keys: S = Q K^T, dP = dO V^T, dQ += dS K.
template <typename T, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dq(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
        const __grid_constant__ CUtensorMap mdo, const AttnArgs p) {
  constexpr int ATOMS = DP / 64, TB = ATOMS * kAtom;
  extern __shared__ char smem_raw[];
  __shared__ __align__(8) unsigned long long bars[21];
  __shared__ float part[2][TILE];
  __shared__ uint32_t tmem_;
  __shared__ Fault fault;
  char* const smem_p = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem = smem_u32(smem_p), bar0 = smem_u32(bars);
  const uint32_t qfull = bar0, kfull = bar0 + 8, kempty = bar0 + 32, vfull = bar0 + 56, vempty = bar0 + 72, sfull = bar0 + 88,
                 dpfull = bar0 + 104, dsfull = bar0 + 112, done = bar0 + 120, ready = bar0 + 128, qempty = bar0 + 144, gfull = bar0 + 152, gempty = bar0 + 160;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == kRowWarps + 1) tmem_alloc(smem_u32(&tmem_), 512);
  if (warp == 0) {
    if (lane == 31) {
      fault.raised = 0;
      fault.status = p.status;
    }
    // (a lane a barrier; the slots of K and V are freed by the products and by the zeros' warp)
    const int count = (lane >= 4 && lane < 7) || lane == 9 || lane == 10 ? 2 : lane == 14 ? kRowThreads : lane == 20 && !kRoom<DP> ? kRowWarps : 1;
    if (lane < 21) bar_init(bar0 + 8 * lane, count);
    bar_init_done();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_;
  dependent_launch();
  const int total = *(volatile const int*)p.listed * p.heads;
  if (p.split > 1)
    for (int i = blockIdx.x * kBwdThreads + threadIdx.x; i < p.pieces; i += gridDim.x * kBwdThreads) p.arrived[i] = 0;
  const uint32_t sq = smem, sdo = smem + TB, sk = smem + 2 * TB, sv = smem + 5 * TB;
  const uint32_t tdp = tmem + 2 * TILE, tdq = tmem + 3 * TILE;
  // tile of queries, and tiles of keys, of a piece
  const auto tiles_of = [](const Work& w) { return (w.len + TILE - 1) / TILE - w.unit; };

  if (warp == kRowWarps) {
    const bool one = elect();
    const auto load_tile = [&](uint32_t dst, const CUtensorMap* m, int row, int h, uint32_t bar) {
      if (one) {
        bar_expect(bar, TB);
#pragma unroll
        for (int a = 0; a < ATOMS; ++a) load3(dst + a * kAtom, m, 64 * a, row, h, bar);
      }
      __syncwarp();
    };
    bool ok = true;
    int g = 0, pieces = 0;
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, p.heads);
      const int head = it.head(p.heads), kvh = head / p.group, n = tiles_of(w);
      if (w.nothing) continue;
      // (dO comes last: its place may be taken by the last piece's way out)
      for (int i = -1; i < n; ++i) {
        if (i >= 0) {
          if (!(ok = bar_wait_warp(vempty + 8 * (g & 1), ((g >> 1) & 1) ^ 1, &fault))) break;
          load_tile(sv + (g & 1) * TB, &mv, w.start + i * TILE, kvh, vfull + 8 * (g & 1));
          ++g;
        }
        if (i + 1 < n) {
          if (!(ok = bar_wait_warp(kempty + 8 * (g % 3), ((g / 3) & 1) ^ 1, &fault))) break;
          load_tile(sk + g % 3 * TB, &mk, w.start + (i + 1) * TILE, kvh, kfull + 8 * (g % 3));
        }
        if (i < 0) {
          if (!(ok = bar_wait_warp(qempty, (pieces & 1) ^ 1, &fault))) break;
          load_tile(sq, &mq, w.start + (n - 1) * TILE, head, qfull);
        } else if (i == 0) {
          if (!(ok = bar_wait_warp(gempty, (pieces++ & 1) ^ 1, &fault))) break;
          load_tile(sdo, &mdo, w.start + (n - 1) * TILE, head, gfull);
        }
      }
    }
  } else if (warp == kRowWarps + 2) {
    bool ok = true;
    int g = 0;
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, p.heads);
      const int n = tiles_of(w);
      if (w.nothing) continue;
      for (int i = 0; i < n; ++i, ++g) {
        const int s3 = g % 3, s2 = g & 1;
        if (!(ok = bar_wait_warp(kfull + 8 * s3, (g / 3) & 1, &fault) && bar_wait_warp(vfull + 8 * s2, (g >> 1) & 1, &fault))) break;
        if (i == n - 1 && n * TILE > w.len) {
          zero_rows(smem_p + 2 * TB + s3 * TB, ATOMS, w.len - i * TILE);
          zero_rows(smem_p + 5 * TB + s2 * TB, ATOMS, w.len - i * TILE);
        }
        if (lane == 0) {
          bar_arrive(ready + 8 * s2);
          bar_arrive(kempty + 8 * s3);
          bar_arrive(vempty + 8 * s2);
        }
      }
    }
  } else if (warp == kRowWarps + 1) {
    const bool one = elect();
    const int ksteps = (p.D + 15) / 16;
    const uint32_t dscore = product_desc<T>(TILE, TILE, false, false);
    const uint32_t dout = product_desc<T>(TILE, ksteps * 16, false, true);
    const uint64_t aq = operand(sq), ado = operand(sdo), k0 = operand(sk), v0 = operand(sv), kt0 = operand(sk, kAtom);
    const auto product = [&](uint32_t acc, uint64_t a, uint64_t b) {
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < ksteps) mma_ss(acc, along(a, k), along(b, k), dscore, k > 0);
    };
    bool ragged = false;
    // scores of the tile that comes as number i, over the dS of number i - 2
    const auto scores = [&](int i) {
      const int s3 = i % 3;
      // (as in the forward pass: the load of V comes behind the zeros' warp's last turn in the slot of `ready`; K's need not)
      if (!(ragged ? bar_wait_warp(vfull + 8 * (i & 1), (i >> 1) & 1, &fault) && bar_wait_warp(ready + 8 * (i & 1), (i >> 1) & 1, &fault)
                   : bar_wait_warp(kfull + 8 * s3, (i / 3) & 1, &fault))) return false;
      if (one) {
        product(tmem + (i & 1) * TILE, aq, k0 + (uint64_t)(s3 * (TB >> 4)));
        commit(sfull + 8 * (i & 1));
      }
      __syncwarp();
      return true;
    };
    const auto dprobs = [&](int i) {
      if (!bar_wait_warp(vfull + 8 * (i & 1), (i >> 1) & 1, &fault)) return false;      // (its scores have waited for the zeros)
      if (one) {
        product(tdp, ado, v0 + (uint64_t)((i & 1) * (TB >> 4)));
        commit(dpfull);
        commit(vempty + 8 * (i & 1));
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    int g = 0, pieces = 0;
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, p.heads);
      const int n = tiles_of(w);
      if (w.nothing) continue;
      ragged = n * TILE > w.len;
      if (!(ok = bar_wait_warp(qfull, pieces & 1, &fault) && scores(g) && bar_wait_warp(gfull, pieces & 1, &fault) && dprobs(g) && (n < 2 || scores(g + 1)))) break;
      ++pieces;
#pragma unroll 1
      for (int i = 0; i < n; ++i, ++g) {
        if (!(ok = bar_wait_warp(dsfull, g & 1, &fault))) break;
        fence_after();
        if (i + 1 < n && !(ok = dprobs(g + 1))) break;
        const uint64_t b = kt0 + (uint64_t)((g % 3) * (TB >> 4));
        if (one) {
#pragma unroll
          for (int k = 0; k < TILE / 16; ++k)
            mma_ts(tdq, tmem + (g & 1) * TILE + (k >> 1) * 32 + (k & 1) * 8, across(b, k), dout, i > 0 || k > 0);
          commit(kempty + 8 * (g % 3));
          if (i + 1 == n) {
            commit(done);
            commit(qempty);
            if (kRoom<DP>) commit(gempty);
          }
        }
        __syncwarp();
        if (i + 2 < n && !(ok = scores(g + 2))) break;
      }
    }
  } else {
    const int quarter = warp >> 2, r0 = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint64_t sl2 = pair(p.scale_log2, p.scale_log2);
    char* const stage = smem_p + (kRoom<DP> ? 7 : 1) * TB + warp * 2048;
    int g = 0, pieces = 0;
    // (as in the forward pass: the warps meet at a barrier for every piece, so none of them leaves)
    for (Walk it; it.next(total);) {
      const Work w = it.work(p, p.heads);
      const int head = it.head(p.heads), n = tiles_of(w), tile = n - 1, row = tile * TILE + r0;
      if (w.nothing) {
        zero_out(p.dq, w.start + tile * TILE, min(TILE, w.len - tile * TILE), p.heads, head, p.D, kRowThreads);
        continue;
      }
      const bool in = row < w.len;
      const long long at = (long long)head * p.T + w.start + row;
      Range range;
      const float2* const sizes = p.sizes + (long long)(head / p.group) * p.T + w.start;
      if (kRanged<T> && lane <= tile) range.take(sizes, lane, lane == tile, true);
      // D.  A piece with one tile of keys has all of P and dP at once and sums them (below): with few keys the rounding of O
      // would weigh (sequences of two tokens, bf16: dQ off by 0.0036 of its norm, 0.0026 like this).  Else D = dO . O, eight rows
      // a warp, a row to kLanes lanes, so that a load takes whole rows.
      constexpr int kLanes = DP / 8, kAtOnce = 32 / kLanes, kSteps = TILE / kRowWarps / kAtOnce;
      if (n > 1) {
        const int col = lane % kLanes * 8;
        uint4 ov[kSteps], gv[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const int tr = tile * TILE + warp * (TILE / kRowWarps) + j * kAtOnce + lane / kLanes;
          ov[j] = gv[j] = make_uint4(0u, 0u, 0u, 0u);
          if (tr < w.len && col < p.D) {
            ov[j] = __ldcg(reinterpret_cast<const uint4*>(p.o + (((long long)(w.start + tr) * p.heads + head) * p.D + col) * 2));
            gv[j] = __ldcg(reinterpret_cast<const uint4*>(p.dout + ((w.start + tr) * p.dout_t + head * p.dout_h + col) * 2));
          }
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const uint32_t av[4] = {ov[j].x, ov[j].y, ov[j].z, ov[j].w}, bv[4] = {gv[j].x, gv[j].y, gv[j].z, gv[j].w};
          float d = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 x = unpack2<T>(av[k]), y = unpack2<T>(bv[k]);
            d = fmaf(x.x, y.x, fmaf(x.y, y.y, d));
          }
#pragma unroll
          for (int o = kLanes / 2; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
          if (lane % kLanes == 0) part[0][warp * (TILE / kRowWarps) + j * kAtOnce + lane / kLanes] = d;
        }
      }
      const float lse = in ? __ldcg(p.lse + at) : 0.f;
      float delta = 0.f;
      const auto meet = [] { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kRowThreads) : "memory"); };
      if (n > 1) {
        meet();
        delta = part[0][r0];
        meet();      // (for the next use)
        if (in && quarter == 0) p.delta[at] = delta;
      }
      float power = 1.f;
      if (kRanged<T>) {
        for (int u = lane + 32; u <= tile; u += 32) range.take(sizes, u, u == tile, true);
        power = power_of_two(range.power());
      }
      const uint64_t nlse2 = pair(-lse, -lse);
#pragma unroll 1
      for (int i = 0; i < n; ++i, ++g) {
        bar_wait_warp(sfull + 8 * (g & 1), (g >> 1) & 1, &fault);
        fence_after();
        const uint32_t ts = tmem + (g & 1) * TILE + quarter * 32 + lanes;
        uint32_t r[32];
        ld32(ts, r);
        wait_ld(r);
        probabilities(r, sl2, nlse2);
        bar_wait_warp(dpfull, g & 1, &fault);
        fence_after();
        uint32_t v[32];
        ld32(tdp + quarter * 32 + lanes, v);
        wait_ld(v);
        if (n == 1) {
          const int last = r0 - quarter * 32;
          float d[2] = {0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 32; ++c) d[c & 1] += c > last ? 0.f : __uint_as_float(r[c]) * __uint_as_float(v[c]);
          // (the quarters' sums: two and two, as shared memory has no room for four)
          d[0] += d[1];
          if (quarter >= 2) part[quarter - 2][r0] = d[0];
          meet();
          if (quarter < 2) d[0] += part[quarter][r0];
          meet();
          if (quarter < 2) part[quarter][r0] = d[0];
          meet();
          delta = part[0][r0] + part[1][r0];
          meet();
          if (in && quarter == 0) p.delta[at] = delta;
        }
        const uint64_t ndelta2 = kRanged<T> ? pair(-delta * power, -delta * power) : pair(-delta, -delta);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float2 t = unpair(mul2(pair(r[2 * c], r[2 * c + 1]), less<T>(pair(v[2 * c], v[2 * c + 1]), ndelta2, power)));
          v[2 * c] = __float_as_uint(t.x);
          v[2 * c + 1] = __float_as_uint(t.y);
        }
        if (i == n - 1) {
          // the last column that the row sees (selected: above the diagonal anything may stand); a row that sees one key has a
          // probability of 1, whatever its score
          const int last = row == 0 ? -1 : r0 - quarter * 32;
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c > last) v[c] = 0u;
        }
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = pack2<T>(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1]));
        st16(ts, v);
        wait_st();
        fence_before();
        bar_arrive(dsfull);
      }
      bar_wait_warp(done, pieces++ & 1, &fault);
      fence_after();
      const int first = tile * TILE + (warp & 3) * 32;
      if (quarter * 32 < DP)
        store_rows<T>(FromTmem{tdq + quarter * 32 + lanes}, 32, kRanged<T> ? p.scale / power : p.scale, stage, p.dq + ((long long)(w.start + first) * p.heads + head) * p.D * 2,
                      (long long)p.heads * p.D * 2, w.len - first, quarter * 32, p.D);
      fence_before();
      if (!kRoom<DP>) {
        fence_async_proxy();      // (the next load comes over what was written there)
        __syncwarp();
        if (lane == 0) bar_arrive(gempty);
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (fault.raised) drain_after_abort();
  if (warp == kRowWarps + 1) tmem_free(tmem, 512);
}

// A tile of keys against the queries that see it, of all heads of the group (or of a share of them): the transposes
// S^T = K Q^T and dP^T = V dO^T, so that dV += P^T dO and dK += dS^T Q have their left operands in tensor memory.
template <typename T, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dkv(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
         const __grid_constant__ CUtensorMap mdo, const AttnArgs p) {
  constexpr int ATOMS = DP / 64, TB = ATOMS * kAtom;
  extern __shared__ char smem_raw[];
  __shared__ __align__(8) unsigned long long bars[21];
  __shared__ __align__(16) float nlse[2][TILE], ndelta[2][TILE];      // of the walked queries: kUp - lse, -D times the next
  __shared__ float power_[2];                                         // the range's power, less kUp
  __shared__ uint32_t tmem_;
  __shared__ Fault fault;
  __shared__ int last_share;
  char* const smem_p = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem = smem_u32(smem_p), bar0 = smem_u32(bars);
  const uint32_t own = bar0, qfull = bar0 + 8, qempty = bar0 + 32, gfull = bar0 + 56, gempty = bar0 + 72, sfull = bar0 + 88,
                 dpfull = bar0 + 96, pfull = bar0 + 104, dsfull = bar0 + 112, done = bar0 + 120, ready = bar0 + 128, free_own = bar0 + 144, vown = bar0 + 152, free_v = bar0 + 160;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == kRowWarps + 1) tmem_alloc(smem_u32(&tmem_), 512);
  if (warp == 0) {
    if (lane == 31) {
      fault.raised = !fits(smem_p + 7 * TB + (kRoom<DP> ? kRowWarps * 2048 : 0), smem_raw);
      fault.status = p.status;
      if (fault.raised) atomicAdd(p.status, 1u);
    }
    // (a lane a barrier: dO arrives with lse and D; slots are freed by the products and by the zeros' warp)
    const int count = lane >= 4 && lane < 11 ? 2 : lane == 13 || lane == 14 ? kRowThreads : lane == 20 && !kRoom<DP> ? kRowWarps : 1;
    if (lane < 21) bar_init(bar0 + 8 * lane, count);
    bar_init_done();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_;
  dependent_launch();
  const int shares = p.kv_heads * p.split, each = p.group / p.split;      // heads of a share
  const int total = *(volatile const int*)p.listed * shares;
  if (fault.raised) {
    __syncthreads();
    if (warp == kRowWarps + 1) tmem_free(tmem, 512);
    return;
  }
  const uint32_t sk = smem, sv = smem + TB, sq = smem + 2 * TB, sg = smem + 5 * TB;
  const uint32_t tdp = tmem + TILE, tdv = tmem + 2 * TILE, tdk = tmem + 3 * TILE;
  const auto tiles_in = [](const Work& w) { return (w.len + TILE - 1) / TILE; };      // tiles of the sequence; the piece's is number `unit`

  if (warp == kRowWarps) {
    const bool one = elect();
    const auto load_tile = [&](uint32_t dst, const CUtensorMap* m, int row, int h, uint32_t bar) {
      if (one) {
        bar_expect(bar, TB);
#pragma unroll
        for (int a = 0; a < ATOMS; ++a) load3(dst + a * kAtom, m, 64 * a, row, h, bar);
      }
      __syncwarp();
    };
    bool ok = true;
    int g = 0, pieces = 0;
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, shares);
      const int share = it.head(shares), kvh = share / p.split, nt = tiles_in(w), n = (nt - w.unit) * each;
      if (w.nothing) continue;
      float power = 1.f;
      for (int i = 0, head = share * each, q = w.unit; i < n; ++i, ++g) {
        const int s3 = g % 3, s2 = g & 1, q0 = q * TILE;
        if (!(ok = bar_wait_warp(qempty + 8 * s3, ((g / 3) & 1) ^ 1, &fault))) break;
        load_tile(sq + s3 * TB, &mq, w.start + q0, head, qfull + 8 * s3);
        if (!(ok = bar_wait_warp(gempty + 8 * s2, ((g >> 1) & 1) ^ 1, &fault))) break;
        load_tile(sg + s2 * TB, &mdo, w.start + q0, head, gfull + 8 * s2);
        if (i == 0) {
          if (!(ok = bar_wait_warp(free_own, (pieces & 1) ^ 1, &fault))) break;
          load_tile(sk, &mk, w.start + w.unit * TILE, kvh, own);
        }
        if (kRanged<T> && i == 0) {
          Range range;
          for (int u = lane; u < nt; u += 32) range.take(p.sizes + (long long)kvh * p.T + w.start, u, u >= w.unit, true);
          power = power_of_two(range.power() - kUp<T>);      // (P has the rest)
        }
        // behind the sequence's end P becomes 0
        if (kRanged<T> && one) power_[s2] = power;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = lane + 32 * j;
          const long long at = (long long)head * p.T + w.start + q0 + r;
          const bool in = q0 + r < w.len;
          nlse[s2][r] = in ? (float)kUp<T> - __ldcg(p.lse + at) : -INFINITY;
          ndelta[s2][r] = in ? -__ldcg(p.delta + at) * power : 0.f;
        }
        __syncwarp();
        if (one) bar_arrive(gfull + 8 * s2);
        if (i == 0) {
          // (V last: its place may be taken by the last piece's way out)
          if (!(ok = bar_wait_warp(free_v, (pieces++ & 1) ^ 1, &fault))) break;
          load_tile(sv, &mv, w.start + w.unit * TILE, kvh, vown);
        }
        if (++q == nt) {
          q = w.unit;
          ++head;
        }
      }
    }
  } else if (warp == kRowWarps + 2) {
    bool ok = true;
    int g = 0;
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, shares);
      const int nt = tiles_in(w), n = (nt - w.unit) * each;
      if (w.nothing) continue;
      for (int i = 0, q = w.unit; i < n; ++i, ++g) {
        const int s3 = g % 3, s2 = g & 1;
        if (!(ok = bar_wait_warp(qfull + 8 * s3, (g / 3) & 1, &fault) && bar_wait_warp(gfull + 8 * s2, (g >> 1) & 1, &fault))) break;
        if (++q == nt) {
          q = w.unit;
          if (nt * TILE > w.len) {
            zero_rows(smem_p + 2 * TB + s3 * TB, ATOMS, w.len - (nt - 1) * TILE);
            zero_rows(smem_p + 5 * TB + s2 * TB, ATOMS, w.len - (nt - 1) * TILE);
          }
        }
        if (lane == 0) {
          bar_arrive(ready + 8 * s2);
          bar_arrive(qempty + 8 * s3);
          bar_arrive(gempty + 8 * s2);
        }
      }
    }
  } else if (warp == kRowWarps + 1) {
    const bool one = elect();
    const int ksteps = (p.D + 15) / 16;
    const uint32_t dscore = product_desc<T>(TILE, TILE, false, false);
    const uint32_t dout = product_desc<T>(TILE, ksteps * 16, false, true);
    const uint64_t ak = operand(sk), av = operand(sv), q0 = operand(sq), g0 = operand(sg), qt0 = operand(sq, kAtom), gt0 = operand(sg, kAtom);
    const auto product = [&](uint32_t acc, uint64_t a, uint64_t b) {
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < ksteps) mma_ss(acc, along(a, k), along(b, k), dscore, k > 0);
    };
    bool ragged = false;
    const auto scores = [&](int i) {
      const int s3 = i % 3;
      // (as in the forward pass: the load of dO comes behind the zeros' warp's last turn in the slot of `ready`; Q's need not)
      if (!(ragged ? bar_wait_warp(gfull + 8 * (i & 1), (i >> 1) & 1, &fault) && bar_wait_warp(ready + 8 * (i & 1), (i >> 1) & 1, &fault)
                   : bar_wait_warp(qfull + 8 * s3, (i / 3) & 1, &fault))) return false;
      if (one) {
        product(tmem, ak, q0 + (uint64_t)(s3 * (TB >> 4)));
        commit(sfull);
      }
      __syncwarp();
      return true;
    };
    const auto dprobs = [&](int i) {
      if (!bar_wait_warp(gfull + 8 * (i & 1), (i >> 1) & 1, &fault)) return false;      // (its scores have waited for the zeros)
      if (one) {
        product(tdp, av, g0 + (uint64_t)((i & 1) * (TB >> 4)));
        commit(dpfull);
      }
      __syncwarp();
      return true;
    };
    const auto outputs = [&](uint32_t acc, uint32_t a, uint64_t b, bool add) {
#pragma unroll
      for (int k = 0; k < TILE / 16; ++k) mma_ts(acc, a + (k >> 1) * 32 + (k & 1) * 8, across(b, k), dout, add || k > 0);
    };
    bool ok = true;
    int g = 0, pieces = 0;
    for (Walk it; ok && it.next(total);) {
      const Work w = it.work(p, shares);
      const int nt = tiles_in(w), n = (nt - w.unit) * each;
      if (w.nothing) continue;
      ragged = nt * TILE > w.len;      // every head's last tile of queries reaches past the sequence
      if (!(ok = bar_wait_warp(own, pieces & 1, &fault) && scores(g) && bar_wait_warp(vown, pieces & 1, &fault) && dprobs(g))) break;
      ++pieces;
#pragma unroll 1
      for (int i = 0; i < n; ++i, ++g) {
        if (!(ok = bar_wait_warp(pfull, g & 1, &fault))) break;
        fence_after();
        if (one) outputs(tdv, tmem, gt0 + (uint64_t)((g & 1) * (TB >> 4)), i > 0);
        __syncwarp();
        if (i + 1 < n && !(ok = scores(g + 1))) break;
        if (!(ok = bar_wait_warp(dsfull, g & 1, &fault))) break;
        fence_after();
        if (one) {
          commit(gempty + 8 * (g & 1));      // dO, lse and D of the tile are no longer read
          outputs(tdk, tdp, qt0 + (uint64_t)((g % 3) * (TB >> 4)), i > 0);
          if (i + 1 == n) {
            commit(done);
            commit(free_own);
            if (kRoom<DP>) commit(free_v);
          }
        }
        __syncwarp();
        if (i + 1 < n && !(ok = dprobs(g + 1))) break;
        if (one) commit(qempty + 8 * (g % 3));
        __syncwarp();
      }
    }
  } else {
    const int quarter = warp >> 2, r0 = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + quarter * 32 + lanes, tp = tdp + quarter * 32 + lanes;
    const uint64_t sl2 = pair(p.scale_log2, p.scale_log2);
    const int first = r0 - quarter * 32;      // on the diagonal: the first column (query) of this quarter that sees the row (key)
    char* const stage = smem_p + (kRoom<DP> ? 7 : 1) * TB + warp * 2048;
    int g = 0, pieces = 0;
    const auto meet = [] { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kRowThreads) : "memory"); };
    // (as in the forward pass: the warps may meet at barriers, so none of them leaves)
    for (Walk it; it.next(total);) {
      const Work w = it.work(p, shares);
      const int share = it.head(shares), kvh = share / p.split, nt = tiles_in(w), tile = w.unit, n = (nt - tile) * each;
      if (w.nothing) {
        if (share % p.split) continue;
        const int rows_here = min(TILE, w.len - tile * TILE);
        zero_out(p.dk, w.start + tile * TILE, rows_here, p.kv_heads, kvh, p.D, kRowThreads);
        zero_out(p.dv, w.start + tile * TILE, rows_here, p.kv_heads, kvh, p.D, kRowThreads);
        continue;
      }
      float power = 1.f;
#pragma unroll 1
      for (int i = 0, q = tile; i < n; ++i, ++g) {
        const float4* l4 = reinterpret_cast<const float4*>(nlse[g & 1] + quarter * 32);
        const float4* d4 = reinterpret_cast<const float4*>(ndelta[g & 1] + quarter * 32);
        const bool diagonal = q == tile;
        if (++q == nt) q = tile;
        bar_wait_warp(gfull + 8 * (g & 1), (g >> 1) & 1, &fault);
        if (kRanged<T>) power = power_[g & 1];
        bar_wait_warp(sfull, g & 1, &fault);
        fence_after();
        uint32_t r[32];
        ld32(ts, r);
        wait_ld(r);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float4 l = l4[c];
          const float2 a = ex2_pair(fma2(pair(r[4 * c], r[4 * c + 1]), sl2, pair(l.x, l.y)));
          const float2 b = ex2_pair(fma2(pair(r[4 * c + 2], r[4 * c + 3]), sl2, pair(l.z, l.w)));
          r[4 * c] = __float_as_uint(a.x);
          r[4 * c + 1] = __float_as_uint(a.y);
          r[4 * c + 2] = __float_as_uint(b.x);
          r[4 * c + 3] = __float_as_uint(b.y);
        }
        if (diagonal) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c < first) r[c] = 0u;
        }
        uint32_t o[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) o[c] = pack2<T>(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]));
        st16(ts, o);
        wait_st();
        fence_before();
        bar_arrive(pfull);
        bar_wait_warp(dpfull, g & 1, &fault);
        fence_after();
        uint32_t v[32];
        ld32(tp, v);
        wait_ld(v);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float4 l = d4[c];
          const float2 a = unpair(mul2(pair(r[4 * c], r[4 * c + 1]), less<T>(pair(v[4 * c], v[4 * c + 1]), pair(l.x, l.y), power)));
          const float2 b = unpair(mul2(pair(r[4 * c + 2], r[4 * c + 3]), less<T>(pair(v[4 * c + 2], v[4 * c + 3]), pair(l.z, l.w), power)));
          v[4 * c] = __float_as_uint(a.x);
          v[4 * c + 1] = __float_as_uint(a.y);
          v[4 * c + 2] = __float_as_uint(b.x);
          v[4 * c + 3] = __float_as_uint(b.y);
        }
        if (diagonal) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c < first) v[c] = 0u;
          if (tile == 0 && quarter == 0) v[0] = 0u;      // (the first query sees one key: its probability is 1)
        }
#pragma unroll
        for (int c = 0; c < 16; ++c) o[c] = pack2<T>(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1]));
        st16(tp, o);
        wait_st();
        fence_before();
        bar_arrive(dsfull);
      }
      bar_wait_warp(done, pieces++ & 1, &fault);
      fence_after();
      // (exact: powers of two)
      const float scale_v = 1.f / (float)(1 << kUp<T>), scale_k = kRanged<T> ? p.scale * scale_v / power : p.scale;
      const int first_row = tile * TILE + (warp & 3) * 32;
      const long long at = ((long long)(w.start + first_row) * p.kv_heads + kvh) * p.D * 2, pitch = (long long)p.kv_heads * p.D * 2;
      // 32 columns of dV and of dK a warp, at DP = 64 of one of them
      constexpr int kOutputs = DP / 64;
      const auto tensor = [&](int k) { return DP == 64 ? quarter >> 1 : k; };
      const int col = DP == 64 ? (quarter & 1) * 32 : quarter * 32;
      if (p.split == 1) {
#pragma unroll
        for (int k = 0; k < kOutputs; ++k) {
          const bool of_k = tensor(k);
          store_rows<T>(FromTmem{(of_k ? tdk : tdv) + col + lanes}, 32, of_k ? scale_k : scale_v, stage, (of_k ? p.dk : p.dv) + at, pitch, w.len - first_row, col, p.D);
        }
      } else {
        const int piece = (int)(it.at() / p.split);
        float* const sums = p.sums + (long long)piece * p.split * 2 * DP * TILE + col * TILE + r0;
#pragma unroll 1
        for (int k = 0; k < kOutputs; ++k) {
          uint32_t r[32];
          __syncwarp();
          FromTmem{(tensor(k) ? tdk : tdv) + col + lanes}(0, r);
          float* const to = sums + (share % p.split * 2 + tensor(k)) * DP * TILE;
#pragma unroll
          for (int c = 0; c < 32; ++c) __stcg(to + c * TILE, __uint_as_float(r[c]));
        }
        // all of the CTA's sums are written before it says so; the last to say so reads all
        __threadfence();
        meet();
        if (threadIdx.x == 0) last_share = atomicAdd(p.arrived + piece, 1) == p.split - 1;
        meet();
        if (last_share) {
          __threadfence();
#pragma unroll 1
          for (int k = 0; k < kOutputs; ++k) {
            const bool of_k = tensor(k);
            const auto summed = [&](int, uint32_t (&r)[32]) {
              float f[32];
#pragma unroll
              for (int c = 0; c < 32; ++c) f[c] = 0.f;
#pragma unroll 1
              for (int j = 0; j < p.split; ++j) {
                const float* from = sums + (j * 2 + of_k) * DP * TILE;
#pragma unroll
                for (int c = 0; c < 32; ++c) f[c] += __ldcg(from + c * TILE);
              }
#pragma unroll
              for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(f[c]);
            };
            store_rows<T>(summed, 32, of_k ? scale_k : scale_v, stage, (of_k ? p.dk : p.dv) + at, pitch, w.len - first_row, col, p.D);
          }
        }
        meet();      // (last_share is read)
      }
      fence_before();
      if (!kRoom<DP>) {
        fence_async_proxy();      // (the next load comes over what was written there)
        __syncwarp();
        if (lane == 0) bar_arrive(free_v);
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (fault.raised) drain_after_abort();
  if (warp == kRowWarps + 1) tmem_free(tmem, 512);
}

// ------------------------------------------------------------------ host side
bool map3(CUtensorMap* m, int dtype, const void* base, long long T, int heads, int D, long long st, long long sh) {
  const unsigned long long d[3] = {(unsigned long long)D, (unsigned long long)T, (unsigned long long)heads};
  const unsigned long long s[2] = {(unsigned long long)st, (unsigned long long)sh};
  return make_map(m, dtype, base, 3, d, s, TILE);
}

// Units (tiles, or pairs of (tile, head)) that T rows in so many sequences can make at most; each sequence has a tile more than
// its rows fill, and there may be rows before the first and behind the last.
long long most_units(long long T, int seqs, bool bounds, int group) {
  long long s = bounds ? seqs + 2ll : 1;
  if (s > T) s = T;
  const long long tiles = T / TILE + s;
  return group ? (tiles * group + s) / 2 : tiles;
}

bool args_ok(int dtype, long long T, int heads, int kv_heads, int D, int seqs, float scale) {
  return (dtype == CHB_BF16 || dtype == CHB_F16) && T >= 1 && T < (1ll << 31) - 2 * TILE && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 &&
         D >= 8 && D % 8 == 0 && D <= 128 && seqs >= 0 && scale > 0.f && scale < INFINITY;
}

AttnArgs common_args(long long T, int heads, int kv_heads, int D, float scale) {
  AttnArgs p{};
  p.T = (int)T;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.D = D;
  p.scale = scale;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = status_word();
  return p;
}

unsigned ctas(long long pieces, int sms) { return (unsigned)(pieces < sms ? pieces : sms); }

template <typename T, int DP>
int run_forward(const CUtensorMap* m, const AttnArgs& p, long long pieces, int sms, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  return launch_big(attn_forward<T, DP>, 6 * DP / 64 * kAtom + 16 * 2048 + 1024, ctas(pieces, sms), kFwdThreads, s, done, m[0], m[1], m[2], p) == cudaSuccess
             ? CHB_SUCCESS : CHB_ERR_CUDA;
}
// Shares of a group's heads in dkv: as many as give every SM four pieces, where there are less than three for two SMs.  Beyond
// that the sums' way through memory costs more than it gives (8191 tokens in 12 sequences, 16 / 4 heads of 128, 248 pieces: 121 us,
// with two shares 134 us; 6000 tokens, 16 / 2 heads, 94 pieces: one share about 560 us by the longest piece, two 334 us, four 305 us).
int head_shares(long long tiles, int kv_heads, int group, int sms) {
  const long long pieces = tiles * kv_heads, want = 2 * pieces >= 3ll * sms ? 1 : (4ll * sms + pieces - 1) / pieces;
  int n = 1;
  for (int d = 2; d <= group && d <= want; ++d)
    if (group % d == 0) n = d;
  return n;
}

struct BackwardWork { float* delta; float2* sizes; int* arrived; float* sums; };
long long backward_layout(char* base, long long T, int heads, int kv_heads, int D, long long tiles, int split, BackwardWork* w) {
  long long at = 0;
  const auto take = [&](long long bytes) {
    char* const r = base ? base + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  w->delta = reinterpret_cast<float*>(take(4 * heads * T));
  w->sizes = reinterpret_cast<float2*>(take(8 * kv_heads * T));      // (few bytes, so bf16 has them too)
  w->arrived = reinterpret_cast<int*>(take(split > 1 ? 4 * tiles * kv_heads : 0));
  w->sums = reinterpret_cast<float*>(take(split > 1 ? tiles * kv_heads * split * 2 * (D <= 64 ? 64 : 128) * TILE * 4 : 0));
  return at;
}

template <typename T, int DP>
int run_backward(const CUtensorMap* m, const AttnArgs& p, long long tiles, int sms, cudaStream_t s) {
  constexpr int kMost = 227 * 1024, kNeed = 7 * DP / 64 * kAtom + (kRoom<DP> ? kRowWarps * 2048 : 0) + 1024;      // (of a CTA, static and dynamic)
  static std::atomic<unsigned long long> done_q{0}, done_kv{0};
  static std::atomic<int> own{0};      // static shared memory of attn_dkv
  if (!own.load(std::memory_order_relaxed)) {
    cudaFuncAttributes f{};
    if (cudaFuncGetAttributes(&f, attn_dkv<T, DP>) != cudaSuccess) return CHB_ERR_CUDA;
    own.store((int)f.sharedSizeBytes, std::memory_order_relaxed);
  }
  const int left = kMost - own.load(std::memory_order_relaxed);
  if (kRanged<T> && launch_overlapped(attn_sizes, dim3((unsigned)(tiles * p.kv_heads)), dim3(kSizesThreads), s, p) != cudaSuccess) return CHB_ERR_CUDA;
  if (launch_big(attn_dq<T, DP>, kNeed, ctas(tiles * p.heads, sms), kBwdThreads, s, done_q, m[0], m[1], m[2], m[3], p) != cudaSuccess ||
      launch_big(attn_dkv<T, DP>, kNeed < left ? kNeed : left, ctas(tiles * p.kv_heads * p.split, sms), kBwdThreads, s, done_kv, m[0], m[1], m[2], m[3], p) != cudaSuccess)
    return CHB_ERR_CUDA;
  return CHB_SUCCESS;
}

}  // namespace
}  // namespace chb

using namespace chb;

extern "C" {

// Bytes of the list of work that the forward pass makes and the backward pass reads.
int chb_attention_plan_bytes(long long T, int group, int seqs, int bounds, long long* out) {
  if (!out || T < 1 || T >= (1ll << 31) - 2 * TILE || group < 1 || seqs < 0) return CHB_ERR_ARG;
  *out = 16 * (kPlanHead + most_units(T, seqs, bounds != 0, group) + most_units(T, seqs, bounds != 0, 0));
  return CHB_SUCCESS;
}

// q [T, heads, D], k and v [T, kv_heads, D] with strides[6] (token and head of each, in elements, multiples of 8; 16-byte aligned);
// cu: seqs + 1 bounds on the device, or null: one sequence.  o [T, heads, D] contiguous, lse [heads, T]; plan: see above.
int chb_attention_forward(int dtype, const void* q, const void* k, const void* v, const long long* strides, long long T, int heads,
                          int kv_heads, int D, const int* cu, int seqs, float scale, void* o, float* lse, void* plan, cudaStream_t stream) {
  if (!args_ok(dtype, T, heads, kv_heads, D, seqs, scale) || !q || !k || !v || !strides || !o || !lse || !plan) return CHB_ERR_ARG;
  if (!on_boundary(16, q, k, v, o, plan) || !on_boundary(8, strides) || !on_boundary(4, cu, lse)) return CHB_ERR_ARG;
  const int group = heads / kv_heads, sms = sm_count();
  const long long pairs = most_units(T, seqs, cu != nullptr, group), tiles = most_units(T, seqs, cu != nullptr, 0);
  if (tiles * heads > 0x7fffffffll) return CHB_ERR_UNSUPPORTED;      // (pieces of work)
  if (!sms) return CHB_ERR_CUDA;
  AttnArgs p = common_args(T, heads, kv_heads, D, scale);
  int4* const list = static_cast<int4*>(plan);
  p.listed = static_cast<const int*>(plan);
  p.list = list + kPlanHead;
  p.o = static_cast<char*>(o);
  p.lse = lse;
  CUtensorMap m[3];
  if (!p.status || !map3(&m[0], dtype, q, T, heads, D, strides[0], strides[1]) || !map3(&m[1], dtype, k, T, kv_heads, D, strides[2], strides[3]) ||
      !map3(&m[2], dtype, v, T, kv_heads, D, strides[4], strides[5])) return CHB_ERR_CUDA;
  if (launch_overlapped(attn_plan, dim3(1), dim3(1024), stream, cu, seqs, (int)T, group, (int)pairs, (int)tiles, list) != cudaSuccess) return CHB_ERR_CUDA;
  const long long n = pairs * kv_heads;
  if (dtype == CHB_F16) return D <= 64 ? run_forward<__half, 64>(m, p, n, sms, stream) : run_forward<__half, 128>(m, p, n, sms, stream);
  return D <= 64 ? run_forward<__nv_bfloat16, 64>(m, p, n, sms, stream) : run_forward<__nv_bfloat16, 128>(m, p, n, sms, stream);
}

int chb_attention_backward_bytes(long long T, int heads, int kv_heads, int D, int bounds, int seqs, long long* out) {
  const int sms = sm_count();
  if (!out || !args_ok(CHB_BF16, T, heads, kv_heads, D, seqs, 1.f)) return CHB_ERR_ARG;
  if (!sms) return CHB_ERR_CUDA;
  const long long tiles = most_units(T, seqs, bounds != 0, 0);
  BackwardWork w;
  *out = backward_layout(nullptr, T, heads, kv_heads, D, tiles, head_shares(tiles, kv_heads, heads / kv_heads, sms), &w);
  return CHB_SUCCESS;
}

// strides[8]: also of dout.  plan: as the forward pass left it.  work: see above; dq, dk, dv contiguous.
int chb_attention_backward(int dtype, const void* q, const void* k, const void* v, const void* o, const void* dout, const long long* strides,
                           const float* lse, const void* plan, long long T, int heads, int kv_heads, int D, int bounds, int seqs, float scale,
                           void* work, void* dq, void* dk, void* dv, cudaStream_t stream) {
  if (!args_ok(dtype, T, heads, kv_heads, D, seqs, scale) || !q || !k || !v || !o || !dout || !strides || !lse || !plan || !work || !dq || !dk || !dv) return CHB_ERR_ARG;
  if (!on_boundary(16, q, k, v, o, dout, plan, work, dq, dk, dv) || !on_boundary(8, strides) || !on_boundary(4, lse)) return CHB_ERR_ARG;
  const int sms = sm_count();
  const long long pairs = most_units(T, seqs, bounds != 0, heads / kv_heads), tiles = most_units(T, seqs, bounds != 0, 0);
  if (tiles * heads > 0x7fffffffll) return CHB_ERR_UNSUPPORTED;
  if (!sms) return CHB_ERR_CUDA;
  AttnArgs p = common_args(T, heads, kv_heads, D, scale);
  p.listed = static_cast<const int*>(plan) + 1;
  p.list = static_cast<const int4*>(plan) + kPlanHead + pairs;
  p.o = static_cast<char*>(const_cast<void*>(o));
  p.lse = const_cast<float*>(lse);
  BackwardWork bw;
  p.split = head_shares(tiles, kv_heads, heads / kv_heads, sms);
  backward_layout(static_cast<char*>(work), T, heads, kv_heads, D, tiles, p.split, &bw);
  p.delta = bw.delta;
  p.sizes = bw.sizes;
  p.v = static_cast<const char*>(v);
  p.v_t = strides[4];
  p.v_h = strides[5];
  p.arrived = bw.arrived;
  p.sums = bw.sums;
  p.pieces = (int)(tiles * kv_heads);
  p.dout = static_cast<const char*>(dout);
  p.dout_t = strides[6];
  p.dout_h = strides[7];
  p.dq = static_cast<char*>(dq);
  p.dk = static_cast<char*>(dk);
  p.dv = static_cast<char*>(dv);
  CUtensorMap m[4];
  if (!p.status || !map3(&m[0], dtype, q, T, heads, D, strides[0], strides[1]) || !map3(&m[1], dtype, k, T, kv_heads, D, strides[2], strides[3]) ||
      !map3(&m[2], dtype, v, T, kv_heads, D, strides[4], strides[5]) || !map3(&m[3], dtype, dout, T, heads, D, strides[6], strides[7])) return CHB_ERR_CUDA;
  if (dtype == CHB_F16) return D <= 64 ? run_backward<__half, 64>(m, p, tiles, sms, stream) : run_backward<__half, 128>(m, p, tiles, sms, stream);
  return D <= 64 ? run_backward<__nv_bfloat16, 64>(m, p, tiles, sms, stream) : run_backward<__nv_bfloat16, 128>(m, p, tiles, sms, stream);
}

}  // extern "C"

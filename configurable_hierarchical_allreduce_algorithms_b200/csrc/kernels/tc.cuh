// What the matrix kernels of the training operators share: bounded waits on shared-memory barriers, tiled loads by
// the bulk-copy engine, and the fifth-generation tensor cores (accumulators and one operand in tensor memory).
//
// Operand tiles.  Every tile is loaded with 128-byte rows and the 128-byte swizzle: `rows` rows of 64 16-bit elements.
// The same bytes serve a product in two ways.  As K-major operand the 64 elements run along the summed axis: groups of
// eight rows are 1024 bytes apart and the next 16 summed elements 32 bytes further.  As MN-major operand the rows run
// along the summed axis: 16 of them are 2048 bytes, and the next 64 elements of the other axis lie one tile further.
//
// Waits.  Every wait ends: after kWaitLimitNs the waiting thread raises the CTA's fault, which ends all other waits of the
// CTA, and counts it in the device's status word, which the host can read.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace chb {
namespace tc {

constexpr unsigned long long kWaitLimitNs = 4000000000ull;

// In shared memory: raised once a wait of the CTA ran out, and where the host finds out.
struct Fault {
  volatile unsigned raised;
  unsigned* status;      // the device's status word: waits of matrix kernels that ran out, since the library was loaded
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// ------------------------------------------------------------------ barriers in shared memory
__device__ __forceinline__ void bar_init(uint32_t bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, unsigned parity) {
  unsigned ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Waits for the phase of the given parity to complete; false: given up (the caller leaves its loops, or goes on without
// waiting).  No function call: one would have to save what a softmax holds in registers.  The timer is read every 256 tries,
// as that takes most of a microsecond.
__device__ __forceinline__ bool bar_wait(uint32_t bar, unsigned parity, Fault* fault) {
  unsigned since = 0;      // (in 2^20 ns; wraps after 52 days)
#pragma unroll 1
  for (unsigned n = 1;; ++n) {
    if (bar_try(bar, parity)) return true;
    if ((n & 255u) == 0) {
      const unsigned now = (unsigned)(now_ns() >> 20);
      if (n == 256) since = now;
      if (fault->raised) return false;
      if (now - since > (unsigned)(kWaitLimitNs >> 20) || n > (1u << 30)) break;
    }
  }
  fault->raised = 1;
  atomicAdd(fault->status, 1u);
  return false;
}
// The same by a whole warp, with one answer for all its lanes (what follows is often a warp-wide instruction).
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, unsigned parity, Fault* fault) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, fault));
}
// True in one lane of a converged warp: the one that issues the warp's products.  The loops around them are left to the
// whole warp, as their operands are kept in registers of the warp.
__device__ __forceinline__ bool elect() {
  unsigned one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}
// End of a CTA whose waits ran out: copies and products already issued end within microseconds; nothing tells when, so
// their shared and tensor memory is kept for a millisecond more.
__device__ __forceinline__ void drain_after_abort() {
  const unsigned long long t0 = now_ns();
  for (int i = 0; i < 100000 && now_ns() - t0 < 1000000ull; ++i) __nanosleep(1000);
}

// ------------------------------------------------------------------ tiled loads
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)m) : "memory");
}
__device__ __forceinline__ void load2(uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"((unsigned long long)m), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void load3(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"((unsigned long long)m), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// shared memory written by ordinary stores becomes visible to products and bulk copies
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ------------------------------------------------------------------ tensor memory
__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, int cols) {      // one warp; blocks until columns are free
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, int cols) {           // the same warp
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Loads from tensor memory have arrived.  The registers pass through here, so that no use of them can be moved ahead.
template <int N>
__device__ __forceinline__ void wait_ld(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: thread l gets / gives lane l
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// ------------------------------------------------------------------ products
// Shared-memory operand: start address, stride between 64-element tiles of the other axis (MN-major only), 1024 bytes
// between groups of eight rows, 128-byte swizzle.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t tile_bytes = 16) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)((tile_bytes >> 4) & 0x3fff) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
template <typename T> struct TypeCode;
template <> struct TypeCode<__half> { static constexpr uint32_t v = 0; };
template <> struct TypeCode<__nv_bfloat16> { static constexpr uint32_t v = 1; };
// fp32 accumulators, M x N tile, operands of type T; a_mn / b_mn: the operand is MN-major
template <typename T>
__host__ __device__ constexpr uint32_t product_desc(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (TypeCode<T>::v << 7) | (TypeCode<T>::v << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// acc[M x N] = (add ? acc : 0) + A[M x 16] B[16 x N]; one thread issues, products of a thread run in issue order
__device__ __forceinline__ void mma_ss(uint32_t acc, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
               ::"r"(acc), "l"(a), "l"(b), "r"(desc), "r"((unsigned)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t acc, uint32_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
               ::"r"(acc), "r"(a), "l"(b), "r"(desc), "r"((unsigned)add) : "memory");
}
// the barrier gets one arrival when all products issued so far by this thread are done
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// ------------------------------------------------------------------ arithmetic
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 operations an instruction; the pairs are neighbouring registers
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float2 ex2_pair(uint64_t x) {
  const float2 v = unpair(x);
  return make_float2(ex2(v.x), ex2(v.y));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);      // a in the low half
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// ------------------------------------------------------------------ host side
unsigned* status_word();      // of the current device; null: no device
int sm_count();               // of the current device; 0: no device

// Lets a kernel have so much dynamic shared memory on the current device: asked for once (a device's bit in `done`, which
// belongs to the kernel), as the question takes as long as a launch.
bool allow_smem(const void* kernel, int bytes, std::atomic<unsigned long long>& done);

// A launch that may start while the one before it drains
template <typename K, typename... A>
inline cudaError_t launch_big(K kernel, int smem, unsigned ctas, int threads, cudaStream_t stream, std::atomic<unsigned long long>& done, const A&... args) {
  if (!allow_smem(reinterpret_cast<const void*>(kernel), smem, done)) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Whether all of these (null included) lie on boundaries of so many bytes: what a kernel reads or writes in words of that size is
// checked before it is launched, as a misaligned word ends the context.
template <typename... P>
inline bool on_boundary(unsigned bytes, const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & (bytes - 1)) == 0;
}

// Tiled view of a 16-bit tensor: `dims` extents from the innermost out, strides in elements (of dims 1..), one box of
// 64 elements x `rows`.  False: the layout cannot be loaded this way.
bool make_map(CUtensorMap* m, int dtype, const void* base, int ndims, const unsigned long long* dims,
              const unsigned long long* strides, unsigned rows);

}  // namespace tc
}  // namespace chb

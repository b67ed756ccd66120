// Host side of the matrix kernels: tensor maps, and the status word in which expired waits are counted.
#include "tc.cuh"

#include <mutex>

#include "../api/chb.h"

namespace chb {
namespace tc {

namespace {
__device__ unsigned int g_status = 0;
__global__ void count_a_fault() { atomicAdd(&g_status, 1u); }

constexpr int kDevices = 64;
std::mutex status_mu;
unsigned status_seen[kDevices];      // what the host was told of

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode() {
  // (looked up in the loaded driver: the library itself is not linked against it and loads on machines without one)
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult st;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &st) != cudaSuccess || st != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}
}  // namespace

bool make_map(CUtensorMap* m, int dtype, const void* base, int ndims, const unsigned long long* dims,
              const unsigned long long* strides, unsigned rows) {
  if (!encode() || ndims < 2 || ndims > 3 || rows > 256) return false;
  cuuint64_t d[3], s[2];
  cuuint32_t box[3] = {64, rows, 1}, one[3] = {1, 1, 1};
  for (int i = 0; i < ndims; ++i) d[i] = dims[i] ? dims[i] : 1;
  for (int i = 0; i + 1 < ndims; ++i) {
    s[i] = strides[i] * 2;
    if (d[i + 1] == 1) s[i] = 16;      // (never taken, but it has to be a legal one)
    if (s[i] % 16 || !s[i]) return false;
  }
  const CUtensorMapDataType t = dtype == CHB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const auto make = [&] {
    return encode()(m, t, (cuuint32_t)ndims, const_cast<void*>(base), d, s, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = make();
  if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
    // (the calling thread has no context yet: a backward pass may be the first thing that autograd's thread does)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return false;
    r = make();
  }
  return r == CUDA_SUCCESS;
}

unsigned* status_word() {
  // (no lock: it could throw through the C entries; two threads that both ask get the same answer)
  static std::atomic<unsigned*> known[kDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return nullptr;
  if (unsigned* p = known[dev].load(std::memory_order_relaxed)) return p;
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_status) != cudaSuccess) return nullptr;
  known[dev].store(static_cast<unsigned*>(p), std::memory_order_relaxed);
  return static_cast<unsigned*>(p);
}

int sm_count() {
  static std::atomic<int> known[kDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return 0;
  if ((n = known[dev].load(std::memory_order_relaxed))) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

bool allow_smem(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (done.load(std::memory_order_relaxed) >> dev & 1) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

}  // namespace tc
}  // namespace chb

// Status of the matrix kernels on the current device (synchronises the stream): 1 if a wait ran out since the last call, else 0.
// The device only counts, and the host remembers how far it has read: a wait that runs out on another stream meanwhile is either
// in what this call reads or left for the next one.
extern "C" int chb_matrix_status(unsigned* out, cudaStream_t stream) try {
  using namespace chb::tc;
  unsigned* p = status_word();
  int dev = 0;
  if (!p || !out || cudaGetDevice(&dev) != cudaSuccess) return CHB_ERR_ARG;
  std::lock_guard<std::mutex> g(status_mu);
  unsigned now = 0;
  if (cudaMemcpyAsync(&now, p, sizeof(unsigned), cudaMemcpyDeviceToHost, stream) != cudaSuccess || cudaStreamSynchronize(stream) != cudaSuccess)
    return CHB_ERR_CUDA;
  *out = now != status_seen[dev];
  status_seen[dev] = now;
  return CHB_SUCCESS;
} catch (...) {
  return CHB_ERR_OTHER;
}

extern "C" int chb_matrix_status_raise(cudaStream_t stream) {
  chb::tc::count_a_fault<<<1, 1, 0, stream>>>();
  return cudaGetLastError() == cudaSuccess ? CHB_SUCCESS : CHB_ERR_CUDA;
}

// The status word of the dense products' kernels.  Their entry points have no handle that could hold one, as a layer has: it is a variable of
// the library, one on each device.
#include "grouped.cuh"

namespace bm {

__device__ int dense_status_word;
static std::atomic<int> g_wait_limit_us{DEFAULT_WAIT_LIMIT_US};

static int status_address(int** out) {
  static std::atomic<int*> known[MAX_DEVICES];
  int dev = -1;
  BM_CUDA(cudaGetDevice(&dev));
  BM_REQUIRE(dev >= 0 && dev < MAX_DEVICES, BM_ERR_UNSUPPORTED, "device ordinal %d out of range", dev);
  int* at = known[dev].load(std::memory_order_acquire);
  if (!at) {
    void* p = nullptr;
    BM_CUDA(cudaGetSymbolAddress(&p, dense_status_word));
    at = static_cast<int*>(p);
    known[dev].store(at, std::memory_order_release);
  }
  *out = at;
  return BM_OK;
}

int dense_guard(DenseGuard* g) {
  g->limit_ns = static_cast<uint64_t>(g_wait_limit_us.load(std::memory_order_relaxed)) * 1000u;
  return status_address(&g->status);
}

}  // namespace bm

using namespace bm;

extern "C" int bm_dense_status(void* stream) {
  int* word = nullptr;
  const int rc = status_address(&word);
  if (rc) return rc;
  int flag = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  BM_CUDA(cudaMemcpyAsync(&flag, word, sizeof(int), cudaMemcpyDeviceToHost, st));
  BM_CUDA(cudaStreamSynchronize(st));
  if (flag != 0) {
    BM_CUDA(cudaMemsetAsync(word, 0, sizeof(int), st));
    return set_error(BM_ERR_TIMEOUT, "a kernel of a dense product gave up a bounded wait; its outputs are undefined");
  }
  return BM_OK;
}

extern "C" int bm_dense_set_wait_limit(int32_t limit_us) {
  BM_REQUIRE(limit_us >= 0 && limit_us <= DEFAULT_WAIT_LIMIT_US, BM_ERR_INVALID_ARG, "dense_set_wait_limit: the wait limit must be 0..%d us", DEFAULT_WAIT_LIMIT_US);
  g_wait_limit_us.store(limit_us, std::memory_order_relaxed);
  return BM_OK;
}

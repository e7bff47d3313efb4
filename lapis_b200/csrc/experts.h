// What the calls of a layer of experts share.
#pragma once
#include <atomic>

#include "kv.h"

namespace lapis_b200 {

constexpr int MAX_EXPERTS = 1024, MAX_CHOSEN = 32;

// Lets a kernel have that much dynamic shared memory, once on every device (the call takes half a microsecond).
template <auto KERNEL>
int allow_smem(int bytes) {
  static std::atomic<uint64_t> allowed{0};
  int device = 0;
  LAPIS_CUDA_TRY(cudaGetDevice(&device));
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (allowed.load(std::memory_order_relaxed) & bit) return LAPIS_OK;
  LAPIS_CUDA_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return LAPIS_OK;
}

// Memory of a call that is given back when it returns.  What the pool did not serve is freed in the mode in which another thread may capture a
// stream meanwhile; in the others cudaFree fails and ends that capture.
struct CallBuf : PoolBuf {
  ~CallBuf() {
    if (pooled || p == nullptr) return;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    cudaFree(p);
    cudaThreadExchangeStreamCaptureMode(&mode);
    p = nullptr;
    pooled = true;
  }
};

// Scratch memory of a call.  The first one of a process makes the pool that it comes from, which a stream that is captured allows in this mode
// only.  What the pool does not serve is freed when the call returns, so a graph may not have it.
inline int scratch(CallBuf *buf, size_t bytes, cudaStream_t st) {
  if (bytes > POOL_LARGEST) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    LAPIS_CUDA_TRY(cudaStreamIsCapturing(st, &capture));
    if (capture != cudaStreamCaptureStatusNone) return fail(LAPIS_ETOOBIG, "%zu bytes of scratch memory under stream capture", bytes);
  }
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  LAPIS_CUDA_TRY(cudaThreadExchangeStreamCaptureMode(&mode));
  const int status = buf->alloc(bytes, st);
  cudaThreadExchangeStreamCaptureMode(&mode);
  return status;
}

int check_expert_lists(const char *what, const lapis_b200_expert_lists *lists);  // experts.cu; 0 or a recorded error

}  // namespace lapis_b200

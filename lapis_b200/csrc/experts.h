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

int check_expert_lists(const char *what, const lapis_b200_expert_lists *lists);  // experts.cu; 0 or a recorded error

}  // namespace lapis_b200

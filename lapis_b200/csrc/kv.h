// What the kernels around attention share: element types, page lists and the places of tokens in a paged cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>

#include "common.h"

namespace lapis_b200 {

// Widest head of the entry points.
constexpr int KV_MAX_DIM = 256;

inline int type_bytes(int type) { return type == LAPIS_F32 ? 4 : type == LAPIS_F16 || type == LAPIS_BF16 ? 2 : 1; }
inline bool is_float_type(int type) { return type == LAPIS_F32 || type == LAPIS_F16 || type == LAPIS_BF16; }
#ifdef __CUDACC__
__host__ __device__
#endif
inline bool is_quantised(int type) { return type == LAPIS_I8 || type == LAPIS_E4M3; }

// log2 of the slots of a page, or -1: places are shifted instead of divided, where that is the same.
inline int page_shift_of(int64_t page_size) { return (page_size & (page_size - 1)) == 0 ? __builtin_ctzll(page_size) : -1; }

// Checks of the descriptions that the entry points take (rotate.cu); 0 or a recorded error.
int check_cache(const char *what, const lapis_b200_kv_cache *cache);
int check_lists(const char *what, const lapis_b200_page_lists *lists);

#ifdef __CUDACC__
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
// To nearest, ties to even: the one rounding of a result that was computed in 32 bits.
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Codes of a quantised row: x * (largest / amax) to the nearest code, ties to even; the row's scale is amax / largest.
__device__ __forceinline__ float largest_code(int type) { return type == LAPIS_I8 ? 127.0f : 448.0f; }
// A row whose largest magnitude is below SMALL_ROW is taken times RAISE, a power of two: 127 / amax is no number of 32 bits where amax
// is below 3.7e-37, 448 / amax below 1.3e-36.  The products are the same numbers.
constexpr float SMALL_ROW = 0x1p-63f, RAISE = 0x1p64f;
// A row that is not finite reads as NaN, whatever its codes are.
__device__ __forceinline__ float scale_of(float amax, float largest) { return amax < INFINITY ? amax / largest : NAN; }
__device__ __forceinline__ int8_t to_i8(float x) {
  const float r = rintf(fminf(fmaxf(x, -127.0f), 127.0f));  // a NaN becomes -127; its row's scale is NaN
  return (int8_t)(int)r;
}
__device__ __forceinline__ uint8_t to_e4m3(float x) { return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float from_e4m3(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}
// The larger of two; a NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two products and sums in 32 bits by one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// An element of a cache or of a dense array whose type is known at run time only.
__device__ __forceinline__ float load_as_f32(const void *p, int64_t i, int type) {
  switch (type) {
    case LAPIS_F32: return static_cast<const float *>(p)[i];
    case LAPIS_F16: return __half2float(static_cast<const __half *>(p)[i]);
    case LAPIS_BF16: return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    case LAPIS_I8: return (float)static_cast<const int8_t *>(p)[i];
    default: return from_e4m3(static_cast<const uint8_t *>(p)[i]);
  }
}

__device__ __forceinline__ int64_t load_index(const void *p, int64_t i, int bytes) {
  return bytes == 4 ? (int64_t)static_cast<const int32_t *>(p)[i] : static_cast<const int64_t *>(p)[i];
}

// Row of the cache (as [pages * heads * page_size, dim]) that holds head 0 of the token at `place` of request `row`, or -1
// where the lists name none (page_shift: page_shift_of, or -1): what the lists say is checked, as nothing on the host has seen it.
__device__ __forceinline__ int64_t cache_row(const lapis_b200_kv_cache &cache, const lapis_b200_page_lists &lists, int64_t row, int64_t place, int page_shift) {
  if (row < 0 || row >= lists.rows || place < 0) return -1;
  const int64_t nth = page_shift >= 0 ? place >> page_shift : place <= 0x7fffffff ? (int64_t)((uint32_t)place / (uint32_t)cache.page_size) : place / cache.page_size;
  const int64_t entry = load_index(lists.d_pos, row, lists.idx_bytes) + nth;
  if (entry < 0 || entry >= load_index(lists.d_pos, row + 1, lists.idx_bytes) || entry >= lists.entries) return -1;
  const int64_t page = load_index(lists.d_crd, entry, lists.idx_bytes);
  if (page < 0 || page >= cache.pages) return -1;
  return page * cache.heads * cache.page_size + (place - nth * cache.page_size);
}
#endif

}  // namespace lapis_b200

// What the kernels of the products with 4-bit weights share: the order of the weights, the operands, codes to numbers.
#pragma once
#include <cstdint>
#include <type_traits>

#include "experts.h"

namespace lapis_b200 {

constexpr int STRIP = 16, BLOCK = 64, BATCH = 256;  // outputs of a strip; columns of a lane's load, and of a record of scales

struct ProductArgs {
  const uint8_t *codes, *records;
  int zeros_at, record_bytes;  // zeros_at: in a record, or 0 for none
  int scale_type, gated, experts;
  int strips, blocks, batches;
  int outputs;  // of the result
  int64_t columns;
  const void *x;
  int64_t x_stride, x_rows;  // x_rows: rows that x has
  int64_t rows;              // of the result
  const int32_t *pos, *crd;  // lists, or null
  int k, fetch;
  int wide;           // rows of x begin at multiples of 16 bytes
  int rows_a_pass, strips_log;  // of int4_few_kernel
  int chunk;  // columns of x in shared memory
  int shares_log;  // of int4_many_kernel: CTAs of a cluster that share a tile's columns
  uint8_t *arranged;
  int *error_flag;
  void *y;
};

// Columns of the product (rows, three for one of 32 bits) up to which it goes to int4_few_kernel, where a second product for the next eight
// would do: 16 rows x 14,336 x 4096 took it 36 us, int4_many_kernel takes 21, as for 9; 8 rows take it 17.
constexpr int FEW_COLUMNS = 8;
int launch_few(int type, ProductArgs &a, int group, int matrices, cudaStream_t st);                     // int4_few.cu
int launch_many(int type, ProductArgs &a, int group, int matrices, int64_t expected, cudaStream_t st);  // int4_many.cu

#ifdef __CUDACC__

// Codes to whole numbers of 16 bits, exactly.  A code's bits behind those of a number 2^m are 2^m + code or, four places up, 2^m + 16
// code (used for weights of 8 and 4 bits by Y. J. Kim et al., "Who Says Elephants Can't Run", 2022); fp16 has room for both (1024), bf16 for one (128).  So of the four pairs of a word, fp16 takes two as they lie and two shifted
// once, and the zero is subtracted by the instruction that brings a code down.  What bounds the conversion are the instructions
// on 32 bits, one every two cycles: five for eight codes, in bf16 seven.
template <typename T>
struct Zero;  // of a row's group
template <>
struct Zero<__half> {
  uint32_t low, high;  // -(1024 + zero), -(64 + zero), twice each
  __device__ __forceinline__ void set(uint32_t zero) { low = 0xe400e400u | zero * 0x10001u, high = 0xd400d400u | zero * 0x100010u; }
};
template <>
struct Zero<__nv_bfloat16> {
  uint32_t low;  // -(128 + zero)
  __device__ __forceinline__ void set(uint32_t zero) { low = 0xc300c300u | zero * 0x10001u; }
};
// Columns 2p and 2p + 1 of a word of codes, p = 0 to 3, less the zero.
__device__ __forceinline__ void pairs_of(uint32_t (&d)[4], uint32_t word, const Zero<__half> &zero) {
  const uint32_t next = word >> 8;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t w = p < 2 ? word : next;
    if (p % 2 == 0) asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d[p]) : "r"((w & 0x000f000fu) | 0x64006400u), "r"(zero.low));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d[p]) : "r"((w & 0x00f000f0u) | 0x64006400u), "r"(0x2c002c00u), "r"(zero.high));
  }
}
__device__ __forceinline__ void pairs_of(uint32_t (&d)[4], uint32_t word, const Zero<__nv_bfloat16> &zero) {
#pragma unroll
  for (int p = 0; p < 4; ++p) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d[p]) : "r"((word >> 4 * p & 0x000f000fu) | 0x43004300u), "r"(0x3f803f80u), "r"(zero.low));
}
#endif

}  // namespace lapis_b200

// Few rows times weights of 4 bits with a scale (and a zero) for every group of columns.
//
//   y[r, n] = sum over groups of  scale[n, group] * sum over the group's columns of (code[n, c] - zero[n, group]) x[r, c]
//
// code - zero is a whole number between -15 and 15, exact in bf16 and fp16; so is x (32 bits: three parts of bf16, three columns of
// the product); their products are added in 32 bits on the tensor cores, a group's sum is scaled in 32 bits, and the result
// is rounded once.  With `gated` outputs the two halves of the result meet in a lane, silu(gate) * up, in 32 bits.
//
// The work is to read the weights once.  They lie in the order in which a warp takes them: a strip of 16 outputs, 64 columns of
// it in one 16-byte load a lane, which is the A operand of four products of 16 x 8 x 16.  The rows x are the B operand, from
// shared memory.  The columns of a product may come in any order, the same for A and B: the lane of a row takes 8 that lie
// next to one another in each half of the 64, so that it has its part of x in two 16-byte loads.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "experts.h"

namespace lapis_b200 {

constexpr int STRIP = 16, BLOCK = 64, BATCH = 256;  // outputs of a strip; columns of a lane's load, and of a record of scales
constexpr int INT4_WARPS = 8, INT4_THREADS = 32 * INT4_WARPS;

struct Int4Layout {
  int64_t strips, blocks, batches;          // of one matrix
  int64_t scale_bytes, record_bytes;        // of a strip's batch: its scales, and with its zeros behind them
  int64_t records_at, bytes;                // in d_packed
};
static Int4Layout layout_of(const lapis_b200_int4 &w) {
  Int4Layout l;
  l.strips = w.gated ? (w.outputs / 2 + 7) / 8 : (w.outputs + STRIP - 1) / STRIP;
  l.blocks = (w.columns + BLOCK - 1) / BLOCK;
  l.batches = (w.columns + BATCH - 1) / BATCH;
  const int groups = BATCH / w.group;
  l.scale_bytes = STRIP * groups * (w.scale_type == LAPIS_F32 ? 4 : 2);
  l.record_bytes = l.scale_bytes + (w.zeros ? STRIP * groups / 2 : 0);
  const int64_t strips = w.experts * l.strips;
  l.records_at = strips * l.blocks * 512;
  l.bytes = l.records_at + strips * l.batches * l.record_bytes;
  return l;
}

// ---- laying out -------------------------------------------------------------------

struct PackArgs {
  int64_t outputs, columns, strips, blocks, batches, items;
  int group, gated, scale_bytes;  // of one scale
  int zeros_at, record_bytes;
  const uint8_t *codes, *zero;
  const void *scale;
  uint8_t *packed_codes, *records;
};
// Output of row r of a strip, or -1.  Gated: rows 0 to 7 are gates, 8 to 15 what they are for.
__device__ __forceinline__ int64_t output_of(const PackArgs &a, int64_t strip, int r) {
  if (!a.gated) return strip * STRIP + r < a.outputs ? strip * STRIP + r : -1;
  const int64_t half = a.outputs / 2, n = strip * 8 + r % 8;
  return n >= half ? -1 : r < 8 ? n : half + n;
}
// A thread a lane's 16 bytes.
__global__ void __launch_bounds__(256) pack_codes_kernel(const __grid_constant__ PackArgs a) {
  const int64_t bytes = (a.columns + 1) / 2;
  for (int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; item < a.items; item += (int64_t)gridDim.x * blockDim.x) {
    const int lane = item % 32;
    const int64_t block = item / 32 % a.blocks, strip = item / 32 / a.blocks, expert = strip / a.strips;
    uint32_t word[4];
    for (int i = 0; i < 4; ++i) {
      const int64_t n = output_of(a, strip % a.strips, lane / 4 + i / 2 * 8);
      const int64_t first = block * BLOCK + i % 2 * 32 + lane % 4 * 8;
      word[i] = 0;
      for (int v = 0; v < 8; ++v) {  // columns 2p and 2p + 1 in halves of 4 bits p and p + 4
        if (n < 0 || first + v >= a.columns) continue;
        const uint32_t code = a.codes[(expert * a.outputs + n) * bytes + (first + v) / 2] >> (first + v) % 2 * 4 & 15;
        word[i] |= code << (v / 2 * 4 + v % 2 * 16);
      }
    }
    reinterpret_cast<uint4 *>(a.packed_codes)[item] = make_uint4(word[0], word[1], word[2], word[3]);
  }
}
// A thread a lane's row of scales and zeros: [rows r and r + 8 of the strip][groups of the batch].
__global__ void __launch_bounds__(256) pack_scales_kernel(const __grid_constant__ PackArgs a) {
  const int groups = BATCH / a.group;
  const int64_t all = (a.columns + a.group - 1) / a.group;
  for (int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; item < a.items; item += (int64_t)gridDim.x * blockDim.x) {
    const int r = item % 8;
    const int64_t batch = item / 8 % a.batches, strip = item / 8 / a.batches, expert = strip / a.strips;
    uint8_t *const record = a.records + item / 8 * a.record_bytes;
    uint64_t zeros = 0;
    for (int i = 0; i < 2 * groups; ++i) {
      const int64_t n = output_of(a, strip % a.strips, r + i / groups * 8), group = batch * groups + i % groups;
      const bool there = n >= 0 && group < all;
      const int64_t from = (expert * a.outputs + n) * all + group;
      const int to = r * 2 * groups + i;
      if (a.scale_bytes == 4) reinterpret_cast<uint32_t *>(record)[to] = there ? static_cast<const uint32_t *>(a.scale)[from] : 0;
      else reinterpret_cast<uint16_t *>(record)[to] = there ? static_cast<const uint16_t *>(a.scale)[from] : 0;
      if (a.zero != nullptr && there) zeros |= (uint64_t)(a.zero[from] & 15) << i * 4;
    }
    if (a.zero != nullptr)
      for (int b = 0; b < groups; ++b) record[a.zeros_at + r * groups + b] = (uint8_t)(zeros >> b * 8);
  }
}

struct QuantiseArgs {
  const void *w;
  int64_t w_stride, columns, groups, items;
  int group, scale_type;
  uint8_t *codes, *zero;
  void *scale;
};
// A warp a group, a lane two neighbouring columns at a time.
template <typename T>
__global__ void __launch_bounds__(256) quantise_kernel(const __grid_constant__ QuantiseArgs a) {
  const int lane = threadIdx.x % 32;
  for (int64_t item = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; item < a.items; item += (int64_t)gridDim.x * 8) {
    const int64_t row = item / a.groups, first = item % a.groups * a.group;
    const T *const w = static_cast<const T *>(a.w) + row * a.w_stride + first;
    const int n = (int)min((int64_t)a.group, a.columns - first);
    float low = 0.0f, high = 0.0f, x[4];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 2 * lane + i / 2 * 64 + i % 2;
      x[i] = c < n ? to_f32(w[c]) : 0.0f;
      finite = finite && fabsf(x[i]) < INFINITY;
      low = fminf(low, x[i]);
      high = fmaxf(high, x[i]);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, d));
      high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
    }
    finite = __all_sync(0xffffffffu, finite);
    // Halves first: the range of two finite numbers may be none of 32 bits.
    float scale = !finite ? NAN : a.zero == nullptr ? fmaxf(-low, high) / 7.0f : (0.5f * high - 0.5f * low) / 7.5f;
    if (a.scale_type == LAPIS_F16) {
      const __half s = __float2half_rn(scale);
      if (lane == 0) static_cast<__half *>(a.scale)[item] = s;
      scale = __half2float(s);
    } else if (a.scale_type == LAPIS_BF16) {
      const __nv_bfloat16 s = __float2bfloat16_rn(scale);
      if (lane == 0) static_cast<__nv_bfloat16 *>(a.scale)[item] = s;
      scale = __bfloat162float(s);
    } else if (lane == 0) {
      static_cast<float *>(a.scale)[item] = scale;
    }
    const bool usable = scale > 0.0f && scale < INFINITY;
    const float zero = a.zero == nullptr ? 8.0f : usable ? fminf(rintf(-low / scale), 15.0f) : 0.0f;
    if (a.zero != nullptr && lane == 0) a.zero[item] = (uint8_t)zero;
    uint8_t *const to = a.codes + row * ((a.columns + 1) / 2) + first / 2;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const int c = 2 * lane + i * 32;
      if (c >= n) continue;
      uint32_t byte = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float q = usable ? rintf(x[i + h] / scale) + zero : zero;
        q = fminf(fmaxf(q, a.zero == nullptr ? 1.0f : 0.0f), 15.0f);
        if (c + h < n) byte |= (uint32_t)q << 4 * h;
      }
      to[c / 2] = (uint8_t)byte;
    }
  }
}

// ---- the product --------------------------------------------------------------------

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
  int strips_a_block;  // warps of a block that take a strip each; the others share their columns
  int rows_a_pass, strips_log;  // of int4_few_kernel: strips_log instead of strips_a_block
  int chunk;          // columns of x in shared memory, a multiple of BATCH times the warps that share a strip
  void *y;
};

// Codes to whole numbers of 16 bits, exactly.  A code's bits behind those of a number 2^m are 2^m + code or, four places up, 2^m + 16
// code; fp16 has room for both (1024), bf16 for one (128).  So of the four pairs of a word, fp16 takes two as they lie and two shifted
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
template <typename T>
__device__ __forceinline__ void multiply(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with sums of zero.
template <typename T>
__device__ __forceinline__ void multiply_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// What a lane holds of a batch: 16 columns of rows r and r + 8 in each of four blocks, their scales and zeros.
template <int GROUP>
struct Batch {
  static constexpr int GROUPS = BATCH / GROUP;
  uint4 code[BATCH / BLOCK];
  uint32_t scale[2 * GROUPS];  // 16-bit ones two in a word, in the first half
  uint32_t zero[2];

  template <int N>
  static __device__ __forceinline__ void fetch(uint32_t *to, const uint8_t *from) {
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(from + i * 4);
        to[i] = v.x, to[i + 1] = v.y, to[i + 2] = v.z, to[i + 3] = v.w;
      }
    } else {
      const uint2 v = *reinterpret_cast<const uint2 *>(from);
      to[0] = v.x, to[1] = v.y;
    }
  }
  __device__ __forceinline__ void load(const ProductArgs &a, int64_t strip, int batch, int lane) {
    const uint4 *const codes = reinterpret_cast<const uint4 *>(a.codes) + (strip * a.blocks + batch * (BATCH / BLOCK)) * 32 + lane;
#pragma unroll
    for (int b = 0; b < BATCH / BLOCK; ++b)
      if (batch * (BATCH / BLOCK) + b < a.blocks) code[b] = codes[b * 32];
    if (a.zeros_at != 0) load_record<true>(a, a.records + (strip * a.batches + batch) * a.record_bytes, lane);
    else load_record<false>(a, a.records + (strip * a.batches + batch) * a.record_bytes, lane);
  }
  template <bool ZEROS>
  __device__ __forceinline__ void load_record(const ProductArgs &a, const uint8_t *record, int lane) {
    const int row = lane / 4;
    if (a.scale_type == LAPIS_F32) fetch<2 * GROUPS>(scale, record + row * GROUPS * 8);
    else fetch<GROUPS>(scale, record + row * GROUPS * 4);
    if constexpr (!ZEROS) {
      zero[0] = zero[1] = 0x88888888u;
    } else if constexpr (GROUPS == 8) {
      const uint2 z = reinterpret_cast<const uint2 *>(record + a.zeros_at)[row];
      zero[0] = z.x, zero[1] = z.y;
    } else if constexpr (GROUPS == 4) {
      const uint32_t z = reinterpret_cast<const uint32_t *>(record + a.zeros_at)[row];
      zero[0] = z, zero[1] = z >> 16;
    } else {
      const uint32_t z = reinterpret_cast<const uint16_t *>(record + a.zeros_at)[row];
      zero[0] = z, zero[1] = z >> 8;
    }
  }
  // Scale of group g of row r (0) or r + 8 (1).
  __device__ __forceinline__ float scale_at(int type, int row, int g) const {
    const int i = row * GROUPS + g;
    if (type == LAPIS_F32) return __uint_as_float(scale[i]);
    const uint32_t bits = scale[i / 2] >> i % 2 * 16;
    return type == LAPIS_BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
  }
};

__host__ __device__ constexpr int x_pitch(int chunk) { return chunk * 2 + 64; }  // bytes: two rows' 64 lie on different banks
constexpr int SUM_PITCH = STRIP + 1;

// Copies columns [first, first + n) of rows [row0, row0 + rows) to shared memory, zeros behind the last column.
template <typename X, typename T>
__device__ __forceinline__ void stage(const ProductArgs &a, uint8_t *xs, int64_t row0, int rows, int64_t first, int n) {
  constexpr bool PARTS = std::is_same<X, float>::value;
  constexpr int V = 8;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, pitch = x_pitch(a.chunk);
  for (int r = warp; r < rows; r += INT4_WARPS) {
    int64_t from = row0 + r;
    if (a.fetch) from = a.crd[from] / a.k;
    const bool there = (uint64_t)from < (uint64_t)a.x_rows;
    const X *const x = static_cast<const X *>(a.x) + from * a.x_stride + first;
    for (int c = lane * V; c < n; c += 32 * V) {
      alignas(16) X v[V];
      if (there && a.wide && first + c + V <= a.columns) {
#pragma unroll
        for (int i = 0; i < (int)(V * sizeof(X) / 16); ++i) reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(x + c)[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = there && first + c + i < a.columns ? x[c + i] : from_f32<X>(0.0f);
      }
      if constexpr (!PARTS) {
        *reinterpret_cast<uint4 *>(xs + r * pitch + c * 2) = *reinterpret_cast<const uint4 *>(v);
      } else {
        alignas(16) T part[3][V];
#pragma unroll
        for (int i = 0; i < V; ++i) {  // 8 bits each; what is not finite has one part only
          float left = v[i];
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            part[p][i] = __float2bfloat16_rz(left);  // to nearest, the largest numbers would become infinite
            const float got = to_f32(part[p][i]);
            left = fabsf(got) < INFINITY ? left - got : 0.0f;
          }
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4 *>(xs + (r * 3 + p) * pitch + c * 2) = *reinterpret_cast<const uint4 *>(part[p]);
      }
    }
  }
}

// X: type of x and y; T: of the products; NT: columns of the product, in eights, of one pass over the weights.
template <typename X, typename T, int GROUP, int NT>
__global__ void __launch_bounds__(INT4_THREADS) int4_kernel(const __grid_constant__ ProductArgs a) {
  constexpr bool PARTS = std::is_same<X, float>::value;
  constexpr int A_ROW = PARTS ? 3 : 1, ROWS = 8 * NT / A_ROW;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int strips = a.strips_a_block, shares = INT4_WARPS / strips, my_strip = warp % strips, my_share = warp / strips;
  const int strip = blockIdx.x * strips + my_strip, pitch = x_pitch(a.chunk);
  const int outs = a.gated ? 8 : STRIP;  // of a strip
  const int expert = blockIdx.y;
  X *const y = static_cast<X *>(a.y);
  pdl_wait();
  pdl_release();
  int64_t begin = 0, end = a.rows;
  if (a.pos != nullptr) {
    begin = min((int64_t)max(a.pos[expert], 0), a.rows);
    end = expert < a.experts ? min((int64_t)a.pos[expert + 1], a.rows) : a.rows;
    if (expert == a.experts) {  // rows of no expert
      const int n = min(outs * strips, a.outputs - (int)blockIdx.x * outs * strips);
      for (int64_t i = threadIdx.x; i < (end - begin) * n; i += INT4_THREADS)
        y[(begin + i / n) * a.outputs + blockIdx.x * outs * strips + i % n] = from_f32<X>(0.0f);
      return;
    }
  }
  for (int64_t row0 = begin; row0 < end; row0 += ROWS) {
    const int rows = (int)min((int64_t)ROWS, end - row0), tiles = (rows * A_ROW + 7) / 8;
    float sum[NT][4] = {};
    for (int64_t first = 0; first < a.columns; first += a.chunk) {
      const int n = (int)min((int64_t)a.chunk, (a.columns - first + BLOCK - 1) / BLOCK * BLOCK);
      __syncthreads();
      stage<X, T>(a, smem, row0, rows, first, n);
      __syncthreads();
      if (strip >= a.strips) continue;
      for (int b = my_share; b * BATCH < n; b += shares) {
        const int batch = (int)(first / BATCH) + b;
        Batch<GROUP> w;
        w.load(a, (int64_t)expert * a.strips + strip, batch, lane);
        const uint8_t *const xs = smem + lane / 4 * pitch + b * BATCH * 2 + lane % 4 * 16;
        float part[NT][4] = {};
#pragma unroll
        for (int half = 0; half < 2 * BATCH / BLOCK; ++half) {
          const int g = half * 32 / GROUP;
          if (batch * (BATCH / BLOCK) + half / 2 < a.blocks) {
            const uint4 c = w.code[half / 2];
            const uint32_t top = half % 2 ? c.y : c.x, low = half % 2 ? c.w : c.z;
            Zero<T> z0, z1;
            z0.set(w.zero[0] >> 4 * g & 15);
            z1.set(w.zero[1] >> 4 * g & 15);
            uint32_t p0[4], p1[4];
            pairs_of(p0, top, z0);
            pairs_of(p1, low, z1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if (t >= tiles) break;
              const uint4 v = *reinterpret_cast<const uint4 *>(xs + t * 8 * pitch + half * 64);
              multiply<T>(part[t], p0[0], p1[0], p0[1], p1[1], v.x, v.y);
              multiply<T>(part[t], p0[2], p1[2], p0[3], p1[3], v.z, v.w);
            }
          }
          if ((half + 1) * 32 % GROUP == 0) {
            const float s0 = w.scale_at(a.scale_type, 0, g), s1 = w.scale_at(a.scale_type, 1, g);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                sum[t][i] = fmaf(i < 2 ? s0 : s1, part[t][i], sum[t][i]);
                part[t][i] = 0.0f;
              }
            }
          }
        }
      }
    }
    // The shares' sums meet in shared memory: [share][strip][column][row].
    float *const sums = reinterpret_cast<float *>(smem);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sums[((my_share * strips + my_strip) * 8 * NT + t * 8 + lane % 4 * 2 + i % 2) * SUM_PITCH + lane / 4 + i / 2 * 8] = sum[t][i];
    __syncthreads();
    const auto total = [&](int s, int r, int n) {
      float v = 0.0f;
      for (int p = A_ROW - 1; p >= 0; --p)  // the small parts first
        for (int share = 0; share < shares; ++share) v += sums[((share * strips + s) * 8 * NT + r * A_ROW + p) * SUM_PITCH + n];
      return v;
    };
    for (int i = threadIdx.x; i < rows * strips * outs; i += INT4_THREADS) {
      const int n = i % (strips * outs), r = i / (strips * outs), s = n / outs, to = blockIdx.x * strips * outs + n;
      if (to >= a.outputs) continue;
      float v = total(s, r, n % outs);
      if (a.gated) v = v / (1.0f + expf(-v)) * total(s, r, n % outs + 8);
      y[(row0 + r) * a.outputs + to] = from_f32<X>(v);
    }
  }
}


// ---- few rows: the weights as fast as they come --------------------------------------

constexpr int FEW_WARPS_LOG = 2, FEW_WARPS = 1 << FEW_WARPS_LOG, FEW_THREADS = 32 * FEW_WARPS;
constexpr int FEW_BLOCKS = 5, FEW_ROOM = 40 << 10;  // blocks of an SM, and the rows x of each in shared memory

// Bytes of a row of x in shared memory: neighbouring rows' pieces of a phase lie on different banks.
__host__ __device__ constexpr int few_pitch(int columns) { return columns * 2 + 64; }

// Columns [first, first + n) of `rows` rows to shared memory, zeros behind the last column; of 32-bit values three parts of 8 bits each.
template <typename X>
__device__ __forceinline__ void stage_few(const ProductArgs &a, uint8_t *xs, const X *const *row_at, int rows, int first, int n, int pitch) {
  constexpr int V = 8;
  const int columns = (int)a.columns;
  for (int r = 0; r < rows; ++r) {
    const X *const x = row_at[r];
    if (sizeof(X) == 2 && a.wide && x != nullptr && first + n <= columns) {
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(xs) + r * pitch;
      for (int c = threadIdx.x * V; c < n; c += FEW_THREADS * V) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + c * 2), "l"(x + first + c) : "memory");
      continue;
    }
    for (int c = threadIdx.x * V; c < n; c += FEW_THREADS * V) {
      const int there = x == nullptr ? 0 : max(0, min(V, columns - first - c));
      alignas(16) X v[V];
      if (a.wide && there == V) {
#pragma unroll
        for (int i = 0; i < (int)(V * sizeof(X) / 16); ++i) reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(x + first + c)[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < there ? x[first + c + i] : from_f32<X>(0.0f);
      }
      if constexpr (sizeof(X) == 2) {
        *reinterpret_cast<uint4 *>(xs + r * pitch + c * 2) = *reinterpret_cast<const uint4 *>(v);
      } else {
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          uint32_t got[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {  // cut, not rounded: the largest numbers would become infinite; what is not finite has one part only
            got[i] = v[i] != v[i] ? 0x7fc00000u : __float_as_uint(v[i]) & 0xffff0000u;
            v[i] = (got[i] & 0x7f800000u) == 0x7f800000u ? 0.0f : v[i] - __uint_as_float(got[i]);
          }
          *reinterpret_cast<uint4 *>(xs + (r * 3 + p) * pitch + c * 2) = make_uint4(__byte_perm(got[0], got[1], 0x7632), __byte_perm(got[2], got[3], 0x7632),
                                                                                    __byte_perm(got[4], got[5], 0x7632), __byte_perm(got[6], got[7], 0x7632));
        }
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// A warp's way through a strip: the batch that it multiplies, whose blocks give way to the next one's as they are used.
template <int GROUP, bool ZEROS>
struct Way {
  static constexpr int GROUPS = BATCH / GROUP;
  Batch<GROUP> next;   // codes: of this batch until they are used, then of the next
  float scale[2][GROUPS];
  uint32_t zero[2];
  const uint4 *codes;  // of the lane, of the next batch
  const uint8_t *record;
  int left;            // blocks from the next batch on
  int code_step, record_step, block_step;

  // shares: by which a warp's batches lie apart
  __device__ __forceinline__ void begin(const ProductArgs &a, int64_t strip, int first, int shares, int lane) {
    codes = reinterpret_cast<const uint4 *>(a.codes) + (strip * a.blocks + first * (BATCH / BLOCK)) * 32 + lane;
    record = a.records + (strip * a.batches + first) * a.record_bytes;
    left = a.blocks - first * (BATCH / BLOCK);
    code_step = shares * (BATCH / BLOCK) * 32, record_step = shares * a.record_bytes, block_step = shares * (BATCH / BLOCK);
#pragma unroll
    for (int b = 0; b < BATCH / BLOCK; ++b) ask(b);
    if (left > 0) next.template load_record<ZEROS>(a, record, lane);
    advance();
  }
  __device__ __forceinline__ void ask(int b) {
    if (b < left) next.code[b] = codes[b * 32];
  }
  __device__ __forceinline__ void advance() {
    codes += code_step;
    record += record_step;
    left -= block_step;
  }
  // Takes over the record of the batch whose codes are there, and asks for the next one's.
  __device__ __forceinline__ void enter(const ProductArgs &a, int lane) {
    if (a.scale_type == LAPIS_F32) {
#pragma unroll
      for (int i = 0; i < 2 * GROUPS; ++i) scale[i / GROUPS][i % GROUPS] = __uint_as_float(next.scale[i]);
    } else if (a.scale_type == LAPIS_BF16) {
#pragma unroll
      for (int i = 0; i < 2 * GROUPS; ++i) scale[i / GROUPS][i % GROUPS] = __uint_as_float(i % 2 ? next.scale[i / 2] & 0xffff0000u : next.scale[i / 2] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * GROUPS; i += 2) {
        const float2 s = __half22float2(*reinterpret_cast<const __half2 *>(&next.scale[i / 2]));
        scale[i / GROUPS][i % GROUPS] = s.x, scale[(i + 1) / GROUPS][(i + 1) % GROUPS] = s.y;
      }
    }
    zero[0] = next.zero[0], zero[1] = next.zero[1];
    if (left > 0) next.template load_record<ZEROS>(a, record, lane);
  }
};

// sum += the product of the batch that `way` is at with the rows x, whose lane's pieces begin at x_at.
template <typename T, int GROUP, int NT, bool ZEROS>
__device__ __forceinline__ void multiply_batch(const ProductArgs &a, float (&sum)[NT][4], Way<GROUP, ZEROS> &way, const uint8_t *x, const int (&x_at)[NT], int tiles,
                                               int lane) {
  float part[NT][4];
  way.enter(a, lane);
#pragma unroll
  for (int half = 0; half < 2 * BATCH / BLOCK; ++half) {
    const int g = half * 32 / GROUP;
    const uint4 c = way.next.code[half / 2];
    Zero<T> z0, z1;
    z0.set(ZEROS ? way.zero[0] >> 4 * g & 15 : 8);
    z1.set(ZEROS ? way.zero[1] >> 4 * g & 15 : 8);
    uint32_t p0[4], p1[4];
    pairs_of(p0, half % 2 ? c.y : c.x, z0);
    pairs_of(p1, half % 2 ? c.w : c.z, z1);
    if (half % 2 == 1) way.ask(half / 2);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t > 0 && t >= tiles) break;
      const uint4 v = *reinterpret_cast<const uint4 *>(x + x_at[t] + half * 64);
      if (half * 32 % GROUP == 0) multiply_first<T>(part[t], p0[0], p1[0], p0[1], p1[1], v.x, v.y);
      else multiply<T>(part[t], p0[0], p1[0], p0[1], p1[1], v.x, v.y);
      multiply<T>(part[t], p0[2], p1[2], p0[3], p1[3], v.z, v.w);
    }
    if ((half + 1) * 32 % GROUP == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t > 0 && t >= tiles) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[t][i] = fmaf(way.scale[i / 2][g], part[t][i], sum[t][i]);
      }
    }
  }
  way.advance();
}

// A block's warps are strips times shares of the columns, both powers of two.  A warp takes its batches of a strip one after the
// other, two more on their way to its registers; the rows x are in shared memory, all of their columns where they fit.
template <typename X, int GROUP, int NT, bool ZEROS>
__global__ void __launch_bounds__(FEW_THREADS, FEW_BLOCKS) int4_few_kernel(const __grid_constant__ ProductArgs a) {
  using T = typename std::conditional<std::is_same<X, float>::value, __nv_bfloat16, X>::type;
  constexpr int A_ROW = std::is_same<X, float>::value ? 3 : 1, ROWS = 8 * NT / A_ROW;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ const X *row_at[ROWS];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int strips_log = a.strips_log, shares_log = FEW_WARPS_LOG - strips_log, shares = 1 << shares_log;
  const int my_strip = warp & ((1 << strips_log) - 1), my_share = warp >> strips_log;
  const int strip = (blockIdx.x << strips_log) + my_strip, pitch = few_pitch(a.chunk);
  const int outs_log = a.gated ? 3 : 4, first_out = blockIdx.x << (strips_log + outs_log), expert = blockIdx.y;
  X *const y = static_cast<X *>(a.y);
  const int batches = strip < a.strips ? a.batches : 0;
  const int64_t of_all = (int64_t)expert * a.strips + min(strip, a.strips - 1);  // the strip's number among all matrices'
  Way<GROUP, ZEROS> way;

  // Weights are nobody's result (int4_pack waits for them), so they are asked for in front of pdl_wait(), unless lists say whose.
  const bool early = a.pos == nullptr;
  if (early) way.begin(a, of_all, my_share, shares, lane);
  pdl_wait();
  pdl_release();
  int64_t begin = 0, end = a.rows;
  if (a.pos != nullptr) {
    begin = min((int64_t)max(a.pos[expert], 0), a.rows);
    end = expert < a.experts ? min((int64_t)a.pos[expert + 1], a.rows) : a.rows;
    if (expert == a.experts) {  // rows of no expert
      const int n = min(1 << (strips_log + outs_log), a.outputs - first_out);
      for (int64_t r = begin + threadIdx.x / n; r < end && threadIdx.x < FEW_THREADS / n * n; r += FEW_THREADS / n)
        y[r * a.outputs + first_out + threadIdx.x % n] = from_f32<X>(0.0f);
      return;
    }
  }
  for (int64_t row0 = begin; row0 < end; row0 += a.rows_a_pass) {
    const int rows = (int)min((int64_t)a.rows_a_pass, end - row0), tiles = (rows * A_ROW + 7) / 8;
    if (!early || row0 != begin) way.begin(a, of_all, my_share, shares, lane);
    if (threadIdx.x < rows) {
      int64_t from = row0 + threadIdx.x;
      if (a.fetch) from = a.crd[from] / a.k;
      row_at[threadIdx.x] = (uint64_t)from < (uint64_t)a.x_rows ? static_cast<const X *>(a.x) + from * a.x_stride : nullptr;
    }
    // Columns of the product beyond the rows take the first row's values: nobody looks at them.
    int x_at[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n = t * 8 + lane / 4;
      x_at[t] = (n < rows * A_ROW ? n : 0) * pitch + lane % 4 * 16;
    }
    float sum[NT][4] = {};
    const int step = a.chunk / BATCH;  // a multiple of the shares
    for (int b0 = 0; b0 < a.batches; b0 += step) {
      __syncthreads();
      stage_few<X>(a, smem, row_at, rows, b0 * BATCH, min(a.chunk, (a.batches - b0) * BATCH), pitch);
      __syncthreads();
      for (int b = b0 + my_share; b < min(b0 + step, batches); b += shares)
        multiply_batch<T, GROUP, NT, ZEROS>(a, sum, way, smem + (b - b0) * (BATCH * 2), x_at, tiles, lane);
    }
    // The shares' sums meet in shared memory: [share][strip][column][row].
    float *const sums = reinterpret_cast<float *>(smem);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[(warp * 8 * NT + t * 8 + lane % 4 * 2 + i % 2) * SUM_PITCH + lane / 4 + i / 2 * 8] = sum[t][i];
    __syncthreads();
    const auto total = [&](int s, int r, int n) {
      float v = 0.0f;
#pragma unroll
      for (int p = A_ROW - 1; p >= 0; --p)  // the small parts first
        for (int share = 0; share < shares; ++share) v += sums[(((share << strips_log) + s) * 8 * NT + r * A_ROW + p) * SUM_PITCH + n];
      return v;
    };
    for (int i = threadIdx.x; i < rows << (strips_log + outs_log); i += FEW_THREADS) {
      const int n = i & ((1 << (strips_log + outs_log)) - 1), r = i >> (strips_log + outs_log), s = n >> outs_log, in = n & ((1 << outs_log) - 1);
      if (first_out + n >= a.outputs) continue;
      float v = total(s, r, in);
      if (a.gated) v = v / (1.0f + expf(-v)) * total(s, r, in + 8);
      y[(row0 + r) * a.outputs + first_out + n] = from_f32<X>(v);
    }
    __syncthreads();
  }
}

template <typename X, int GROUP, int NT>
static int launch_few_as(ProductArgs &a, int matrices, cudaStream_t st) {
  constexpr int A_ROW = std::is_same<X, float>::value ? 3 : 1;
  a.rows_a_pass = (int)std::min<int64_t>(a.rows, 8 * NT / A_ROW);
  a.strips_log = 0;
  while (a.strips_log < FEW_WARPS_LOG && (int64_t)(a.strips >> (1 + a.strips_log)) * a.experts >= 4 * sm_count()) ++a.strips_log;
  const int strips = 1 << a.strips_log, turn = BATCH * (FEW_WARPS >> a.strips_log), room = FEW_ROOM;
  a.chunk = std::max(turn, (room / (a.rows_a_pass * A_ROW) - 64) / 2 / turn * turn);
  a.chunk = (int)std::min<int64_t>(a.chunk, (a.columns + turn - 1) / turn * turn);
  const int smem = std::max(a.rows_a_pass * A_ROW * few_pitch(a.chunk), FEW_WARPS * 8 * NT * SUM_PITCH * 4);
  const dim3 grid((a.strips + strips - 1) / strips, matrices);
  const auto kernel = a.zeros_at ? int4_few_kernel<X, GROUP, NT, true> : int4_few_kernel<X, GROUP, NT, false>;
  LAPIS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 << 10));
  LAPIS_CUDA_TRY(launch_pdl(kernel, grid, FEW_THREADS, smem, st, a));
  return LAPIS_OK;
}

template <typename X, typename T, int GROUP, int NT>
static int launch_product_as(ProductArgs &a, int matrices, cudaStream_t st) {
  constexpr int MOST_SHARES = NT == 1 || NT == 2 ? 8 : NT == 4 ? 4 : 2;
  // As many strips a block as leave two blocks an SM: they share the rows x in shared memory.
  a.strips_a_block = INT4_WARPS / MOST_SHARES;
  while (a.strips_a_block < INT4_WARPS && (int64_t)(a.strips / (2 * a.strips_a_block)) * a.experts >= 2 * sm_count()) a.strips_a_block *= 2;
  const int step = BATCH * (INT4_WARPS / a.strips_a_block), room = (64 << 10) / (8 * NT) - 64;  // bytes of a row of x
  a.chunk = std::max(step, room / 2 / step * step);
  a.chunk = (int)std::min<int64_t>(a.chunk, (a.columns + step - 1) / step * step);
  const int smem = std::max(8 * NT * x_pitch(a.chunk), INT4_WARPS * 8 * NT * SUM_PITCH * 4);
  const dim3 grid((a.strips + a.strips_a_block - 1) / a.strips_a_block, matrices);
  LAPIS_CUDA_TRY(cudaFuncSetAttribute(int4_kernel<X, T, GROUP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 << 10));
  LAPIS_CUDA_TRY(launch_pdl(int4_kernel<X, T, GROUP, NT>, grid, INT4_THREADS, smem, st, a));
  return LAPIS_OK;
}
template <typename X, typename T, int GROUP>
static int launch_product_of(ProductArgs &a, int matrices, int64_t expected, cudaStream_t st) {
  const int64_t columns = expected * (std::is_same<X, float>::value ? 3 : 1);
  if (columns <= 8) return launch_few_as<X, GROUP, 1>(a, matrices, st);
  if (columns <= 16) return launch_few_as<X, GROUP, 2>(a, matrices, st);
  if (columns <= 32) return launch_product_as<X, T, GROUP, 4>(a, matrices, st);
  return launch_product_as<X, T, GROUP, 8>(a, matrices, st);
}
template <typename X, typename T>
static int launch_product(ProductArgs &a, int group, int matrices, int64_t expected, cudaStream_t st) {
  switch (group) {
    case 32: return launch_product_of<X, T, 32>(a, matrices, expected, st);
    case 64: return launch_product_of<X, T, 64>(a, matrices, expected, st);
    default: return launch_product_of<X, T, 128>(a, matrices, expected, st);
  }
}

static int check_int4(const char *what, const lapis_b200_int4 *w) {
  if (w == nullptr) return fail(LAPIS_EBADARG, "%s: null weights", what);
  if (w->experts < 0 || w->outputs < 0 || w->columns < 0) return fail(LAPIS_EBADSHAPE, "%s: negative size", what);
  if (w->group != 32 && w->group != 64 && w->group != 128) return fail(LAPIS_EBADSHAPE, "%s: groups of 32, 64 or 128 columns", what);
  if (!is_float_type(w->scale_type)) return fail(LAPIS_EBADARG, "%s: scale_type must be LAPIS_F32, LAPIS_F16 or LAPIS_BF16", what);
  if (w->gated && w->outputs % 2 != 0) return fail(LAPIS_EBADSHAPE, "%s: gated weights have an even number of outputs", what);
  if (w->experts > MAX_EXPERTS) return fail(LAPIS_ETOOBIG, "%s: more than %d experts", what, MAX_EXPERTS);
  if (w->outputs > 1 << 24 || w->columns > 1 << 24) return fail(LAPIS_ETOOBIG, "%s: more than 2^24 outputs or columns", what);
  return LAPIS_OK;
}
static bool no_weights(const lapis_b200_int4 *w) { return w->experts == 0 || w->outputs == 0 || w->columns == 0; }

}  // namespace lapis_b200

using namespace lapis_b200;

extern "C" int64_t lapis_b200_int4_bytes(const lapis_b200_int4 *w) {
  clear_error();
  if (check_int4("int4_bytes", w) != LAPIS_OK) return -1;
  return no_weights(w) ? 0 : layout_of(*w).bytes;
}

extern "C" int lapis_b200_int4_pack(const lapis_b200_int4 *w, const void *d_codes, const void *d_scale, const void *d_zero, void *d_packed, void *stream) {
  clear_error();
  const char *what = "int4_pack";
  LAPIS_TRY(check_int4(what, w));
  if (no_weights(w)) return LAPIS_OK;
  if (d_codes == nullptr || d_scale == nullptr || d_packed == nullptr || (w->zeros && d_zero == nullptr)) return fail(LAPIS_EBADARG, "%s: null operand", what);
  if (reinterpret_cast<uintptr_t>(d_packed) % 16 != 0) return fail(LAPIS_EBADARG, "%s: d_packed must be aligned to 16 bytes", what);
  const Int4Layout l = layout_of(*w);
  const cudaStream_t st = as_stream(stream);
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  LAPIS_CUDA_TRY(cudaStreamIsCapturing(st, &capture));
  if (capture != cudaStreamCaptureStatusNone) return fail(LAPIS_EBADARG, "%s: not under stream capture, it waits for the stream", what);
  PackArgs a = {};
  a.outputs = w->outputs;
  a.columns = w->columns;
  a.strips = l.strips;
  a.blocks = l.blocks;
  a.batches = l.batches;
  a.group = w->group;
  a.gated = w->gated;
  a.scale_bytes = type_bytes(w->scale_type);
  a.codes = static_cast<const uint8_t *>(d_codes);
  a.scale = d_scale;
  a.zero = w->zeros ? static_cast<const uint8_t *>(d_zero) : nullptr;
  a.packed_codes = static_cast<uint8_t *>(d_packed);
  a.records = a.packed_codes + l.records_at;
  a.zeros_at = (int)l.scale_bytes;
  a.record_bytes = (int)l.record_bytes;
  const unsigned most = 32 * sm_count();
  a.items = w->experts * l.strips * l.blocks * 32;
  pack_codes_kernel<<<(unsigned)std::min<int64_t>(most, (a.items + 255) / 256), 256, 0, st>>>(a);
  LAPIS_CUDA_TRY(cudaGetLastError());
  a.items = w->experts * l.strips * l.batches * 8;
  pack_scales_kernel<<<(unsigned)std::min<int64_t>(most, (a.items + 255) / 256), 256, 0, st>>>(a);
  LAPIS_CUDA_TRY(cudaGetLastError());
  LAPIS_CUDA_TRY(cudaStreamSynchronize(st));
  return LAPIS_OK;
}

extern "C" int lapis_b200_int4_quantise(int type, int64_t rows, int64_t columns, const void *d_w, int64_t w_stride, int group, int scale_type, void *d_codes,
                                        void *d_scale, void *d_zero, void *stream) {
  clear_error();
  const char *what = "int4_quantise";
  if (!is_float_type(type)) return fail(LAPIS_EBADARG, "%s: type must be LAPIS_F32, LAPIS_F16 or LAPIS_BF16", what);
  const lapis_b200_int4 w = {1, 0, columns, group, scale_type, d_zero != nullptr, 0, nullptr};
  LAPIS_TRY(check_int4(what, &w));
  if (rows < 0) return fail(LAPIS_EBADSHAPE, "%s: negative size", what);
  if (rows == 0 || columns == 0) return LAPIS_OK;
  if (d_w == nullptr || d_codes == nullptr || d_scale == nullptr) return fail(LAPIS_EBADARG, "%s: null operand", what);
  QuantiseArgs a = {};
  a.w = d_w;
  a.w_stride = w_stride;
  a.columns = columns;
  a.groups = (columns + group - 1) / group;
  a.items = rows * a.groups;
  a.group = group;
  a.scale_type = scale_type;
  a.codes = static_cast<uint8_t *>(d_codes);
  a.zero = static_cast<uint8_t *>(d_zero);
  a.scale = d_scale;
  const unsigned grid = (unsigned)std::min<int64_t>(32 * sm_count(), (a.items + 7) / 8);
  const cudaStream_t st = as_stream(stream);
  if (type == LAPIS_F32) quantise_kernel<float><<<grid, 256, 0, st>>>(a);
  else if (type == LAPIS_F16) quantise_kernel<__half><<<grid, 256, 0, st>>>(a);
  else quantise_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  LAPIS_CUDA_TRY(cudaGetLastError());
  return LAPIS_OK;
}

extern "C" int lapis_b200_int4_matmul(int type, const lapis_b200_int4 *w, int64_t rows, const void *d_x, int64_t x_stride, const lapis_b200_expert_lists *lists,
                                      int fetch, void *d_y, void *stream) {
  clear_error();
  const char *what = "int4_matmul";
  if (!is_float_type(type)) return fail(LAPIS_EBADARG, "%s: type must be LAPIS_F32, LAPIS_F16 or LAPIS_BF16", what);
  LAPIS_TRY(check_int4(what, w));
  if (rows < 0) return fail(LAPIS_EBADSHAPE, "%s: negative size", what);
  if (rows > 0x7fffffff) return fail(LAPIS_ETOOBIG, "%s: 2^31 rows or more", what);
  ProductArgs a = {};
  a.rows = a.x_rows = rows;
  if (lists != nullptr) {
    LAPIS_TRY(check_expert_lists(what, lists));
    if (lists->experts != w->experts) return fail(LAPIS_EBADSHAPE, "%s: lists of another number of experts", what);
    a.rows = lists->tokens * lists->k;
    if (rows != (fetch ? lists->tokens : a.rows)) return fail(LAPIS_EBADSHAPE, "%s: rows of x do not fit the lists", what);
  } else if (w->experts != 1) {
    return fail(LAPIS_EBADSHAPE, "%s: weights of several experts need lists", what);
  }
  if (a.rows == 0 || w->outputs == 0) return LAPIS_OK;
  if (d_y == nullptr || (!no_weights(w) && (d_x == nullptr || w->d_packed == nullptr))) return fail(LAPIS_EBADARG, "%s: null operand", what);
  a.outputs = (int)(w->gated ? w->outputs / 2 : w->outputs);
  const cudaStream_t st = as_stream(stream);
  if (no_weights(w)) {
    LAPIS_CUDA_TRY(cudaMemsetAsync(d_y, 0, (size_t)a.rows * a.outputs * type_bytes(type), st));
    return LAPIS_OK;
  }
  const Int4Layout l = layout_of(*w);
  a.codes = static_cast<const uint8_t *>(w->d_packed);
  a.records = a.codes + l.records_at;
  a.zeros_at = w->zeros ? (int)l.scale_bytes : 0;
  a.record_bytes = (int)l.record_bytes;
  a.scale_type = w->scale_type;
  a.gated = w->gated != 0;
  a.experts = (int)w->experts;
  a.strips = (int)l.strips;
  a.blocks = (int)l.blocks;
  a.batches = (int)l.batches;
  a.columns = w->columns;
  a.x = d_x;
  a.x_stride = x_stride;
  a.y = d_y;
  a.wide = reinterpret_cast<uintptr_t>(d_x) % 16 == 0 && (rows == 1 || x_stride * type_bytes(type) % 16 == 0);
  if (lists != nullptr) {
    a.pos = lists->d_pos;
    a.crd = lists->d_crd;
    a.k = (int)lists->k;
    a.fetch = fetch != 0;
  }
  const int matrices = a.experts + (lists != nullptr ? 1 : 0);
  // Lists are ragged: most have no more than twice the mean.
  const int64_t expected = lists == nullptr ? a.rows : std::min(a.rows, 2 * ((a.rows + a.experts - 1) / a.experts));
  switch (type) {
    case LAPIS_F32: return launch_product<float, __nv_bfloat16>(a, w->group, matrices, expected, st);
    case LAPIS_F16: return launch_product<__half, __half>(a, w->group, matrices, expected, st);
    default: return launch_product<__nv_bfloat16, __nv_bfloat16>(a, w->group, matrices, expected, st);
  }
}

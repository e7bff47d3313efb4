// Products of few rows with 4-bit weights (int4.cu) on mma.sync: 8 columns of the product, 16 outputs a warp.
//
// The weights go from memory to registers, a batch ahead, and need nothing but their own warp; the rows x, the B operand, are in shared
// memory.  What bounds it are the instructions on 32 bits that make numbers of codes: of one every two cycles a batch of 16 x 256 takes 150 to
// 190, its bytes as long as 170.  48 x 8 rows over 128 experts (2048 x 2048, groups of 32, gated) 76 us, 3.8 TB/s; one row times 14,336 x 4096 10.9 us,
// 2.8 TB/s; 4096 x 4096 5.0 us, most of it launch and latency.  tcgen05 (int4_many.cu) with 8 columns would convert as many codes and add its
// hand-overs: 16 rows x 14,336 x 4096 take it 21 us where 8 take this 17.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "int4.h"

namespace lapis_b200 {

template <typename T>
__device__ __forceinline__ void multiply(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with sums of zero.
template <typename T>
__device__ __forceinline__ void multiply_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// What a lane holds of a batch: 16 columns of rows r and r + 8 in each of four blocks, their scales and zeros.
template <int GROUP, bool FULL>
struct Batch {
  static constexpr int GROUPS = BATCH / GROUP, SCALES = FULL ? 2 * GROUPS : GROUPS;  // words of scales: FULL those of 32 bits, else two in a word
  uint4 code[BATCH / BLOCK];
  uint32_t scale[SCALES];
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
  template <bool ZEROS>
  __device__ __forceinline__ void load_record(const ProductArgs &a, const uint8_t *record, int lane) {
    const int row = lane / 4;
    fetch<SCALES>(scale, record + row * SCALES * 4);
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
};

constexpr int SUM_PITCH = STRIP + 1;

constexpr int FEW_WARPS_LOG = 2, FEW_WARPS = 1 << FEW_WARPS_LOG, FEW_THREADS = 32 * FEW_WARPS;
// Blocks of an SM, and the rows x of each in shared memory.  48 x 8 rows over 128 experts take 79 us with 5 blocks, 82 with 4, 78 with 6, for
// which scales of 32 bits have to be spilled (with 5 only where groups are of 32: 8 to 20 bytes); with two of eight warps 87.
constexpr int FEW_BLOCKS = 5, FEW_ROOM = 40 << 10;

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
template <int GROUP, bool ZEROS, bool FULL>
struct Way {
  static constexpr int GROUPS = BATCH / GROUP, SCALES = Batch<GROUP, FULL>::SCALES;
  Batch<GROUP, FULL> next;  // codes: of this batch until they are used, then of the next
  uint32_t scale[SCALES];
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
#pragma unroll
    for (int i = 0; i < SCALES; ++i) scale[i] = next.scale[i];
    zero[0] = next.zero[0], zero[1] = next.zero[1];
    if (left > 0) next.template load_record<ZEROS>(a, record, lane);
  }
  // Scale of group g of row r (0) or r + 8 (1).
  __device__ __forceinline__ float scale_of(int row, int g, bool bf16) const {
    const int i = row * GROUPS + g;
    if constexpr (FULL) return __uint_as_float(scale[i]);
    const uint32_t w = scale[i / 2];
    if (bf16) return __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
    return __half2float(__ushort_as_half((unsigned short)(i % 2 ? w >> 16 : w & 0xffffu)));
  }
};

// sum += the product of the batch that `way` is at with the rows x, of which the lane's pieces begin at x.
template <typename T, int GROUP, bool ZEROS, bool FULL>
__device__ __forceinline__ void multiply_batch(const ProductArgs &a, float (&sum)[4], Way<GROUP, ZEROS, FULL> &way, const uint8_t *x, int lane) {
  float part[4];
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
    const uint4 v = *reinterpret_cast<const uint4 *>(x + half * 64);
    if (half * 32 % GROUP == 0) multiply_first<T>(part, p0[0], p1[0], p0[1], p1[1], v.x, v.y);
    else multiply<T>(part, p0[0], p1[0], p0[1], p1[1], v.x, v.y);
    multiply<T>(part, p0[2], p1[2], p0[3], p1[3], v.z, v.w);
    if ((half + 1) * 32 % GROUP == 0) {
      const float s0 = way.scale_of(0, g, a.scale_type == LAPIS_BF16), s1 = way.scale_of(1, g, a.scale_type == LAPIS_BF16);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = fmaf(i < 2 ? s0 : s1, part[i], sum[i]);
    }
  }
  way.advance();
}

// A block's warps are strips times shares of the columns, both powers of two.  A warp takes its batches of a strip one after the
// other, the next on its way to its registers; the rows x are in shared memory, all of their columns where they fit.
template <typename X, int GROUP, bool ZEROS, bool FULL>
__global__ void __launch_bounds__(FEW_THREADS, FEW_BLOCKS) int4_few_kernel(const __grid_constant__ ProductArgs a) {
  using T = typename std::conditional<std::is_same<X, float>::value, __nv_bfloat16, X>::type;
  constexpr int A_ROW = std::is_same<X, float>::value ? 3 : 1, ROWS = FEW_COLUMNS / A_ROW;
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
  Way<GROUP, ZEROS, FULL> way;

  // Weights are nobody's result (int4_pack waits for them), so they are asked for in front of pdl_wait(), unless lists say whose.
  const bool early = a.pos == nullptr;
  if (early) way.begin(a, of_all, my_share, shares, lane);
  pdl_wait();
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
    const int rows = (int)min((int64_t)a.rows_a_pass, end - row0);
    if (!early || row0 != begin) way.begin(a, of_all, my_share, shares, lane);
    if (threadIdx.x < rows) {
      int64_t from = row0 + threadIdx.x;
      if (a.fetch) from = a.crd[from] / a.k;
      row_at[threadIdx.x] = (uint64_t)from < (uint64_t)a.x_rows ? static_cast<const X *>(a.x) + from * a.x_stride : nullptr;
    }
    // Columns of the product beyond the rows take the first row's values: nobody looks at them.
    const uint8_t *const x = smem + (lane / 4 < rows * A_ROW ? lane / 4 : 0) * pitch + lane % 4 * 16;
    float sum[4] = {};
    const int step = a.chunk / BATCH;  // a multiple of the shares
    for (int b0 = 0; b0 < a.batches; b0 += step) {
      __syncthreads();
      stage_few<X>(a, smem, row_at, rows, b0 * BATCH, min(a.chunk, (a.batches - b0) * BATCH), pitch);
      __syncthreads();
      for (int b = b0 + my_share; b < min(b0 + step, batches); b += shares)
        multiply_batch<T, GROUP, ZEROS, FULL>(a, sum, way, x + (b - b0) * (BATCH * 2), lane);
    }
    // The shares' sums meet in shared memory: [share][strip][column][row].
    float *const sums = reinterpret_cast<float *>(smem);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[(warp * FEW_COLUMNS + lane % 4 * 2 + i % 2) * SUM_PITCH + lane / 4 + i / 2 * 8] = sum[i];
    __syncthreads();
    const auto total = [&](int s, int r, int n) {
      float v = 0.0f;
#pragma unroll
      for (int p = A_ROW - 1; p >= 0; --p)  // the small parts first
        for (int share = 0; share < shares; ++share) v += sums[(((share << strips_log) + s) * FEW_COLUMNS + r * A_ROW + p) * SUM_PITCH + n];
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

template <typename X, int GROUP, bool ZEROS, bool FULL>
static int launch_few_as(ProductArgs &a, int matrices, cudaStream_t st) {
  constexpr int A_ROW = std::is_same<X, float>::value ? 3 : 1;
  a.rows_a_pass = (int)std::min<int64_t>(a.rows, FEW_COLUMNS / A_ROW);
  a.strips_log = 0;
  // Warps that take whole strips share the rows x, warps that share a strip fill the GPU: as many strips as leave four blocks an SM.  14,336 x
  // 4096 (896 strips), one row: a strip a block 12.4 us, two 15.0; 128 experts of 128 strips: a strip 127 us, two 95, four 85.
  while (a.strips_log < FEW_WARPS_LOG && (int64_t)(a.strips >> (1 + a.strips_log)) * a.experts >= 4 * sm_count()) ++a.strips_log;
  const int strips = 1 << a.strips_log, turn = BATCH * (FEW_WARPS >> a.strips_log);
  a.chunk = std::max(turn, (FEW_ROOM / (a.rows_a_pass * A_ROW) - 64) / 2 / turn * turn);
  a.chunk = (int)std::min<int64_t>(a.chunk, (a.columns + turn - 1) / turn * turn);
  const int smem = std::max(a.rows_a_pass * A_ROW * few_pitch(a.chunk), FEW_WARPS * FEW_COLUMNS * SUM_PITCH * 4);
  const dim3 grid((a.strips + strips - 1) / strips, matrices);
  LAPIS_TRY((allow_smem<int4_few_kernel<X, GROUP, ZEROS, FULL>>(160 << 10)));
  LAPIS_CUDA_TRY(launch_pdl(int4_few_kernel<X, GROUP, ZEROS, FULL>, grid, FEW_THREADS, smem, st, a));
  return LAPIS_OK;
}

template <typename X, int GROUP>
static int launch_few_as(ProductArgs &a, int matrices, cudaStream_t st) {
  if (a.scale_type == LAPIS_F32) return a.zeros_at ? launch_few_as<X, GROUP, true, true>(a, matrices, st) : launch_few_as<X, GROUP, false, true>(a, matrices, st);
  return a.zeros_at ? launch_few_as<X, GROUP, true, false>(a, matrices, st) : launch_few_as<X, GROUP, false, false>(a, matrices, st);
}
template <typename X>
static int launch_few_of(ProductArgs &a, int group, int matrices, cudaStream_t st) {
  switch (group) {
    case 32: return launch_few_as<X, 32>(a, matrices, st);
    case 64: return launch_few_as<X, 64>(a, matrices, st);
    default: return launch_few_as<X, 128>(a, matrices, st);
  }
}
int launch_few(int type, ProductArgs &a, int group, int matrices, cudaStream_t st) {
  switch (type) {
    case LAPIS_F32: return launch_few_of<float>(a, group, matrices, st);
    case LAPIS_F16: return launch_few_of<__half>(a, group, matrices, st);
    default: return launch_few_of<__nv_bfloat16>(a, group, matrices, st);
  }
}

}  // namespace lapis_b200

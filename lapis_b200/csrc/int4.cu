// Few rows times weights of 4 bits with a scale (and a zero) for every group of columns.
//
//   y[r, n] = sum over groups of  scale[n, group] * sum over the group's columns of (code[n, c] - zero[n, group]) x[r, c]
//
// code - zero is a whole number between -15 and 15, exact in bf16 and fp16; so is x (32 bits: three parts of bf16, three columns of
// the product, which hold all 24 bits from 2^-110 on, where the last of them is 2^-133 or more, bf16's smallest subnormal number); their products
// are added in 32 bits on the tensor cores, which cut where other additions round, a group's sum is scaled in 32 bits, and the result
// is rounded once.  With `gated` outputs the two halves of the result meet in a lane, silu(gate) * up, in 32 bits.
//
// The work is to read the weights once.  They lie in the order in which a warp takes them: a strip of 16 outputs, 64 columns of
// it in one 16-byte load a lane, which is the A operand of four products of 16 x 8 x 16 (int4_few.cu) or, converted, of a warp's store to
// tensor memory (int4_many.cu).  The columns of a product may come in any order, the same for A and B: the lane of a row takes 8 that
// lie next to one another in each half of the 64.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "int4.h"

namespace lapis_b200 {


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
  // Lists are ragged, and nobody here knows how: what is chosen serves experts of up to twice the mean by one pass, others by several (128 experts of 2 rows
  // x 2048 x 2048 81 us; one of them with 40 rows more 84, with 200 more 196).
  const int64_t expected = lists == nullptr ? a.rows : std::min(a.rows, 2 * ((a.rows + a.experts - 1) / a.experts));
  const bool few = expected * (type == LAPIS_F32 ? 3 : 1) <= FEW_COLUMNS;
  return few ? launch_few(type, a, w->group, matrices, st) : launch_many(type, a, w->group, matrices, expected, st);
}

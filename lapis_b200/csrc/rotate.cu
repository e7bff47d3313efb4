// Norms of the queries and keys of each head with their rotation by position, forward and backward, and the cache that keys
// and values are written to on the same pass and read back from.
//
// A row x is one head of one token, `dim` values:
//   n_i = x_i r w_i,  r = 1 / sqrt(mean_i x_i^2 + eps)
//   the first `rot` of them are turned in pairs (a, b) by the angle of the token's place:  a' = a cos - b sin,  b' = b cos + a sin
// with the pairs (i, i + rot/2) or, interleaved, (2i, 2i + 1).  Backward, with dn the gradient turned the other way and
// g_i = w_i dn_i:
//   dx_i = r (g_i - x_i r^2 mean_j g_j x_j),   dw_i = sum over rows of dn_i x_i r
// Everything is computed in 32 bits and rounded once, when it is stored.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "kv.h"

namespace lapis_b200 {

constexpr int ROW_THREADS = 128;
constexpr int ROW_WARPS = ROW_THREADS / 32;
constexpr int PER_LANE = KV_MAX_DIM / 32;

struct Rows {
  const void *d;
  int64_t token_stride, head_stride;
};

struct RotateArgs {
  int64_t tokens;
  int dim, rot, interleaved, heads[3];  // heads of q, k and v
  Rows in[3];                           // q, k, v
  Rows grad[2];                         // backward: of the outputs q, k
  void *out[2];                         // q, k: [tokens, heads, dim]
  int norm;
  const void *weight[2];
  int weight_f32;
  const float *cos, *sin;
  int64_t places;
  float eps;
  int idx_bytes;
  const void *place, *row;
  int to_cache;
  lapis_b200_kv_cache cache;
  lapis_b200_page_lists lists;
  int page_shift;  // log2 of the slots of a page, or -1
  float *partial;  // backward: [blocks][2][dim]
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

template <typename T>
__device__ __forceinline__ float weight_at(const RotateArgs &a, int which, int i) {
  return a.weight_f32 ? static_cast<const float *>(a.weight[which])[i] : to_f32(static_cast<const T *>(a.weight[which])[i]);
}

// The other element of the pair of element i < rot, the pair's number, and whether i is its first.
__device__ __forceinline__ int partner(int i, int rot, int interleaved, int *pair, bool *first) {
  if (interleaved) {
    *pair = i / 2;
    *first = (i & 1) == 0;
    return i ^ 1;
  }
  const int half = rot / 2;
  *first = i < half;
  *pair = *first ? i : i - half;
  return *first ? i + half : i - half;
}

// Any width, stride and alignment: a warp per row, the row in shared memory for the partners of the rotation.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) rotate_any_kernel(const __grid_constant__ RotateArgs a) {
  __shared__ float rows[ROW_WARPS][KV_MAX_DIM];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int per_token = a.heads[0] + a.heads[1] + a.heads[2];
  const int64_t task = (int64_t)blockIdx.x * ROW_WARPS + warp;
  if (task >= a.tokens * per_token) return;
  const int64_t token = task / per_token;
  int head = (int)(task % per_token), which = 0;
  while (head >= a.heads[which]) head -= a.heads[which++];
  float *const x = rows[warp];
  const T *const in = static_cast<const T *>(a.in[which].d) + token * a.in[which].token_stride + head * a.in[which].head_stride;
  const int64_t place = a.place != nullptr ? load_index(a.place, token, a.idx_bytes) : 0;
  const bool norm = a.norm && which < 2, real = !a.norm || (place >= 0 && place < a.places);
  float sum = 0.0f;
  for (int i = lane; i < a.dim; i += 32) {
    x[i] = real ? to_f32(in[i]) : 0.0f;
    sum = fmaf(x[i], x[i], sum);
  }
  __syncwarp();
  float y[PER_LANE];
  if (norm && real) {
    const float r = 1.0f / sqrtf(warp_sum(sum) / (float)a.dim + a.eps);
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
      const int i = lane + 32 * j;
      y[j] = 0.0f;
      if (i >= a.dim) continue;
      y[j] = x[i] * r * weight_at<T>(a, which, i);
      if (i < a.rot) {
        int pair;
        bool first;
        const int o = partner(i, a.rot, a.interleaved, &pair, &first);
        const float c = a.cos[place * (a.rot / 2) + pair], s = a.sin[place * (a.rot / 2) + pair];
        const float other = x[o] * r * weight_at<T>(a, which, o);
        y[j] = first ? y[j] * c - other * s : y[j] * c + other * s;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) y[j] = lane + 32 * j < a.dim ? x[lane + 32 * j] : 0.0f;
  }
  if (which == 0 || !a.to_cache) {
    T *const out = static_cast<T *>(a.out[which]) + (token * a.heads[which] + head) * a.dim;
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j)
      if (lane + 32 * j < a.dim) out[lane + 32 * j] = from_f32<T>(y[j]);
    return;
  }
  if (!real) return;
  const int64_t first_row = cache_row(a.cache, a.lists, load_index(a.row, token, a.idx_bytes), place, a.page_shift);
  if (first_row < 0) return;
  const int64_t row = first_row + head * a.cache.page_size;
  void *const store = which == 1 ? a.cache.d_k : a.cache.d_v;
  if (!is_quantised(a.cache.type)) {
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j)
      if (lane + 32 * j < a.dim) static_cast<T *>(store)[row * a.dim + lane + 32 * j] = from_f32<T>(y[j]);
    return;
  }
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < PER_LANE; ++j) most = max_nan(most, fabsf(y[j]));
#pragma unroll
  for (int d = 16; d > 0; d /= 2) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, d));
  const float big = largest_code(a.cache.type);
  if (lane == 0) (which == 1 ? a.cache.d_k_scale : a.cache.d_v_scale)[row] = scale_of(most, big);
  if (most < SMALL_ROW) {
    most *= RAISE;
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) y[j] *= RAISE;
  }
  const float by = most == 0.0f ? 0.0f : big / most;
#pragma unroll
  for (int j = 0; j < PER_LANE; ++j) {
    if (lane + 32 * j >= a.dim) continue;
    const float code = y[j] * by;
    if (a.cache.type == LAPIS_I8) static_cast<int8_t *>(store)[row * a.dim + lane + 32 * j] = to_i8(code);
    else static_cast<uint8_t *>(store)[row * a.dim + lane + 32 * j] = to_e4m3(code);
  }
}

// Backward, any width, stride and alignment: a warp takes whole tokens, a grid apart, and keeps its share of the weights'
// gradients in registers; the warps of a block are added in order, the blocks by rotate_weights_kernel.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) rotate_any_backward_kernel(const __grid_constant__ RotateArgs a) {
  __shared__ float rows[ROW_WARPS][2][KV_MAX_DIM];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  float *const x = rows[warp][0], *const dy = rows[warp][1];
  float dw[2][PER_LANE];
#pragma unroll
  for (int j = 0; j < PER_LANE; ++j) dw[0][j] = dw[1][j] = 0.0f;
  for (int64_t token = (int64_t)blockIdx.x * ROW_WARPS + warp; token < a.tokens; token += (int64_t)gridDim.x * ROW_WARPS) {
    const int64_t place = load_index(a.place, token, a.idx_bytes);
    const bool real = place >= 0 && place < a.places;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      for (int head = 0; head < a.heads[which]; ++head) {
        const T *const in = static_cast<const T *>(a.in[which].d) + token * a.in[which].token_stride + head * a.in[which].head_stride;
        const T *const grad = static_cast<const T *>(a.grad[which].d) + token * a.grad[which].token_stride + head * a.grad[which].head_stride;
        T *const out = static_cast<T *>(a.out[which]) + (token * a.heads[which] + head) * a.dim;
        float sum = 0.0f, inner = 0.0f, dn[PER_LANE];
        __syncwarp();
        for (int i = lane; i < a.dim; i += 32) {
          x[i] = real ? to_f32(in[i]) : 0.0f;
          dy[i] = real ? to_f32(grad[i]) : 0.0f;
          sum = fmaf(x[i], x[i], sum);
        }
        __syncwarp();
        const float mean = warp_sum(sum) / (float)a.dim, r = real ? 1.0f / sqrtf(mean + a.eps) : 0.0f;  // eps may be zero
#pragma unroll
        for (int j = 0; j < PER_LANE; ++j) {
          const int i = lane + 32 * j;
          dn[j] = 0.0f;
          if (i >= a.dim) continue;
          dn[j] = dy[i];
          if (real && i < a.rot) {
            int pair;
            bool first;
            const int o = partner(i, a.rot, a.interleaved, &pair, &first);
            const float c = a.cos[place * (a.rot / 2) + pair], s = a.sin[place * (a.rot / 2) + pair];
            dn[j] = first ? dy[i] * c + dy[o] * s : dy[i] * c - dy[o] * s;
          }
          inner = fmaf(dn[j] * weight_at<T>(a, which, i), x[i], inner);
          dw[which][j] = fmaf(dn[j] * x[i], r, dw[which][j]);
        }
        inner = warp_sum(inner) / (float)a.dim * r * r;
#pragma unroll
        for (int j = 0; j < PER_LANE; ++j) {
          const int i = lane + 32 * j;
          if (i < a.dim) out[i] = from_f32<T>(r * (dn[j] * weight_at<T>(a, which, i) - x[i] * inner));
        }
      }
    }
  }
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) rows[warp][0][lane + 32 * j] = dw[which][j];
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += ROW_THREADS) {
      float sum = 0.0f;
      for (int w = 0; w < ROW_WARPS; ++w) sum += rows[w][0][i];
      a.partial[((int64_t)blockIdx.x * 2 + which) * a.dim + i] = sum;
    }
  }
}

// dw = sum of the blocks' shares, in the order of the blocks: 32 sums a block apart, then those.
__global__ void __launch_bounds__(1024) rotate_weights_kernel(const float *partial, int blocks, int dim, float *dqw, float *dkw) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x % 32, nth = threadIdx.x / 32, i = blockIdx.x * 32 + lane, which = blockIdx.y;
  float sum = 0.0f;
  pdl_wait();
  if (i < dim) {
#pragma unroll 8
    for (int b = nth; b < blocks; b += 32) sum += partial[((int64_t)b * 2 + which) * dim + i];
  }
  sums[nth][lane] = sum;
  __syncthreads();
  if (nth == 0 && i < dim) {
#pragma unroll
    for (int b = 1; b < 32; ++b) sum += sums[b][lane];
    (which == 0 ? dqw : dkw)[i] = sum;
  }
}

// Keys and values of listed tokens out of the cache: a warp per row.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS)
kv_read_any_kernel(lapis_b200_kv_cache cache, lapis_b200_page_lists lists, int64_t tokens, const void *row, const void *place, T *k, T *v) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t task = (int64_t)blockIdx.x * ROW_WARPS + warp;
  if (task >= tokens * cache.heads) return;
  const int64_t token = task / cache.heads, head = task % cache.heads;
  const int64_t first = cache_row(cache, lists, load_index(row, token, lists.idx_bytes), load_index(place, token, lists.idx_bytes), -1);
  const int64_t at = first + head * cache.page_size;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T *const out = (which == 0 ? k : v) + task * cache.dim;
    const void *const store = which == 0 ? cache.d_k : cache.d_v;
    float scale = 1.0f;
    if (first >= 0 && is_quantised(cache.type)) scale = (which == 0 ? cache.d_k_scale : cache.d_v_scale)[at];
    for (int i = lane; i < cache.dim; i += 32)
      out[i] = from_f32<T>(first < 0 ? 0.0f : load_as_f32(store, at * cache.dim + i, cache.type) * scale);
  }
}

// ---- whole 16 bytes ---------------------------------------------------------------
//
// Bound by memory: every element is read and written once, so what a row costs in instructions has to stay small next to the
// 0.7 pieces of 16 bytes that an SM can read and write in a cycle, and enough has to be on its way.  A row is held by LANES
// neighbouring lanes, two pieces each, so chosen that a value and its partner in the rotation are in one lane; a warp holds
// 32 / LANES rows at a time (a round) and walks the rows of a token, so that the token's line of the tables, the weights and
// the place in the cache are looked up once for many rows.  Rows come by cp.async, DEPTH rounds ahead, into a ring that every
// lane uses for itself: what is on its way takes no registers.  Weight and rotation are one product each with a value and
// its partner, y = r (x wc + x' ws), wc = w cos, ws = -+ w' sin, two values an instruction.
// Measured, bf16 heads of 128: 8192 tokens of 32 + 8 heads 31 us (5.5 TB/s; 40 us with the partner in another lane, 180
// instructions for two rows; 33 with six blocks an SM, which spill), backward of 16,384 85 us (6.0 TB/s) and 4.6 to add up the
// weights' gradients, 32,768 tokens of 32 + 8 + 8 normalised and written as int8 139 us (5.3 TB/s), read back 40 (5.0 TB/s).

__device__ __forceinline__ uint32_t shared_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes on their way to shared memory, zeros where there is nothing.
__device__ __forceinline__ void bring(uint32_t to, const void *from, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void brought() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void wait_for_all_but() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// fma2 and mul2 for all of a piece, or of any even number of floats.
template <int N>
__device__ __forceinline__ void fma_all(float (&d)[N], const float (&a)[N], const float (&b)[N], const float (&c)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const float2 r = fma2({a[j], a[j + 1]}, {b[j], b[j + 1]}, {c[j], c[j + 1]});
    d[j] = r.x;
    d[j + 1] = r.y;
  }
}
template <int N>
__device__ __forceinline__ void mul_all(float (&d)[N], const float (&a)[N], const float (&b)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const float2 r = mul2({a[j], a[j + 1]}, {b[j], b[j + 1]});
    d[j] = r.x;
    d[j + 1] = r.y;
  }
}
template <int N>
__device__ __forceinline__ void mul_all(float (&d)[N], const float (&a)[N], float b) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const float2 r = mul2({a[j], a[j + 1]}, {b, b});
    d[j] = r.x;
    d[j + 1] = r.y;
  }
}

template <typename T>
struct Piece {
  static constexpr int V = 16 / sizeof(T);
  float x[V];
  __device__ __forceinline__ void set(uint4 raw) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ void take(uint32_t at) {
    uint4 w;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
    set(w);
  }
  __device__ __forceinline__ uint4 get() const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(x[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// V codes of a piece, one behind the other.  int8: adding 1.5 * 2^23 rounds to a whole number, ties to even, and leaves it in
// the low byte; a product is at most 127 (1 + 2^-23).
template <int V>
__device__ __forceinline__ void store_codes(void *to, const float *x, float by, int type) {
  uint32_t w[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const float *const y = x + 4 * i;
    if (type == LAPIS_I8) {
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(y[j], by), 12582912.0f));
      w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0] * by, y[1] * by), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2] * by, y[3] * by), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | hi << 16;
    }
  }
  if constexpr (V == 8) *static_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
  else *static_cast<uint32_t *>(to) = w[0];
}
// The values of V codes.  int8: 2^23 + 128 + code is a float with the biased code in its low byte.
template <int V>
__device__ __forceinline__ void values_of(float *x, uint2 raw, float scale, int type) {
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const uint32_t w = i == 0 ? raw.x : raw.y;
    if (type == LAPIS_I8) {
      const uint32_t u = w ^ 0x80808080u;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + j)) - 8388736.0f;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (8 * j)), __NV_E4M3)));
        x[4 * i + j] = f.x;
        x[4 * i + j + 1] = f.y;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const float2 f = mul2({x[4 * i + j], x[4 * i + j + 1]}, {scale, scale});
      x[4 * i + j] = f.x;
      x[4 * i + j + 1] = f.y;
    }
  }
}

// N floats from an address that is a multiple of their size, up to 16 bytes.
template <int N>
__device__ __forceinline__ void load_floats(float (&x)[N], const float *from) {
  if constexpr (N == 2) {
    const float2 f = *reinterpret_cast<const float2 *>(from);
    x[0] = f.x;
    x[1] = f.y;
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 f = *reinterpret_cast<const float4 *>(from + j);
      x[j] = f.x;
      x[j + 1] = f.y;
      x[j + 2] = f.z;
      x[j + 3] = f.w;
    }
  }
}

// The two pieces of a row that a lane holds: the halves of pairs, and what is not turned two by two.
template <typename T, int LANES>
struct Pieces {
  static constexpr int V = Piece<T>::V;
  int at[2];
  bool in[2], turned;
  __device__ __forceinline__ Pieces(int dim, int half) {
    const int lane = threadIdx.x % LANES, apart = half / V;
    turned = lane < apart;
    at[0] = turned ? lane : 2 * lane;
    at[1] = turned ? lane + apart : 2 * lane + 1;
    in[0] = at[0] * V < dim;
    in[1] = at[1] * V < dim;
  }
};

// Cosines and sines of a lane's V pairs: (piece 0, piece 1) value by value, or, interleaved, neighbours in piece 0, then in piece 1.
template <typename T, int LANES>
struct Turn {
  static constexpr int V = Piece<T>::V;
  float c[V], s[V];
  __device__ __forceinline__ void load(const RotateArgs &a, const Pieces<T, LANES> &p, int64_t place, bool real) {
    const int half = a.rot / 2;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      c[j] = 1.0f;
      s[j] = 0.0f;
    }
    if (!real) return;
    const int64_t line = place * half;
    if (!a.interleaved) {
      if (!p.turned) return;
      load_floats(c, a.cos + line + p.at[0] * V);
      load_floats(s, a.sin + line + p.at[0] * V);
      return;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (p.at[k] * V >= a.rot) continue;
      float ct[V / 2], st[V / 2];
      load_floats(ct, a.cos + line + p.at[k] * (V / 2));
      load_floats(st, a.sin + line + p.at[k] * (V / 2));
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        c[k * (V / 2) + j] = ct[j];
        s[k * (V / 2) + j] = st[j];
      }
    }
  }
};

template <typename T, int LANES>
__device__ __forceinline__ void load_weights(const RotateArgs &a, int which, const Pieces<T, LANES> &p, float (&w)[2][Piece<T>::V]) {
  constexpr int V = Piece<T>::V;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) w[k][j] = 0.0f;
    if (!p.in[k]) continue;
    if (a.weight_f32) {
      load_floats(w[k], static_cast<const float *>(a.weight[which]) + p.at[k] * V);
    } else {
      Piece<T> x;
      x.set(*reinterpret_cast<const uint4 *>(static_cast<const T *>(a.weight[which]) + p.at[k] * V));
#pragma unroll
      for (int j = 0; j < V; ++j) w[k][j] = x.x[j];
    }
  }
}

// The rows of a token that a warp walks, kind by kind, as they are sent on their way: KINDS kinds of ARRAYS arrays each.  A
// lane's pieces lie at slot * 1024 * ARRAYS + i * 1024 + k * 512 of its place in the ring.
template <typename T, int LANES, int KINDS, int ARRAYS>
struct Supply {
  static constexpr int GROUPS = 32 / LANES;
  const char *at[ARRAYS];
  int64_t step[ARRAYS];
  int kind, round, rounds, head, heads, left;

  __device__ __forceinline__ void enter(const RotateArgs &a, const Rows *const (&rows)[ARRAYS], int64_t token) {
    heads = a.heads[kind];
    rounds = (heads + GROUPS - 1) / GROUPS;
    head = round * GROUPS + threadIdx.x % 32 / LANES;
#pragma unroll
    for (int i = 0; i < ARRAYS; ++i) {
      const Rows &r = rows[i][kind];
      at[i] = static_cast<const char *>(r.d) + (token * r.token_stride + head * r.head_stride) * (int)sizeof(T);
      step[i] = GROUPS * r.head_stride * (int)sizeof(T);
    }
  }
  // Round `from` of all of them is the first one.
  __device__ __forceinline__ void begin(const RotateArgs &a, const Rows *const (&rows)[ARRAYS], int64_t token, int from, int count) {
    round = from;
    left = count;
    for (kind = 0; kind < KINDS - 1; ++kind) {
      const int n = (a.heads[kind] + GROUPS - 1) / GROUPS;
      if (round < n) break;
      round -= n;
    }
    enter(a, rows, token);
  }
  // Sends the next round to `to`, this lane's place in a slot of the ring; commits in any case.
  __device__ __forceinline__ void send(const RotateArgs &a, const Rows *const (&rows)[ARRAYS], const Pieces<T, LANES> &p, int64_t token, uint32_t to) {
    if (left > 0) {
      --left;
#pragma unroll
      for (int i = 0; i < ARRAYS; ++i) {
#pragma unroll
        for (int k = 0; k < 2; ++k) bring(to + i * 1024 + k * 512, at[i] + (head < heads && p.in[k] ? p.at[k] * 16 : 0), head < heads && p.in[k]);
        at[i] += step[i];
      }
      head += GROUPS;
      if (++round == rounds && left > 0) {
        do {
          round = 0;
          ++kind;
          enter(a, rows, token);
        } while (rounds == 0);
      }
    }
    brought();
  }
};

// Rounds [from, to) of one kind: the rows come out of the ring, results go to `out`.
template <typename T, int LANES, int DEPTH, bool NORM, bool CODES, typename Next>
__device__ __forceinline__ void rotate_rows(const RotateArgs &a, const Pieces<T, LANES> &p, int count, int from, int to,
                                            const float (&wc)[2][Piece<T>::V], const float (&ws)[2][Piece<T>::V], char *out, int64_t out_stride,
                                            float *scales, int64_t scale_stride, bool real, uint32_t ring, int &slot, Next next) {
  constexpr int V = Piece<T>::V, GROUPS = 32 / LANES, PIECE = CODES ? V : 16;
  const int group = threadIdx.x % 32 / LANES;
  const float by_dim = 1.0f / (float)a.dim;
  int head = from * GROUPS + group;
  out += head * out_stride;
  if (CODES) scales += head * scale_stride;
  for (int round = from; round < to; ++round) {
    wait_for_all_but<DEPTH - 1>();
    const uint32_t row = ring + slot * 1024;
    Piece<T> x[2];
    x[0].take(row);
    x[1].take(row + 512);
    next(row);
    slot = slot + 1 == DEPTH ? 0 : slot + 1;
    if constexpr (NORM) {
      float2 pair = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < V; j += 2) pair = fma2({x[k].x[j], x[k].x[j + 1]}, {x[k].x[j], x[k].x[j + 1]}, pair);
      float sum = pair.x + pair.y;
#pragma unroll
      for (int d = LANES / 2; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float r = rsqrtf(fmaf(sum, by_dim, a.eps));
      float y[2][V];
      if (a.interleaved) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            const float2 t = mul2({x[k].x[j + 1], x[k].x[j]}, {ws[k][j], ws[k][j + 1]});
            const float2 u = fma2({x[k].x[j], x[k].x[j + 1]}, {wc[k][j], wc[k][j + 1]}, t);
            y[k][j] = u.x;
            y[k][j + 1] = u.y;
          }
      } else {
        mul_all(y[0], x[1].x, ws[0]);
        fma_all(y[0], x[0].x, wc[0], y[0]);
        mul_all(y[1], x[0].x, ws[1]);
        fma_all(y[1], x[1].x, wc[1], y[1]);
      }
      mul_all(x[0].x, y[0], r);
      mul_all(x[1].x, y[1], r);
      if (!real) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[0].x[j] = x[1].x[j] = 0.0f;
      }
    }
    if constexpr (CODES) {
      float most = 0.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) most = max_nan(most, fabsf(x[k].x[j]));
#pragma unroll
      for (int d = LANES / 2; d > 0; d /= 2) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, d));
      const float big = largest_code(a.cache.type);
      if (head < count && threadIdx.x % LANES == 0) *scales = scale_of(most, big);
      if (most < SMALL_ROW) {
        most *= RAISE;
        mul_all(x[0].x, x[0].x, RAISE);
        mul_all(x[1].x, x[1].x, RAISE);
      }
      const float by = most == 0.0f ? 0.0f : big / most;
      if (head < count) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (p.in[k]) store_codes<V>(out + p.at[k] * PIECE, x[k].x, by, a.cache.type);
      }
      scales += GROUPS * scale_stride;
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (head < count && p.in[k]) *reinterpret_cast<uint4 *>(out + p.at[k] * PIECE) = x[k].get();
    }
    head += GROUPS;
    out += GROUPS * out_stride;
  }
}

// A warp takes `each` of the rounds of one token: those of the queries come first, then the keys', then the values'.  CACHE: keys
// and values go to the cache, CODES: as codes.
template <typename T, int LANES, bool NORM, bool CACHE, bool CODES>
__global__ void __launch_bounds__(ROW_THREADS) rotate_kernel(const __grid_constant__ RotateArgs a, int parts, int each) {
  constexpr int V = Piece<T>::V, GROUPS = 32 / LANES, DEPTH = 4, KINDS = CACHE ? 3 : 2;
  __shared__ __align__(16) unsigned char rings[ROW_WARPS][DEPTH * 1024];
  const int64_t task = (int64_t)blockIdx.x * ROW_WARPS + threadIdx.x / 32, token = task / parts;
  if (token >= a.tokens) return;
  pdl_wait();
  const uint32_t ring = shared_at(rings[threadIdx.x / 32]) + threadIdx.x % 32 * 16;
  const Pieces<T, LANES> p(a.dim, NORM && !a.interleaved ? a.rot / 2 : 0);
  int from = (int)(task - token * parts) * each, rounds[KINDS], all = 0;
#pragma unroll
  for (int which = 0; which < KINDS; ++which) all += rounds[which] = (a.heads[which] + GROUPS - 1) / GROUPS;
  int to = min(from + each, all);
  const Rows *const rows[1] = {a.in};
  Supply<T, LANES, KINDS, 1> supply;
  supply.begin(a, rows, token, from, to - from);
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) supply.send(a, rows, p, token, ring + i * 1024);
  const int64_t place = load_index(a.place, token, a.idx_bytes);
  const bool real = !NORM || (place >= 0 && place < a.places);
  int64_t first_row = -1;
  if (CACHE && real && to > rounds[0]) first_row = cache_row(a.cache, a.lists, load_index(a.row, token, a.idx_bytes), place, a.page_shift);
  int slot = 0;
  auto next = [&](uint32_t free) { supply.send(a, rows, p, token, free); };
#pragma unroll
  for (int which = 0; which < KINDS; ++which) {
    if (from < rounds[which] && to > 0) {
      if (CACHE && which > 0 && first_row < 0) {  // nowhere to write
        wait_for_all_but<0>();
        return;
      }
      float wc[2][V], ws[2][V];
      if (NORM && which < 2) {
        Turn<T, LANES> turn;
        turn.load(a, p, place, real);
        load_weights(a, which, p, wc);
        if (a.interleaved) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) ws[k][j] = wc[k][j ^ 1] * (j % 2 == 0 ? -turn.s[k * (V / 2) + j / 2] : turn.s[k * (V / 2) + j / 2]);
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) wc[k][j] *= turn.c[k * (V / 2) + j / 2];
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            ws[0][j] = wc[1][j] * -turn.s[j];
            ws[1][j] = wc[0][j] * turn.s[j];
            wc[0][j] *= turn.c[j];
            wc[1][j] *= turn.c[j];
          }
        }
      }
      const int lo = max(from, 0), hi = min(to, rounds[which]);
      if (which == 0 || !CACHE) {
        rotate_rows<T, LANES, DEPTH, NORM, false>(a, p, a.heads[which], lo, hi, wc, ws,
                                                  static_cast<char *>(a.out[which]) + token * a.heads[which] * a.dim * (int)sizeof(T),
                                                  a.dim * (int)sizeof(T), nullptr, 0, real, ring, slot, next);
      } else {
        const int size = CODES ? 1 : sizeof(T);
        char *const store = static_cast<char *>(which == 1 ? a.cache.d_k : a.cache.d_v) + first_row * a.dim * size;
        float *const scales = CODES ? (which == 1 ? a.cache.d_k_scale : a.cache.d_v_scale) + first_row : nullptr;
        const int64_t stride = a.cache.page_size * a.dim * size;
        if (which == 1)
          rotate_rows<T, LANES, DEPTH, NORM, CODES>(a, p, a.heads[1], lo, hi, wc, ws, store, stride, scales, a.cache.page_size, true, ring, slot, next);
        else
          rotate_rows<T, LANES, DEPTH, false, CODES>(a, p, a.heads[2], lo, hi, wc, ws, store, stride, scales, a.cache.page_size, true, ring, slot, next);
      }
    }
    from -= rounds[which];
    to -= rounds[which];
  }
  pdl_release();
}

// Backward: warps take tokens a grid apart and keep their share of the weights' gradients in registers.  The warps' lane groups
// are added in order by the block, the blocks by rotate_weights_kernel.
constexpr int backward_blocks(int size) { return size == 4 ? 4 : 3; }  // an SM, by registers
template <typename T, int LANES>
__global__ void __launch_bounds__(ROW_THREADS, backward_blocks(sizeof(T))) rotate_backward_kernel(const __grid_constant__ RotateArgs a, int parts, int each) {
  constexpr int V = Piece<T>::V, GROUPS = 32 / LANES, DEPTH = 3;
  __shared__ __align__(16) unsigned char rings[ROW_WARPS][DEPTH * 2048];
  __shared__ float shares[ROW_THREADS / LANES][LANES * 2 * V];
  const uint32_t ring = shared_at(rings[threadIdx.x / 32]) + threadIdx.x % 32 * 16;
  const Pieces<T, LANES> p(a.dim, a.interleaved ? 0 : a.rot / 2);
  float dw[2][2][V];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[0][k][j] = dw[1][k][j] = 0.0f;
  const float by_dim = 1.0f / (float)a.dim;
  const int64_t tasks = a.tokens * parts;
  const int rounds[2] = {(a.heads[0] + GROUPS - 1) / GROUPS, (a.heads[1] + GROUPS - 1) / GROUPS};
  const Rows *const rows[2] = {a.in, a.grad};
  pdl_wait();
  for (int64_t task = (int64_t)blockIdx.x * ROW_WARPS + threadIdx.x / 32; task < tasks; task += (int64_t)gridDim.x * ROW_WARPS) {
    const int64_t token = task / parts;
    int from = (int)(task - token * parts) * each, to = min(from + each, rounds[0] + rounds[1]);
    Supply<T, LANES, 2, 2> supply;
    supply.begin(a, rows, token, from, to - from);
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) supply.send(a, rows, p, token, ring + i * 2048);
    const int64_t place = load_index(a.place, token, a.idx_bytes);
    const bool real = place >= 0 && place < a.places;
    Turn<T, LANES> turn;
    turn.load(a, p, place, real);
    int slot = 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int lo = max(from, 0), hi = min(to, rounds[which]);
      from -= rounds[which];
      to -= rounds[which];
      if (lo >= hi) continue;
      float weight[2][V];
      load_weights(a, which, p, weight);
      int head = lo * GROUPS + threadIdx.x % 32 / LANES;
      char *out = static_cast<char *>(a.out[which]) + (token * a.heads[which] + head) * a.dim * (int)sizeof(T);
      for (int round = lo; round < hi; ++round) {
        wait_for_all_but<DEPTH - 1>();
        const uint32_t row = ring + slot * 2048;
        Piece<T> x[2], dy[2];
        x[0].take(row);
        x[1].take(row + 512);
        dy[0].take(row + 1024);
        dy[1].take(row + 1536);
        supply.send(a, rows, p, token, row);
        slot = slot + 1 == DEPTH ? 0 : slot + 1;
        if (!real) {
#pragma unroll
          for (int j = 0; j < V; ++j) x[0].x[j] = x[1].x[j] = dy[0].x[j] = dy[1].x[j] = 0.0f;
        }
        float dn[2][V], g[2][V], part[V];
        if (a.interleaved) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < V; j += 2) {
              const float c = turn.c[k * (V / 2) + j / 2], s = turn.s[k * (V / 2) + j / 2];
              dn[k][j] = fmaf(dy[k].x[j], c, dy[k].x[j + 1] * s);
              dn[k][j + 1] = fmaf(dy[k].x[j + 1], c, -(dy[k].x[j] * s));
            }
        } else {
          mul_all(dn[0], dy[1].x, turn.s);
          fma_all(dn[0], dy[0].x, turn.c, dn[0]);
          mul_all(part, dy[0].x, turn.s);
          mul_all(dn[1], dy[1].x, turn.c);
#pragma unroll
          for (int j = 0; j < V; ++j) dn[1][j] -= part[j];
        }
        float2 squares = {0.0f, 0.0f}, products = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          mul_all(g[k], dn[k], weight[k]);
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            squares = fma2({x[k].x[j], x[k].x[j + 1]}, {x[k].x[j], x[k].x[j + 1]}, squares);
            products = fma2({g[k][j], g[k][j + 1]}, {x[k].x[j], x[k].x[j + 1]}, products);
          }
        }
        float sum = squares.x + squares.y, inner = products.x + products.y;
#pragma unroll
        for (int d = LANES / 2; d > 0; d /= 2) {
          sum += __shfl_xor_sync(0xffffffffu, sum, d);
          inner += __shfl_xor_sync(0xffffffffu, inner, d);
        }
        // What is no row, padding or beside the last head, is zeros and adds nothing; with an eps of zero its 1 / sqrt(0) would.
        const float eps = real && head < a.heads[which] ? a.eps : 1.0f;
        const float r = rsqrtf(fmaf(sum, by_dim, eps)), back = -inner * by_dim * r * r;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          mul_all(x[k].x, x[k].x, r);
          fma_all(dw[which][k], dn[k], x[k].x, dw[which][k]);
          mul_all(g[k], g[k], r);
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            const float2 t = fma2({x[k].x[j], x[k].x[j + 1]}, {back, back}, {g[k][j], g[k][j + 1]});
            x[k].x[j] = t.x;
            x[k].x[j + 1] = t.y;
          }
          if (head < a.heads[which] && p.in[k]) *reinterpret_cast<uint4 *>(out + p.at[k] * 16) = x[k].get();
        }
        head += GROUPS;
        out += GROUPS * a.dim * (int)sizeof(T);
      }
    }
  }
  pdl_release();
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (p.in[k]) {
#pragma unroll
        for (int j = 0; j < V; ++j) shares[threadIdx.x / LANES][p.at[k] * V + j] = which ? dw[1][k][j] : dw[0][k][j];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += ROW_THREADS) {
      float sum = 0.0f;
#pragma unroll
      for (int g = 0; g < ROW_THREADS / LANES; ++g) sum += shares[g][i];
      a.partial[((int64_t)blockIdx.x * 2 + which) * a.dim + i] = sum;
    }
  }
}

// Keys and values of listed tokens: a warp takes `each` rounds of a token's heads, two neighbouring pieces a lane; the cache's
// rows are codes or T.
template <typename T, int LANES, bool CODES>
__global__ void __launch_bounds__(ROW_THREADS)
kv_read_kernel(const __grid_constant__ lapis_b200_kv_cache cache, const __grid_constant__ lapis_b200_page_lists lists, int64_t tokens, const void *row,
               const void *place, int page_shift, int parts, int each, T *k, T *v) {
  constexpr int V = Piece<T>::V, GROUPS = 32 / LANES, SIZE = CODES ? 1 : sizeof(T);
  const int64_t task = (int64_t)blockIdx.x * ROW_WARPS + threadIdx.x / 32, token = task / parts;
  if (token >= tokens) return;
  const int lane = threadIdx.x % LANES, dim = (int)cache.dim, heads = (int)cache.heads;
  const int from = (int)(task - token * parts) * each, to = min(from + each, (heads + GROUPS - 1) / GROUPS);
  pdl_wait();
  const int64_t first = cache_row(cache, lists, load_index(row, token, lists.idx_bytes), load_index(place, token, lists.idx_bytes), page_shift);
  const bool in[2] = {2 * lane * V < dim, (2 * lane + 1) * V < dim}, wide = dim % (2 * V) == 0;
  int head = from * GROUPS + threadIdx.x % 32 / LANES;
  const int64_t at = (max(first, (int64_t)0) + head * cache.page_size), step = GROUPS * cache.page_size;
  const int64_t bytes = (at * dim + 2 * lane * V) * SIZE, byte_step = step * dim * SIZE, out = (token * heads + head) * dim + 2 * lane * V;
  const char *rows[2] = {static_cast<const char *>(cache.d_k) + bytes, static_cast<const char *>(cache.d_v) + bytes};
  const float *scales[2] = {cache.d_k_scale + at, cache.d_v_scale + at};
  T *to_rows[2] = {k + out, v + out};
  for (int round = from; round < to; ++round) {
    uint4 raw[2][2];
    float scale[2];
    const bool mine = head < heads, real = first >= 0 && mine;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      raw[w][0] = raw[w][1] = make_uint4(0, 0, 0, 0);
      if (CODES) {
        scale[w] = real ? *scales[w] : 0.0f;
        scales[w] += step;
        uint32_t c[4] = {0, 0, 0, 0};
        if (real && wide && in[0]) {  // both pieces in one
          if constexpr (V == 8) {
            const uint4 x = *reinterpret_cast<const uint4 *>(rows[w]);
            c[0] = x.x;
            c[1] = x.y;
            c[2] = x.z;
            c[3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(rows[w]);
            c[0] = x.x;
            c[1] = x.y;
          }
        } else if (real) {  // a row that begins at a multiple of one piece only
#pragma unroll
          for (int i = 0; i < 2 * V / 4; ++i)
            if (in[i / (V / 4)]) c[i] = reinterpret_cast<const uint32_t *>(rows[w])[i];
        }
        raw[w][0] = make_uint4(c[0], c[1], c[2], c[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (real && in[i]) raw[w][i] = reinterpret_cast<const uint4 *>(rows[w])[i];
      }
      rows[w] += byte_step;
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if constexpr (CODES) {
        const uint4 r = raw[w][0];
        Piece<T> p[2];
        if constexpr (V == 8) {
          values_of<V>(p[0].x, make_uint2(r.x, r.y), scale[w], cache.type);
          values_of<V>(p[1].x, make_uint2(r.z, r.w), scale[w], cache.type);
        } else {
          values_of<V>(p[0].x, make_uint2(r.x, 0), scale[w], cache.type);
          values_of<V>(p[1].x, make_uint2(r.y, 0), scale[w], cache.type);
        }
        raw[w][0] = p[0].get();
        raw[w][1] = p[1].get();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (mine && in[i]) reinterpret_cast<uint4 *>(to_rows[w])[i] = raw[w][i];
      to_rows[w] += GROUPS * dim;
    }
    head += GROUPS;
  }
  pdl_release();
}

// ---- host -------------------------------------------------------------------

int check_cache(const char *what, const lapis_b200_kv_cache *c) {
  if (c == nullptr) return fail(LAPIS_EBADARG, "%s: null cache", what);
  if (!is_float_type(c->type) && !is_quantised(c->type)) return fail(LAPIS_EBADARG, "%s: unknown type of the cache", what);
  if (c->pages < 0 || c->heads < 1 || c->page_size < 1 || c->dim < 1) return fail(LAPIS_EBADSHAPE, "%s: bad sizes of the cache", what);
  if (c->dim > KV_MAX_DIM) return fail(LAPIS_ETOOBIG, "%s: heads of more than %d values", what, KV_MAX_DIM);
  if (c->page_size > (1 << 20) || c->heads > (1 << 16) || c->pages > 0xffffffffLL / (c->heads * c->page_size))
    return fail(LAPIS_ETOOBIG, "%s: more than 2^32 - 1 rows in the cache", what);
  if (c->pages > 0 && (c->d_k == nullptr || c->d_v == nullptr)) return fail(LAPIS_EBADARG, "%s: null cache arrays", what);
  if (c->pages > 0 && is_quantised(c->type) && (c->d_k_scale == nullptr || c->d_v_scale == nullptr))
    return fail(LAPIS_EBADARG, "%s: a quantised cache needs scales", what);
  return LAPIS_OK;
}

int check_lists(const char *what, const lapis_b200_page_lists *l) {
  if (l == nullptr) return fail(LAPIS_EBADARG, "%s: null page lists", what);
  if (l->idx_bytes != 4 && l->idx_bytes != 8) return fail(LAPIS_EBADARG, "%s: idx_bytes must be 4 or 8", what);
  if (l->rows < 0 || l->entries < 0) return fail(LAPIS_EBADSHAPE, "%s: negative size of the page lists", what);
  if (l->rows > 0 && l->d_pos == nullptr) return fail(LAPIS_EBADARG, "%s: null pos", what);
  if (l->entries > 0 && l->d_crd == nullptr) return fail(LAPIS_EBADARG, "%s: null crd", what);
  return LAPIS_OK;
}

static int check_heads(const char *what, const char *name, const lapis_b200_heads *h, int64_t tokens) {
  if (h == nullptr) return fail(LAPIS_EBADARG, "%s: null description of %s", what, name);
  if (h->heads < 0 || h->heads > (1 << 16)) return fail(LAPIS_EBADSHAPE, "%s: bad number of heads of %s", what, name);
  if (tokens > 0 && h->heads > 0 && h->d == nullptr) return fail(LAPIS_EBADARG, "%s: null %s", what, name);
  return LAPIS_OK;
}

static int check_how(const char *what, int type, int64_t dim, const lapis_b200_norm_rope *how, RotateArgs *a) {
  if (how == nullptr) return fail(LAPIS_EBADARG, "%s: null weights and tables", what);
  if (how->rot < 0 || how->rot > dim || how->rot % 2 != 0) return fail(LAPIS_EBADSHAPE, "%s: rot must be even and at most dim", what);
  if (how->places < 0) return fail(LAPIS_EBADSHAPE, "%s: negative length of the tables", what);
  if (how->weight_type != LAPIS_F32 && how->weight_type != type) return fail(LAPIS_EBADARG, "%s: weights must be float32 or of the rows' type", what);
  if (how->d_q_weight == nullptr || how->d_k_weight == nullptr) return fail(LAPIS_EBADARG, "%s: null weights", what);
  if (how->rot > 0 && how->places > 0 && (how->d_cos == nullptr || how->d_sin == nullptr)) return fail(LAPIS_EBADARG, "%s: null tables", what);
  if (!(how->eps >= 0.0)) return fail(LAPIS_EBADARG, "%s: eps must not be negative", what);
  a->norm = 1;
  a->rot = (int)how->rot;
  a->interleaved = how->interleaved != 0;
  a->weight[0] = how->d_q_weight;
  a->weight[1] = how->d_k_weight;
  a->weight_f32 = how->weight_type == LAPIS_F32;
  a->cos = how->d_cos;
  a->sin = how->d_sin;
  a->places = how->places;
  a->eps = (float)how->eps;
  return LAPIS_OK;
}

static int check_sizes(const char *what, int type, int64_t tokens, int64_t dim, int64_t heads) {
  if (!is_float_type(type)) return fail(LAPIS_EBADARG, "%s: rows must be float32, float16 or bfloat16", what);
  if (tokens < 0 || dim < 1) return fail(LAPIS_EBADSHAPE, "%s: bad sizes", what);
  if (dim > KV_MAX_DIM) return fail(LAPIS_ETOOBIG, "%s: heads of more than %d values", what, KV_MAX_DIM);
  if (heads > 0 && tokens > 0x7fffffffLL / heads) return fail(LAPIS_ETOOBIG, "%s: more than 2^31 - 1 rows", what);
  return LAPIS_OK;
}

static Rows rows_of(const lapis_b200_heads *h) { return {h->d, h->token_stride, h->head_stride}; }

template <typename F>
static int with_type(int type, F run) {
  if (type == LAPIS_F32) return run(float());
  if (type == LAPIS_F16) return run(__half());
  return run(__nv_bfloat16());
}

static bool aligned(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
static bool aligned(const Rows &r, int size) {
  return aligned(r.d, 16) && r.token_stride * size % 16 == 0 && r.head_stride * size % 16 == 0;
}
// Whether 16-byte pieces fit the rows of a type, the pairs of their rotation and all arrays; rows that they do not fit are taken
// value by value (8192 tokens of 32 + 8 heads of 128: 196 us, not 31; backward of 16,384 669, not 85).
static bool pieces_fit(int type, const RotateArgs &a, bool backward) {
  const int size = type_bytes(type), v = 16 / size;
  if (a.dim % v != 0) return false;
  if (a.norm && (a.interleaved ? a.rot % v != 0 : a.rot / 2 % v != 0)) return false;
  if (a.norm && !(aligned(a.cos, 16) && aligned(a.sin, 16) && aligned(a.weight[0], 16) && aligned(a.weight[1], 16))) return false;
  for (int w = 0; w < 3; ++w)
    if (a.heads[w] > 0 && !aligned(a.in[w], size)) return false;
  for (int w = 0; w < 2; ++w)
    if (a.heads[w] > 0 && ((backward && !aligned(a.grad[w], size)) || !aligned(a.out[w], 16))) return false;
  return !a.to_cache || (aligned(a.cache.d_k, 16) && aligned(a.cache.d_v, 16));
}

// Calls run(LANES) as a compile-time number: two pieces a lane of rows of `dim` values.
template <typename T, typename F>
static int with_lanes(int dim, F run) {
  using std::integral_constant;
  const int pairs = (dim / Piece<T>::V + 1) / 2;
  if constexpr (KV_MAX_DIM / Piece<T>::V / 2 > 16)
    if (pairs > 16) return run(integral_constant<int, 32>());
  if (pairs <= 4) return run(integral_constant<int, 4>());
  if (pairs <= 8) return run(integral_constant<int, 8>());
  return run(integral_constant<int, 16>());
}

// How the rounds of a token are shared out: few tokens are cut into parts, down to a round, so that there are eight warps' work for
// every SM's scheduler; many are walked by one warp each, since every part looks its token up again: with four times as many parts
// 8192 tokens take 39 us, not 31, and 5003 tokens of 5 heads written as e4m3 and read 22.8, not 18.5.
struct Parts {
  int parts, each;
  unsigned blocks;
};
static Parts parts_of(int64_t tokens, int rounds) {
  const int64_t wanted = 32LL * sm_count();
  Parts p;
  p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(rounds, (wanted + tokens - 1) / tokens));
  p.each = (rounds + p.parts - 1) / p.parts;
  p.parts = (rounds + p.each - 1) / p.each;
  p.blocks = (unsigned)((tokens * p.parts + ROW_WARPS - 1) / ROW_WARPS);
  return p;
}

static int launch_rotate(int type, const RotateArgs &a, cudaStream_t st) {
  const int64_t rows = a.tokens * (a.heads[0] + a.heads[1] + a.heads[2]);
  if (rows == 0) return LAPIS_OK;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    if (!pieces_fit(type, a, false)) {
      rotate_any_kernel<T><<<(unsigned)((rows + ROW_WARPS - 1) / ROW_WARPS), ROW_THREADS, 0, st>>>(a);
      LAPIS_CUDA_TRY(cudaGetLastError());
      return (int)LAPIS_OK;
    }
    return with_lanes<T>(a.dim, [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value, GROUPS = 32 / LANES;
      int rounds = 0;
      for (int heads : a.heads) rounds += (heads + GROUPS - 1) / GROUPS;
      const Parts p = parts_of(a.tokens, rounds);
      cudaError_t launched;
      if (!a.to_cache) launched = launch_pdl(rotate_kernel<T, LANES, true, false, false>, dim3(p.blocks), ROW_THREADS, 0, st, a, p.parts, p.each);
      else if (a.norm && is_quantised(a.cache.type)) launched = launch_pdl(rotate_kernel<T, LANES, true, true, true>, dim3(p.blocks), ROW_THREADS, 0, st, a, p.parts, p.each);
      else if (a.norm) launched = launch_pdl(rotate_kernel<T, LANES, true, true, false>, dim3(p.blocks), ROW_THREADS, 0, st, a, p.parts, p.each);
      else if (is_quantised(a.cache.type)) launched = launch_pdl(rotate_kernel<T, LANES, false, true, true>, dim3(p.blocks), ROW_THREADS, 0, st, a, p.parts, p.each);
      else launched = launch_pdl(rotate_kernel<T, LANES, false, true, false>, dim3(p.blocks), ROW_THREADS, 0, st, a, p.parts, p.each);
      LAPIS_CUDA_TRY(launched);
      return (int)LAPIS_OK;
    });
  });
}

// Launches the backward kernel that fits and leaves in *blocks how many shares of the weights' gradients there are.
static int launch_backward(int type, RotateArgs &a, PoolBuf &partial, int *blocks, cudaStream_t st) {
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    auto room = [&](int64_t wanted) {
      *blocks = (int)std::min<int64_t>(wanted, backward_blocks(sizeof(T)) * sm_count());  // what is resident
      const int status = partial.alloc((size_t)*blocks * 2 * a.dim * sizeof(float), st);
      a.partial = static_cast<float *>(partial.p);
      return status;
    };
    if (!pieces_fit(type, a, true)) {
      LAPIS_TRY(room((a.tokens + ROW_WARPS - 1) / ROW_WARPS));
      if (*blocks > 0) rotate_any_backward_kernel<T><<<*blocks, ROW_THREADS, 0, st>>>(a);
      LAPIS_CUDA_TRY(cudaGetLastError());
      return (int)LAPIS_OK;
    }
    return with_lanes<T>(a.dim, [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value, GROUPS = 32 / LANES;
      const int rounds = (a.heads[0] + GROUPS - 1) / GROUPS + (a.heads[1] + GROUPS - 1) / GROUPS;
      const Parts p = a.tokens > 0 && rounds > 0 ? parts_of(a.tokens, rounds) : Parts{1, 1, 0};
      LAPIS_TRY(room(p.blocks));
      if (*blocks > 0) LAPIS_CUDA_TRY(launch_pdl(rotate_backward_kernel<T, LANES>, dim3(*blocks), ROW_THREADS, 0, st, a, p.parts, p.each));
      return (int)LAPIS_OK;
    });
  });
}

}  // namespace lapis_b200

using namespace lapis_b200;

extern "C" int lapis_b200_qk_norm_rope(int type, int64_t tokens, int64_t dim, const lapis_b200_heads *q, const lapis_b200_heads *k,
                                       const lapis_b200_norm_rope *how, int idx_bytes, const void *d_place, void *d_q_out,
                                       void *d_k_out, void *stream) {
  clear_error();
  const char *what = "qk_norm_rope";
  LAPIS_TRY(check_heads(what, "q", q, tokens));
  LAPIS_TRY(check_heads(what, "k", k, tokens));
  LAPIS_TRY(check_sizes(what, type, tokens, dim, q->heads + k->heads));
  RotateArgs a = {};
  LAPIS_TRY(check_how(what, type, dim, how, &a));
  if (idx_bytes != 4 && idx_bytes != 8) return fail(LAPIS_EBADARG, "%s: idx_bytes must be 4 or 8", what);
  if (tokens > 0 && (d_place == nullptr || (q->heads > 0 && d_q_out == nullptr) || (k->heads > 0 && d_k_out == nullptr)))
    return fail(LAPIS_EBADARG, "%s: null operand", what);
  a.tokens = tokens;
  a.dim = (int)dim;
  a.heads[0] = (int)q->heads;
  a.heads[1] = (int)k->heads;
  a.in[0] = rows_of(q);
  a.in[1] = rows_of(k);
  a.out[0] = d_q_out;
  a.out[1] = d_k_out;
  a.idx_bytes = idx_bytes;
  a.place = d_place;
  return launch_rotate(type, a, as_stream(stream));
}

extern "C" int lapis_b200_qk_norm_rope_backward(int type, int64_t tokens, int64_t dim, const lapis_b200_heads *dq,
                                                const lapis_b200_heads *dk, const lapis_b200_heads *q, const lapis_b200_heads *k,
                                                const lapis_b200_norm_rope *how, int idx_bytes, const void *d_place, void *d_q_grad,
                                                void *d_k_grad, float *d_q_weight_grad, float *d_k_weight_grad, void *stream) {
  clear_error();
  const char *what = "qk_norm_rope_backward";
  LAPIS_TRY(check_heads(what, "q", q, tokens));
  LAPIS_TRY(check_heads(what, "k", k, tokens));
  LAPIS_TRY(check_heads(what, "dq", dq, tokens));
  LAPIS_TRY(check_heads(what, "dk", dk, tokens));
  if (dq->heads != q->heads || dk->heads != k->heads) return fail(LAPIS_EBADSHAPE, "%s: gradients of another number of heads", what);
  LAPIS_TRY(check_sizes(what, type, tokens, dim, q->heads + k->heads));
  RotateArgs a = {};
  LAPIS_TRY(check_how(what, type, dim, how, &a));
  if (idx_bytes != 4 && idx_bytes != 8) return fail(LAPIS_EBADARG, "%s: idx_bytes must be 4 or 8", what);
  if (d_q_weight_grad == nullptr || d_k_weight_grad == nullptr ||
      (tokens > 0 && (d_place == nullptr || (q->heads > 0 && d_q_grad == nullptr) || (k->heads > 0 && d_k_grad == nullptr))))
    return fail(LAPIS_EBADARG, "%s: null operand", what);
  a.tokens = tokens;
  a.dim = (int)dim;
  a.heads[0] = (int)q->heads;
  a.heads[1] = (int)k->heads;
  a.in[0] = rows_of(q);
  a.in[1] = rows_of(k);
  a.grad[0] = rows_of(dq);
  a.grad[1] = rows_of(dk);
  a.out[0] = d_q_grad;
  a.out[1] = d_k_grad;
  a.idx_bytes = idx_bytes;
  a.place = d_place;
  cudaStream_t st = as_stream(stream);
  int blocks = 0;
  PoolBuf partial;
  LAPIS_TRY(launch_backward(type, a, partial, &blocks, st));
  LAPIS_CUDA_TRY(launch_pdl(rotate_weights_kernel, dim3((unsigned)((dim + 31) / 32), 2), 1024, 0, st, a.partial, blocks, (int)dim, d_q_weight_grad, d_k_weight_grad));
  return LAPIS_OK;
}

extern "C" int lapis_b200_kv_append(int type, int64_t tokens, const lapis_b200_heads *q, const lapis_b200_heads *k,
                                    const lapis_b200_heads *v, const lapis_b200_norm_rope *how, const lapis_b200_kv_cache *cache,
                                    const lapis_b200_page_lists *lists, const void *d_row, const void *d_place, void *d_q_out,
                                    void *stream) {
  clear_error();
  const char *what = "kv_append";
  LAPIS_TRY(check_cache(what, cache));
  LAPIS_TRY(check_lists(what, lists));
  LAPIS_TRY(check_heads(what, "k", k, tokens));
  LAPIS_TRY(check_heads(what, "v", v, tokens));
  if (how != nullptr) LAPIS_TRY(check_heads(what, "q", q, tokens));
  const int64_t q_heads = how != nullptr ? q->heads : 0;
  LAPIS_TRY(check_sizes(what, type, tokens, cache->dim, q_heads + k->heads + v->heads));
  if (k->heads != cache->heads || v->heads != cache->heads) return fail(LAPIS_EBADSHAPE, "%s: the cache has another number of heads", what);
  if (!is_quantised(cache->type) && cache->type != type) return fail(LAPIS_EBADARG, "%s: rows of another type than the cache", what);
  RotateArgs a = {};
  if (how != nullptr) LAPIS_TRY(check_how(what, type, cache->dim, how, &a));
  if (tokens > 0 && (d_row == nullptr || d_place == nullptr || (q_heads > 0 && d_q_out == nullptr)))
    return fail(LAPIS_EBADARG, "%s: null operand", what);
  a.tokens = tokens;
  a.dim = (int)cache->dim;
  a.heads[0] = (int)q_heads;
  a.heads[1] = (int)k->heads;
  a.heads[2] = (int)v->heads;
  if (q_heads > 0) a.in[0] = rows_of(q);
  a.in[1] = rows_of(k);
  a.in[2] = rows_of(v);
  a.out[0] = d_q_out;
  a.idx_bytes = lists->idx_bytes;
  a.place = d_place;
  a.row = d_row;
  a.to_cache = 1;
  a.cache = *cache;
  a.page_shift = page_shift_of(cache->page_size);
  a.lists = *lists;
  return launch_rotate(type, a, as_stream(stream));
}

extern "C" int lapis_b200_kv_read(const lapis_b200_kv_cache *cache, const lapis_b200_page_lists *lists, int64_t tokens,
                                  const void *d_row, const void *d_place, int type, void *d_k, void *d_v, void *stream) {
  clear_error();
  const char *what = "kv_read";
  LAPIS_TRY(check_cache(what, cache));
  LAPIS_TRY(check_lists(what, lists));
  LAPIS_TRY(check_sizes(what, type, tokens, cache->dim, cache->heads));
  if (tokens == 0) return LAPIS_OK;
  if (d_row == nullptr || d_place == nullptr || d_k == nullptr || d_v == nullptr) return fail(LAPIS_EBADARG, "%s: null operand", what);
  const int size = type_bytes(type);
  const bool pieces = cache->dim * size % 16 == 0 && (is_quantised(cache->type) || cache->type == type) && aligned(cache->d_k, 16) &&
                      aligned(cache->d_v, 16) && aligned(d_k, 16) && aligned(d_v, 16);
  cudaStream_t st = as_stream(stream);
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    T *const k = static_cast<T *>(d_k), *const v = static_cast<T *>(d_v);
    if (!pieces) {
      kv_read_any_kernel<T><<<(unsigned)((tokens * cache->heads + ROW_WARPS - 1) / ROW_WARPS), ROW_THREADS, 0, st>>>(*cache, *lists, tokens, d_row, d_place, k, v);
      LAPIS_CUDA_TRY(cudaGetLastError());
      return (int)LAPIS_OK;
    }
    return with_lanes<T>((int)cache->dim, [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value, GROUPS = 32 / LANES;
      const Parts p = parts_of(tokens, (int)((cache->heads + GROUPS - 1) / GROUPS));
      const int shift = page_shift_of(cache->page_size);
      if (is_quantised(cache->type))
        LAPIS_CUDA_TRY(launch_pdl(kv_read_kernel<T, LANES, true>, dim3(p.blocks), ROW_THREADS, 0, st, *cache, *lists, tokens, d_row, d_place, shift, p.parts, p.each, k, v));
      else
        LAPIS_CUDA_TRY(launch_pdl(kv_read_kernel<T, LANES, false>, dim3(p.blocks), ROW_THREADS, 0, st, *cache, *lists, tokens, d_row, d_place, shift, p.parts, p.each, k, v));
      return (int)LAPIS_OK;
    });
  });
}

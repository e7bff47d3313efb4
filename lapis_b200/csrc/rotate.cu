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
  const int64_t first_row = cache_row(a.cache, a.lists, load_index(a.row, token, a.idx_bytes), place);
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
  const float big = largest_code(a.cache.type), by = most == 0.0f ? 0.0f : big / most;
  if (lane == 0) (which == 1 ? a.cache.d_k_scale : a.cache.d_v_scale)[row] = scale_of(most, big);
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
        const float r = 1.0f / sqrtf(warp_sum(sum) / (float)a.dim + a.eps);
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
  const int i = blockIdx.x * 32 + threadIdx.x, which = blockIdx.y;
  float sum = 0.0f;
  if (i < dim)
    for (int b = threadIdx.y; b < blocks; b += 32) sum += partial[((int64_t)b * 2 + which) * dim + i];
  sums[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && i < dim) {
    for (int b = 1; b < 32; ++b) sum += sums[b][threadIdx.x];
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
  const int64_t first = cache_row(cache, lists, load_index(row, token, lists.idx_bytes), load_index(place, token, lists.idx_bytes));
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
// Bound by memory: every element is read and written once.  A row is held by LANES neighbouring lanes, CHUNKS pieces of 16
// bytes each; the sums over a row and the partners of its rotation are shuffles among them.  A block takes up to ROWS rows a
// lane group of one token, so that the weights and the token's line of the tables are read once for all of them, and has all
// their loads in flight together.

template <typename T>
struct Piece {
  static constexpr int V = 16 / sizeof(T);
  float x[V];
  __device__ __forceinline__ void set(uint4 raw) {
    if constexpr (sizeof(T) == 4) {
      x[0] = __uint_as_float(raw.x);
      x[1] = __uint_as_float(raw.y);
      x[2] = __uint_as_float(raw.z);
      x[3] = __uint_as_float(raw.w);
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        } else {
          x[2 * i] = __uint_as_float(w[i] << 16);
          x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
  }
  __device__ __forceinline__ uint4 get() const {
    if constexpr (sizeof(T) == 4) {
      return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// V codes of a piece, as bytes one behind the other.
template <int V>
__device__ __forceinline__ void store_codes(void *to, const float *x, float by, int type) {
  uint32_t w[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    w[i] = 0;
    if (type == LAPIS_I8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i] |= (uint32_t)(uint8_t)to_i8(x[4 * i + j] * by) << (8 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j += 2)
        w[i] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + j] * by, x[4 * i + j + 1] * by), __NV_SATFINITE, __NV_E4M3) << (8 * j);
    }
  }
  if constexpr (V == 8) *static_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
  else *static_cast<uint32_t *>(to) = w[0];
}
template <int V>
__device__ __forceinline__ void load_codes(float *x, const void *from, int type) {
  uint32_t w[V / 4];
  if constexpr (V == 8) {
    const uint2 raw = *static_cast<const uint2 *>(from);
    w[0] = raw.x;
    w[1] = raw.y;
  } else {
    w[0] = *static_cast<const uint32_t *>(from);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint8_t c = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
    x[i] = type == LAPIS_I8 ? (float)(int8_t)c : from_e4m3(c);
  }
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d /= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
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

// The cosines and sines that a lane's pieces are turned by, and where the partners are: for pairs of halves the same place of
// another piece, `apart` pieces away (negative: this is the second half, whose sine counts the other way).
template <typename T, int LANES, int CHUNKS>
struct Turn {
  static constexpr int V = Piece<T>::V;
  float c[CHUNKS][V], s[CHUNKS][V];
  int from[CHUNKS];  // piece of the partner

  // back: the other way round, for gradients.  Pieces that are not turned have cosine 1 and sine 0.
  __device__ __forceinline__ void load(const RotateArgs &a, int64_t place, int lane, bool back) {
    const int half = a.rot / 2;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      const int piece = lane + k * LANES, i = piece * V;
      from[k] = piece;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        c[k][j] = 1.0f;
        s[k][j] = 0.0f;
      }
      if (i >= a.rot) continue;
      const bool second = !a.interleaved && i >= half;
      const float *const cs = a.cos + place * half + (a.interleaved ? i / 2 : second ? i - half : i);
      const float *const sn = a.sin + (cs - a.cos);
      if (!a.interleaved) from[k] = second ? piece - half / V : piece + half / V;
      // first of a pair: a cos - b sin; second: b cos + a sin
      if (a.interleaved) {
        float ct[V / 2], st[V / 2];
        load_floats(ct, cs);
        load_floats(st, sn);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[k][j] = ct[j / 2];
          s[k][j] = (j % 2 == 1) != back ? st[j / 2] : -st[j / 2];
        }
      } else {
        load_floats(c[k], cs);
        load_floats(s[k], sn);
#pragma unroll
        for (int j = 0; j < V; ++j) s[k][j] = second != back ? s[k][j] : -s[k][j];
      }
    }
  }
  // y = x turned.
  __device__ __forceinline__ void apply(const RotateArgs &a, const float (&x)[CHUNKS][V], float (&y)[CHUNKS][V]) const {
    if (a.interleaved) {
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) y[k][j] = fmaf(x[k][j], c[k][j], x[k][j ^ 1] * s[k][j]);
      return;
    }
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float other = __shfl_sync(0xffffffffu, x[0][j], from[k] % LANES, LANES);
#pragma unroll
        for (int q = 1; q < CHUNKS; ++q) {
          const float there = __shfl_sync(0xffffffffu, x[q][j], from[k] % LANES, LANES);
          other = from[k] / LANES == q ? there : other;
        }
        y[k][j] = fmaf(x[k][j], c[k][j], other * s[k][j]);
      }
    }
  }
};

template <typename T, int LANES, int CHUNKS>
__device__ __forceinline__ void load_weights(const RotateArgs &a, int which, int lane, float (&w)[CHUNKS][Piece<T>::V]) {
  constexpr int V = Piece<T>::V;
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k) {
    const int i = (lane + k * LANES) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) w[k][j] = 0.0f;
    if (i >= a.dim) continue;
    if (a.weight_f32) {
      load_floats(w[k], static_cast<const float *>(a.weight[which]) + i);
    } else {
      Piece<T> p;
      p.set(*reinterpret_cast<const uint4 *>(static_cast<const T *>(a.weight[which]) + i));
#pragma unroll
      for (int j = 0; j < V; ++j) w[k][j] = p.x[j];
    }
  }
}

template <typename T, int LANES, int CHUNKS, int ROWS>
__global__ void __launch_bounds__(ROW_THREADS) rotate_kernel(const __grid_constant__ RotateArgs a) {
  constexpr int V = Piece<T>::V, GROUPS = ROW_THREADS / LANES;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int64_t token = blockIdx.x;
  const int all = a.heads[0] + a.heads[1] + a.heads[2], first = blockIdx.y * GROUPS * ROWS + group;
  uint4 raw[ROWS][CHUNKS];
  int which[ROWS], head[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int row = first + u * GROUPS;
    which[u] = row < a.heads[0] ? 0 : row < a.heads[0] + a.heads[1] ? 1 : row < all ? 2 : -1;
    head[u] = row - (which[u] > 0 ? a.heads[0] : 0) - (which[u] > 1 ? a.heads[1] : 0);
    const Rows &in = a.in[which[u] < 0 ? 0 : which[u]];
    const T *const from = static_cast<const T *>(in.d) + token * in.token_stride + head[u] * in.head_stride;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      const int i = (lane + k * LANES) * V;
      raw[u][k] = which[u] >= 0 && i < a.dim ? *reinterpret_cast<const uint4 *>(from + i) : make_uint4(0, 0, 0, 0);
    }
  }
  const int64_t place = load_index(a.place, token, a.idx_bytes);
  const bool real = !a.norm || (place >= 0 && place < a.places);
  Turn<T, LANES, CHUNKS> turn;
  float weight[2][CHUNKS][V];
  if (a.norm && real) {
    turn.load(a, place, lane, false);
    load_weights<T, LANES, CHUNKS>(a, 0, lane, weight[0]);
    load_weights<T, LANES, CHUNKS>(a, 1, lane, weight[1]);
  }
  int64_t first_row = -1;
  if (a.to_cache && real && blockIdx.y * GROUPS * ROWS + GROUPS * ROWS > a.heads[0])
    first_row = cache_row(a.cache, a.lists, load_index(a.row, token, a.idx_bytes), place);
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    if (first - group + u * GROUPS >= all) break;  // the whole block is through
    const bool turned = which[u] >= 0 && which[u] < 2 && a.norm && real;
    float x[CHUNKS][V], y[CHUNKS][V];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      Piece<T> p;
      p.set(raw[u][k]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[k][j] = real ? p.x[j] : 0.0f;
        y[k][j] = x[k][j];
        sum = fmaf(x[k][j], x[k][j], sum);
      }
    }
    if (a.norm && real) {  // all lanes: a group's rows may be of two kinds, a warp's groups too
      const float r = 1.0f / sqrtf(lanes_sum<LANES>(sum) / (float)a.dim + a.eps);
      float n[CHUNKS][V], z[CHUNKS][V];
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) n[k][j] = x[k][j] * r * (which[u] == 1 ? weight[1][k][j] : weight[0][k][j]);
      turn.apply(a, n, z);
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) y[k][j] = turned ? z[k][j] : y[k][j];
    }
    float most = 0.0f;
    const bool codes = a.to_cache && is_quantised(a.cache.type);
    if (codes) {
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) most = max_nan(most, fabsf(y[k][j]));
#pragma unroll
      for (int d = LANES / 2; d > 0; d /= 2) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, d));
    }
    if (which[u] < 0) continue;
    if (which[u] == 0 || !a.to_cache) {
      T *const out = static_cast<T *>(a.out[which[u]]) + (token * a.heads[which[u]] + head[u]) * a.dim;
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int i = (lane + k * LANES) * V;
        Piece<T> p;
#pragma unroll
        for (int j = 0; j < V; ++j) p.x[j] = y[k][j];
        if (i < a.dim) *reinterpret_cast<uint4 *>(out + i) = p.get();
      }
      continue;
    }
    if (first_row < 0) continue;
    const int64_t row = first_row + head[u] * a.cache.page_size;
    void *const store = which[u] == 1 ? a.cache.d_k : a.cache.d_v;
    const float big = largest_code(a.cache.type), by = most == 0.0f ? 0.0f : big / most;
    if (codes && lane == 0) (which[u] == 1 ? a.cache.d_k_scale : a.cache.d_v_scale)[row] = scale_of(most, big);
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      const int i = (lane + k * LANES) * V;
      if (i >= a.dim) continue;
      if (codes) {
        store_codes<V>(static_cast<char *>(store) + row * a.dim + i, y[k], by, a.cache.type);
      } else {
        Piece<T> p;
#pragma unroll
        for (int j = 0; j < V; ++j) p.x[j] = y[k][j];
        *reinterpret_cast<uint4 *>(static_cast<T *>(store) + row * a.dim + i) = p.get();
      }
    }
  }
}

// Backward: blocks take tokens a grid apart, a lane group rows of a token, and a lane keeps its share of the weights' gradients.
// The lane groups of a block are added in order, the blocks by rotate_weights_kernel.
template <typename T, int LANES, int CHUNKS, int ROWS>
__global__ void __launch_bounds__(ROW_THREADS) rotate_backward_kernel(const __grid_constant__ RotateArgs a) {
  constexpr int V = Piece<T>::V, GROUPS = ROW_THREADS / LANES;
  __shared__ float shares[GROUPS][LANES * CHUNKS * V];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  float weight[2][CHUNKS][V], dw[2][CHUNKS][V];
  load_weights<T, LANES, CHUNKS>(a, 0, lane, weight[0]);
  load_weights<T, LANES, CHUNKS>(a, 1, lane, weight[1]);
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[0][k][j] = dw[1][k][j] = 0.0f;
  const int all = a.heads[0] + a.heads[1];
  for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
    const int64_t place = load_index(a.place, token, a.idx_bytes);
    const bool real = place >= 0 && place < a.places;
    Turn<T, LANES, CHUNKS> turn;
    turn.load(a, real ? place : 0, lane, true);
    for (int row0 = 0; row0 < all; row0 += GROUPS * ROWS) {
      uint4 raw[ROWS][2][CHUNKS];
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int row = row0 + u * GROUPS + group, which = row >= a.heads[0], head = row - (which ? a.heads[0] : 0);
        const T *const x = static_cast<const T *>(a.in[which].d) + token * a.in[which].token_stride + head * a.in[which].head_stride;
        const T *const dy = static_cast<const T *>(a.grad[which].d) + token * a.grad[which].token_stride + head * a.grad[which].head_stride;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
          const int i = (lane + k * LANES) * V;
          const bool in = row < all && i < a.dim && real;
          raw[u][0][k] = in ? *reinterpret_cast<const uint4 *>(x + i) : make_uint4(0, 0, 0, 0);
          raw[u][1][k] = in ? *reinterpret_cast<const uint4 *>(dy + i) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        if (row0 + u * GROUPS >= all) break;
        const int row = row0 + u * GROUPS + group, which = row >= a.heads[0], head = row - (which ? a.heads[0] : 0);
        float x[CHUNKS][V], dy[CHUNKS][V], dn[CHUNKS][V];
        float sum = 0.0f, inner = 0.0f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
          Piece<T> p, q;
          p.set(raw[u][0][k]);
          q.set(raw[u][1][k]);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            x[k][j] = p.x[j];
            dy[k][j] = q.x[j];
          }
        }
        turn.apply(a, dy, dn);
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            sum = fmaf(x[k][j], x[k][j], sum);
            inner = fmaf(dn[k][j] * (which ? weight[1][k][j] : weight[0][k][j]), x[k][j], inner);
          }
#pragma unroll
        for (int d = LANES / 2; d > 0; d /= 2) {
          sum += __shfl_xor_sync(0xffffffffu, sum, d);
          inner += __shfl_xor_sync(0xffffffffu, inner, d);
        }
        const float r = 1.0f / sqrtf(sum / (float)a.dim + a.eps), back = inner / (float)a.dim * r * r;
        T *const out = static_cast<T *>(a.out[which]) + (token * a.heads[which] + head) * a.dim;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
          const int i = (lane + k * LANES) * V;
          Piece<T> p;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float t = dn[k][j] * x[k][j] * r;
            if (which) dw[1][k][j] += t;
            else dw[0][k][j] += t;
            p.x[j] = r * (dn[k][j] * (which ? weight[1][k][j] : weight[0][k][j]) - x[k][j] * back);
          }
          if (row < all && i < a.dim) *reinterpret_cast<uint4 *>(out + i) = p.get();
        }
      }
    }
  }
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) shares[group][(lane + k * LANES) * V + j] = which ? dw[1][k][j] : dw[0][k][j];
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += ROW_THREADS) {
      float sum = 0.0f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) sum += shares[g][i];
      a.partial[((int64_t)blockIdx.x * 2 + which) * a.dim + i] = sum;
    }
  }
}

// Keys and values of listed tokens, a lane group a head of TOKENS tokens; the cache's rows are codes or T.
template <typename T, int LANES, int CHUNKS, int TOKENS>
__global__ void __launch_bounds__(ROW_THREADS)
kv_read_kernel(const __grid_constant__ lapis_b200_kv_cache cache, const __grid_constant__ lapis_b200_page_lists lists, int64_t tokens, const void *row, const void *place, T *k, T *v) {
  constexpr int V = Piece<T>::V, GROUPS = ROW_THREADS / LANES;
  const int lane = threadIdx.x % LANES, head = blockIdx.y * GROUPS + threadIdx.x / LANES;
  if (head >= cache.heads) return;
  const bool codes = is_quantised(cache.type);
  const int dim = (int)cache.dim;
  int64_t at[TOKENS];
#pragma unroll
  for (int u = 0; u < TOKENS; ++u) {
    const int64_t token = (int64_t)blockIdx.x * TOKENS + u;
    at[u] = token < tokens ? cache_row(cache, lists, load_index(row, token, lists.idx_bytes), load_index(place, token, lists.idx_bytes)) : -1;
    if (at[u] >= 0) at[u] += head * cache.page_size;
  }
  Piece<T> got[TOKENS][2][CHUNKS];
#pragma unroll
  for (int u = 0; u < TOKENS; ++u)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const void *const store = w == 0 ? cache.d_k : cache.d_v;
      float scale = 1.0f;
      if (codes && at[u] >= 0) scale = (w == 0 ? cache.d_k_scale : cache.d_v_scale)[at[u]];
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int i = (lane + c * LANES) * V;
        Piece<T> &p = got[u][w][c];
#pragma unroll
        for (int j = 0; j < V; ++j) p.x[j] = 0.0f;
        if (at[u] < 0 || i >= dim) continue;
        if (codes) {
          load_codes<V>(p.x, static_cast<const char *>(store) + at[u] * dim + i, cache.type);
#pragma unroll
          for (int j = 0; j < V; ++j) p.x[j] *= scale;
        } else {
          p.set(*reinterpret_cast<const uint4 *>(static_cast<const T *>(store) + at[u] * dim + i));
        }
      }
    }
#pragma unroll
  for (int u = 0; u < TOKENS; ++u) {
    const int64_t token = (int64_t)blockIdx.x * TOKENS + u;
    if (token >= tokens) break;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int i = (lane + c * LANES) * V;
        if (i < dim) *reinterpret_cast<uint4 *>((w == 0 ? k : v) + (token * cache.heads + head) * dim + i) = got[u][w][c].get();
      }
  }
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
// Whether 16-byte pieces fit the rows of a type, the pairs of their rotation and all arrays.
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

// Calls run(LANES, CHUNKS) as compile-time numbers for rows of `dim` values.
template <typename T, typename F>
static int with_lanes(int dim, F run) {
  using std::integral_constant;
  const int pieces = dim / Piece<T>::V;
  if (pieces <= 4) return run(integral_constant<int, 4>(), integral_constant<int, 1>());
  if (pieces <= 8) return run(integral_constant<int, 8>(), integral_constant<int, 1>());
  if (pieces <= 16) return run(integral_constant<int, 16>(), integral_constant<int, 1>());
  if constexpr (KV_MAX_DIM / Piece<T>::V > 32)
    if (pieces > 32) return run(integral_constant<int, 32>(), integral_constant<int, 2>());
  return run(integral_constant<int, 32>(), integral_constant<int, 1>());
}

static int launch_rotate(int type, const RotateArgs &a, cudaStream_t st) {
  const int64_t heads = a.heads[0] + a.heads[1] + a.heads[2], rows = a.tokens * heads;
  if (rows == 0) return LAPIS_OK;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    if (!pieces_fit(type, a, false)) {
      rotate_any_kernel<T><<<(unsigned)((rows + ROW_WARPS - 1) / ROW_WARPS), ROW_THREADS, 0, st>>>(a);
      LAPIS_CUDA_TRY(cudaGetLastError());
      return (int)LAPIS_OK;
    }
    return with_lanes<T>(a.dim, [&](auto lanes, auto chunks) {
      constexpr int LANES = decltype(lanes)::value, CHUNKS = decltype(chunks)::value, GROUPS = ROW_THREADS / LANES;
      // few tokens: a block for each round of rows
      if (a.tokens * heads <= (int64_t)GROUPS * 4 * sm_count()) {
        rotate_kernel<T, LANES, CHUNKS, 1><<<dim3((unsigned)a.tokens, (unsigned)((heads + GROUPS - 1) / GROUPS)), ROW_THREADS, 0, st>>>(a);
      } else {
        constexpr int ROWS = CHUNKS == 1 ? 4 : 2;
        rotate_kernel<T, LANES, CHUNKS, ROWS><<<dim3((unsigned)a.tokens, (unsigned)((heads + GROUPS * ROWS - 1) / (GROUPS * ROWS))), ROW_THREADS, 0, st>>>(a);
      }
      LAPIS_CUDA_TRY(cudaGetLastError());
      return (int)LAPIS_OK;
    });
  });
}

// Launches the backward kernel that fits and leaves in *blocks how many shares of the weights' gradients there are.
static int launch_backward(int type, RotateArgs &a, PoolBuf &partial, int *blocks, cudaStream_t st) {
  const bool pieces = pieces_fit(type, a, true);
  const int most = 8 * sm_count();
  *blocks = (int)std::min<int64_t>(pieces ? a.tokens : (a.tokens + ROW_WARPS - 1) / ROW_WARPS, most);
  LAPIS_TRY(partial.alloc((size_t)*blocks * 2 * a.dim * sizeof(float), st));
  a.partial = static_cast<float *>(partial.p);
  if (*blocks == 0) return LAPIS_OK;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    if (!pieces) {
      rotate_any_backward_kernel<T><<<*blocks, ROW_THREADS, 0, st>>>(a);
      LAPIS_CUDA_TRY(cudaGetLastError());
      return (int)LAPIS_OK;
    }
    return with_lanes<T>(a.dim, [&](auto lanes, auto chunks) {
      constexpr int LANES = decltype(lanes)::value, CHUNKS = decltype(chunks)::value;
      rotate_backward_kernel<T, LANES, CHUNKS, CHUNKS == 1 ? 2 : 1><<<*blocks, ROW_THREADS, 0, st>>>(a);
      LAPIS_CUDA_TRY(cudaGetLastError());
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
  rotate_weights_kernel<<<dim3((unsigned)((dim + 31) / 32), 2), dim3(32, 32), 0, st>>>(a.partial, blocks, (int)dim, d_q_weight_grad, d_k_weight_grad);
  LAPIS_CUDA_TRY(cudaGetLastError());
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
    return with_lanes<T>((int)cache->dim, [&](auto lanes, auto chunks) {
      constexpr int LANES = decltype(lanes)::value, CHUNKS = decltype(chunks)::value, GROUPS = ROW_THREADS / LANES;
      const unsigned rounds = (unsigned)((cache->heads + GROUPS - 1) / GROUPS);
      if (tokens * rounds <= 8LL * sm_count()) {
        kv_read_kernel<T, LANES, CHUNKS, 1><<<dim3((unsigned)tokens, rounds), ROW_THREADS, 0, st>>>(*cache, *lists, tokens, d_row, d_place, k, v);
      } else {
        constexpr int TOKENS = CHUNKS == 1 ? 4 : 2;
        kv_read_kernel<T, LANES, CHUNKS, TOKENS><<<dim3((unsigned)((tokens + TOKENS - 1) / TOKENS), rounds), ROW_THREADS, 0, st>>>(*cache, *lists, tokens, d_row, d_place, k, v);
      }
      LAPIS_CUDA_TRY(cudaGetLastError());
      return (int)LAPIS_OK;
    });
  });
}

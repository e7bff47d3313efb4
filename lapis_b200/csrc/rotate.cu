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

static int launch_rotate(int type, const RotateArgs &a, cudaStream_t st) {
  const int64_t rows = a.tokens * (a.heads[0] + a.heads[1] + a.heads[2]);
  if (rows == 0) return LAPIS_OK;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    rotate_any_kernel<T><<<(unsigned)((rows + ROW_WARPS - 1) / ROW_WARPS), ROW_THREADS, 0, st>>>(a);
    LAPIS_CUDA_TRY(cudaGetLastError());
    return (int)LAPIS_OK;
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
  const int blocks = (int)std::min<int64_t>((tokens + ROW_WARPS - 1) / ROW_WARPS, 8LL * sm_count());
  PoolBuf partial;
  LAPIS_TRY(partial.alloc((size_t)blocks * 2 * dim * sizeof(float), st));
  a.partial = static_cast<float *>(partial.p);
  if (blocks > 0) {
    LAPIS_TRY(with_type(type, [&](auto t) {
      using T = decltype(t);
      rotate_any_backward_kernel<T><<<blocks, ROW_THREADS, 0, st>>>(a);
      LAPIS_CUDA_TRY(cudaGetLastError());
      return (int)LAPIS_OK;
    }));
  }
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
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    kv_read_any_kernel<T><<<(unsigned)((tokens * cache->heads + ROW_WARPS - 1) / ROW_WARPS), ROW_THREADS, 0, as_stream(stream)>>>(
        *cache, *lists, tokens, d_row, d_place, static_cast<T *>(d_k), static_cast<T *>(d_v));
    LAPIS_CUDA_TRY(cudaGetLastError());
    return (int)LAPIS_OK;
  });
}

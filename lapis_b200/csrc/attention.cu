// Attention of one new token per request over a paged cache.
//
// For a request b of n tokens (of the last `window` of them, with one), a query head h and the keys k_j and values v_j of the
// key head h / group that serves it:
//   s_j = scale q.k_j,   out = sum_j exp(s_j - m) v_j / l,   m = max_j s_j,   l = sum_j exp(s_j - m),   lse = m + log l
// in one pass over the keys and values, with the running m and l of the softmax in 32 bits: what has been summed under an
// older m is scaled by exp(m_old - m_new).  A request without tokens gets zeros and lse = -inf.
//
// The work is the cache, which is read once.  It is cut along its length, whatever the lengths are: a unit is a request, a
// key head and up to HEADS of the query heads that share it, its keys are cut into tiles, and the tiles of all units, one
// after the other, are dealt to the blocks in equal, contiguous shares.  A unit that lies in one share is finished there; the
// others leave (m, l, sum) in a workspace and join_kernel adds them up in the order of the blocks, so that results are the
// same from run to run.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "kv.h"

namespace lapis_b200 {

constexpr int ATT_THREADS = 128;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct AttendArgs {
  const void *q;
  int64_t q_token_stride, q_head_stride;
  int requests, q_heads, group, head_blocks;  // group: query heads of a key head; head_blocks: units of a request and key head
  int dim;
  float scale2;  // scale * log2(e): the softmax is computed in powers of two
  int64_t window;
  lapis_b200_kv_cache cache;
  lapis_b200_page_lists lists;
  const void *length;
  void *out;
  float *lse;
  float *partial;  // [blocks][2][HEADS][dim + 2]
  int blocks, min_tiles;
};

// Keys [lo, hi) of request b that are attended.
struct Span {
  int64_t lo, hi;
};
__device__ __forceinline__ Span span_of(const AttendArgs &a, int64_t b) {
  const int64_t first = load_index(a.lists.d_pos, b, a.lists.idx_bytes), last = load_index(a.lists.d_pos, b + 1, a.lists.idx_bytes);
  const int64_t room = (last - first) * a.cache.page_size, n = load_index(a.length, b, a.lists.idx_bytes);
  Span s;
  s.hi = max((int64_t)0, min(n, room));
  s.lo = a.window > 0 ? max((int64_t)0, s.hi - a.window) : 0;
  return s;
}
// Tiles of a unit of a request; a request without tokens has one, which writes its zeros.
__device__ __forceinline__ int64_t tiles_of(const Span &s, int tile) { return max((int64_t)1, (s.hi - s.lo + tile - 1) / tile); }

// Where a share of the tiles begins: all threads of the block return the same.
struct Share {
  int64_t all;         // tiles of all units
  int64_t shares;      // blocks that get some
  int64_t from, to;    // this block's tiles
  int64_t request, in_request;  // the request of the first one, and its number among the request's
};
__device__ __forceinline__ int64_t share_start(int64_t i, int64_t all, int64_t shares) { return i * all / shares; }

// Sums the tiles of all requests (a thread takes a run of them), and finds the request of tile `at(all, shares)`.
template <typename At>
__device__ __forceinline__ Share find_share(const AttendArgs &a, int tile, At at) {
  __shared__ int64_t warp_sums[ATT_THREADS / 32], found[2];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, units = (int)a.cache.heads * a.head_blocks;
  const int run = (a.requests + ATT_THREADS - 1) / ATT_THREADS, first = threadIdx.x * run;
  int64_t sum = 0;
  for (int b = first; b < min(first + run, a.requests); ++b) sum += tiles_of(span_of(a, b), tile) * units;
  int64_t upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t below = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += below;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  Share s;
  s.all = 0;
  for (int w = 0; w < ATT_THREADS / 32; ++w) {
    if (w < warp) upto += warp_sums[w];
    s.all += warp_sums[w];
  }
  s.shares = max((int64_t)1, min((int64_t)a.blocks, s.all / a.min_tiles));
  s.from = at(s);
  s.to = s.from;
  if (s.from >= upto - sum && s.from < upto) {
    int64_t left = s.from - (upto - sum);
    for (int b = first; b < min(first + run, a.requests); ++b) {
      const int64_t n = tiles_of(span_of(a, b), tile) * units;
      if (left < n) {
        found[0] = b;
        found[1] = left;
        break;
      }
      left -= n;
    }
  }
  __syncthreads();
  s.request = found[0];
  s.in_request = found[1];
  __syncthreads();
  return s;
}

// ---- any type, width, stride and alignment --------------------------------------

constexpr int ANY_HEADS = 8, ANY_TILE = 32;

__host__ __device__ constexpr int any_smem(int dim) { return (ANY_HEADS * dim + 2 * ANY_TILE * (dim + 1) + ANY_HEADS * ANY_TILE + 2 * ANY_HEADS) * 4; }

// A block walks its tiles of 32 keys: keys and values to shared memory in 32 bits, a thread a key and two heads for the
// scores, a thread a dimension or two for the sums.
template <typename T>
__global__ void __launch_bounds__(ATT_THREADS) attend_any_kernel(const __grid_constant__ AttendArgs a) {
  extern __shared__ float smem[];
  const int dim = a.dim, pitch = dim + 1;
  float *const qs = smem, *const ks = qs + ANY_HEADS * dim, *const vs = ks + ANY_TILE * pitch, *const ps = vs + ANY_TILE * pitch;
  float *const factor = ps + ANY_HEADS * ANY_TILE, *const total = factor + ANY_HEADS;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Share s = find_share(a, ANY_TILE, [&](const Share &x) { return share_start(min((int64_t)blockIdx.x, x.shares - 1), x.all, x.shares); });
  if (blockIdx.x >= s.shares) return;
  s.to = share_start(blockIdx.x + 1, s.all, s.shares);
  int64_t request = s.request;
  Span span = span_of(a, request);
  int64_t tiles = tiles_of(span, ANY_TILE);
  int unit = (int)(s.in_request / tiles);
  int64_t tile = s.in_request % tiles;
  const int units = (int)a.cache.heads * a.head_blocks;
  for (int64_t at = s.from; at < s.to;) {
    const int kv_head = unit / a.head_blocks, head0 = (unit % a.head_blocks) * ANY_HEADS, heads = min(ANY_HEADS, a.group - head0);
    const int64_t end = min(tiles, tile + (s.to - at));
    __syncthreads();
    for (int i = threadIdx.x; i < heads * dim; i += ATT_THREADS)
      qs[i] = to_f32(static_cast<const T *>(a.q)[request * a.q_token_stride + (int64_t)(kv_head * a.group + head0 + i / dim) * a.q_head_stride + i % dim]);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, acc[2][ANY_HEADS] = {};
    for (int64_t t = tile; t < end; ++t) {
      const int64_t key0 = span.lo + t * ANY_TILE;
      __syncthreads();
      for (int j = warp; j < ANY_TILE; j += ATT_THREADS / 32) {
        const bool in = key0 + j < span.hi;
        const int64_t row0 = in ? cache_row(a.cache, a.lists, request, key0 + j) : -1, row = row0 + kv_head * a.cache.page_size;
        float kscale = 1.0f, vscale = 1.0f;
        if (row0 >= 0 && is_quantised(a.cache.type)) {
          kscale = a.cache.d_k_scale[row];
          vscale = a.cache.d_v_scale[row];
        }
        for (int i = lane; i < dim; i += 32) {
          ks[j * pitch + i] = row0 < 0 ? 0.0f : load_as_f32(a.cache.d_k, row * dim + i, a.cache.type) * kscale;
          vs[j * pitch + i] = row0 < 0 ? 0.0f : load_as_f32(a.cache.d_v, row * dim + i, a.cache.type) * vscale;
        }
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int h = warp + 4 * u;
        if (h >= heads) continue;
        float score = 0.0f;
        for (int i = 0; i < dim; ++i) score = fmaf(qs[h * dim + i], ks[lane * pitch + i], score);
        score = key0 + lane < span.hi ? score * a.scale2 : -INFINITY;
        float most = score;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        most = fmaxf(most, m[u]);
        const float base = most == -INFINITY ? 0.0f : most, p = exp2f(score - base), f = exp2f(m[u] - base);
        m[u] = most;
        l[u] = l[u] * f + p;
        ps[h * ANY_TILE + lane] = p;
        if (lane == 0) factor[h] = f;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = threadIdx.x + e * ATT_THREADS;
        if (i >= dim) continue;
#pragma unroll
        for (int h = 0; h < ANY_HEADS; ++h) {
          if (h >= heads) continue;
          float x = acc[e][h] * factor[h];
          for (int j = 0; j < ANY_TILE; ++j) x = fmaf(ps[h * ANY_TILE + j], vs[j * pitch + i], x);
          acc[e][h] = x;
        }
      }
    }
    const bool whole = tile == 0 && end == tiles;
    float *const slot = a.partial + ((int64_t)blockIdx.x * 2 + (at == s.from ? 0 : 1)) * ANY_HEADS * (dim + 2);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int h = warp + 4 * u;
      if (h >= heads) continue;
      float sum = l[u];
#pragma unroll
      for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane != 0) continue;
      total[h] = sum;
      if (whole && a.lse != nullptr)
        a.lse[request * a.q_heads + kv_head * a.group + head0 + h] = sum > 0.0f || sum != sum ? m[u] * LN2 + logf(sum) : -INFINITY;
      if (!whole) {
        slot[h * (dim + 2)] = m[u];
        slot[h * (dim + 2) + 1] = sum;
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = threadIdx.x + e * ATT_THREADS;
      if (i >= dim) continue;
#pragma unroll
      for (int h = 0; h < ANY_HEADS; ++h) {
        if (h >= heads) continue;
        if (whole)
          static_cast<T *>(a.out)[(request * a.q_heads + kv_head * a.group + head0 + h) * dim + i] = from_f32<T>(total[h] == 0.0f ? 0.0f : acc[e][h] / total[h]);
        else
          slot[h * (dim + 2) + 2 + i] = acc[e][h];
      }
    }
    at += end - tile;
    tile = 0;
    if (++unit == units && at < s.to) {
      unit = 0;
      span = span_of(a, ++request);
      tiles = tiles_of(span, ANY_TILE);
    }
  }
}

// Adds up what the blocks left of the units that were cut: block (unit, request), a thread a dimension or two of each head.
template <typename T>
__global__ void __launch_bounds__(ATT_THREADS) attend_join_kernel(const __grid_constant__ AttendArgs a, int tile_keys, int heads_of_unit) {
  const int64_t request = blockIdx.y;
  const int unit = blockIdx.x, dim = a.dim;
  int64_t before = 0;  // tiles of the requests in front
  const Span span = span_of(a, request);
  const int64_t tiles = tiles_of(span, tile_keys);
  const int units = (int)a.cache.heads * a.head_blocks;
  __shared__ int64_t sums[2][ATT_THREADS / 32];
  int64_t front = 0, all = 0;
  for (int b = threadIdx.x; b < a.requests; b += ATT_THREADS) {
    const int64_t n = tiles_of(span_of(a, b), tile_keys) * units;
    all += n;
    if (b < request) front += n;
  }
#pragma unroll
  for (int d = 16; d > 0; d /= 2) {
    all += __shfl_xor_sync(0xffffffffu, all, d);
    front += __shfl_xor_sync(0xffffffffu, front, d);
  }
  if (threadIdx.x % 32 == 0) {
    sums[0][threadIdx.x / 32] = front;
    sums[1][threadIdx.x / 32] = all;
  }
  __syncthreads();
  all = 0;
  for (int w = 0; w < ATT_THREADS / 32; ++w) {
    before += sums[0][w];
    all += sums[1][w];
  }
  const int64_t shares = max((int64_t)1, min((int64_t)a.blocks, all / a.min_tiles));
  const int64_t from = before + unit * tiles, to = from + tiles;
  // the last share that begins at or in front of a tile t: the largest i with i * all / shares < t + 1
  const int64_t first = ((from + 1) * shares + all - 1) / all - 1, last = (to * shares + all - 1) / all - 1;
  if (first == last) return;
  const int kv_head = unit / a.head_blocks, head0 = (unit % a.head_blocks) * heads_of_unit, heads = min(heads_of_unit, a.group - head0);
  for (int h = 0; h < heads; ++h) {
    auto slot = [&](int64_t i) {
      const int which = i > first || share_start(first, all, shares) == from ? 0 : 1;
      return a.partial + ((i * 2 + which) * heads_of_unit + h) * (dim + 2);
    };
    float most = -INFINITY, sum = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int64_t i = first; i <= last; ++i) most = fmaxf(most, slot(i)[0]);
    const float base = most == -INFINITY ? 0.0f : most;
    for (int64_t i = first; i <= last; ++i) {
      const float *p = slot(i);
      const float f = exp2f(p[0] - base);
      sum = fmaf(p[1], f, sum);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = threadIdx.x + e * ATT_THREADS;
        if (d < dim) acc[e] = fmaf(p[2 + d], f, acc[e]);
      }
    }
    const int64_t head = request * a.q_heads + kv_head * a.group + head0 + h;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = threadIdx.x + e * ATT_THREADS;
      if (d < dim) static_cast<T *>(a.out)[head * dim + d] = from_f32<T>(sum == 0.0f ? 0.0f : acc[e] / sum);
    }
    if (threadIdx.x == 0 && a.lse != nullptr) a.lse[head] = sum > 0.0f || sum != sum ? most * LN2 + logf(sum) : -INFINITY;
  }
}

template <typename T>
static int launch_any(AttendArgs a, int dev, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};  // devices on which this kernel may use its shared memory
  if ((allowed.load(std::memory_order_relaxed) >> dev & 1) == 0) {
    LAPIS_CUDA_TRY(cudaFuncSetAttribute(attend_any_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, any_smem(KV_MAX_DIM)));
    allowed.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  a.head_blocks = (a.group + ANY_HEADS - 1) / ANY_HEADS;
  a.blocks = 2 * sm_count();
  a.min_tiles = 4;
  PoolBuf partial;
  LAPIS_TRY(partial.alloc((size_t)a.blocks * 2 * ANY_HEADS * (a.dim + 2) * sizeof(float), st));
  a.partial = static_cast<float *>(partial.p);
  attend_any_kernel<T><<<a.blocks, ATT_THREADS, any_smem(a.dim), st>>>(a);
  LAPIS_CUDA_TRY(cudaGetLastError());
  attend_join_kernel<T><<<dim3((unsigned)(a.cache.heads * a.head_blocks), (unsigned)a.requests), ATT_THREADS, 0, st>>>(a, ANY_TILE, ANY_HEADS);
  LAPIS_CUDA_TRY(cudaGetLastError());
  return LAPIS_OK;
}

}  // namespace lapis_b200

using namespace lapis_b200;

extern "C" int lapis_b200_paged_attention(int type, int64_t requests, const lapis_b200_heads *q, const lapis_b200_kv_cache *cache,
                                          const lapis_b200_page_lists *lists, const void *d_length, double scale, int64_t window,
                                          void *d_out, float *d_lse, void *stream) {
  clear_error();
  const char *what = "paged_attention";
  LAPIS_TRY(check_cache(what, cache));
  LAPIS_TRY(check_lists(what, lists));
  if (!is_float_type(type)) return fail(LAPIS_EBADARG, "%s: q must be float32, float16 or bfloat16", what);
  if (!is_quantised(cache->type) && cache->type != type) return fail(LAPIS_EBADARG, "%s: q of another type than the cache", what);
  if (q == nullptr) return fail(LAPIS_EBADARG, "%s: null description of q", what);
  if (requests < 0 || q->heads < 1 || q->heads % cache->heads != 0)
    return fail(LAPIS_EBADSHAPE, "%s: the query heads must be a multiple of the cache's", what);
  if (requests > 65535 || q->heads > (1 << 16)) return fail(LAPIS_ETOOBIG, "%s: more than 65535 requests or 65536 heads", what);
  if (lists->rows != requests) return fail(LAPIS_EBADSHAPE, "%s: a page list for each request", what);
  if (window < 0) return fail(LAPIS_EBADARG, "%s: negative window", what);
  if (!std::isfinite(scale)) return fail(LAPIS_EBADARG, "%s: scale must be finite", what);
  if (requests == 0) return LAPIS_OK;
  if (q->d == nullptr || d_length == nullptr || d_out == nullptr) return fail(LAPIS_EBADARG, "%s: null operand", what);
  int dev = 0;
  LAPIS_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64) return fail(LAPIS_EBADARG, "%s: more than 64 devices", what);
  AttendArgs a = {};
  a.q = q->d;
  a.q_token_stride = q->token_stride;
  a.q_head_stride = q->head_stride;
  a.requests = (int)requests;
  a.q_heads = (int)q->heads;
  a.group = (int)(q->heads / cache->heads);
  a.dim = (int)cache->dim;
  a.scale2 = (float)(scale * 1.4426950408889634);
  a.window = window;
  a.cache = *cache;
  a.lists = *lists;
  a.length = d_length;
  a.out = d_out;
  a.lse = d_lse;
  cudaStream_t st = as_stream(stream);
  if (type == LAPIS_F32) return launch_any<float>(a, dev, st);
  if (type == LAPIS_F16) return launch_any<__half>(a, dev, st);
  return launch_any<__nv_bfloat16>(a, dev, st);
}

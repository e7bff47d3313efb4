// Attention of one new token per request over a paged cache.
//
// For a request b of n tokens (of the last `window` of them, with one), a query head h and the keys k_j and values v_j of the
// key head h / group that serves it:
//   s_j = scale q.k_j,   out = sum_j exp(s_j - m) v_j / l,   m = max_j s_j,   l = sum_j exp(s_j - m),   lse = m + log l
// in one pass over the keys and values, with the running m and l of the softmax in 32 bits: what has been summed under an
// older m is scaled by exp(m_old - m_new).  A request without tokens gets zeros and lse = -inf.
//
// The work is the cache, which is read once.  It is cut along its length, whatever the lengths are: a unit is a request, a
// key head and up to 8 or 16 of the query heads that share it, its keys are cut into tiles, and the tiles of all units, one
// after the other, are dealt to the blocks in equal, contiguous shares.  A unit that lies in one share is finished there; the
// others leave (m, l, sum) in a workspace, and a second kernel adds them up in a fixed order, so that results are the same from
// run to run.
//
// Three kernels share this, one for each way to multiply: attend_mma_kernel (16-bit queries, and 32-bit ones over codes),
// attend_f32_kernel (32 bits throughout), attend_any_kernel (rows that no copy of 8 bytes fits).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kv.h"

namespace lapis_b200 {

constexpr int ATT_THREADS = 128;
constexpr int UNIT_COST = 2;      // what a unit costs beside its tiles, in tiles: 128 x 8192 int8 214 us with 1, 204 with 2 or 3
// Of a share, if there is more than one: 2 x 3000 tokens of 256 take 12.5 us with 2, 17.7 with 3; 1 x 4000 of int8 12.9 and 13.3.
constexpr int MIN_WORK = 2;
// By which a unit may be longer than a share and is not cut: 1 x 300 tokens take 7.8 us with 6, 10.3 with 4 (and a join).
constexpr int WHOLE_TILES = 6;
constexpr int MOST_BLOCKS = 1 << 10;  // shares
constexpr float LN2 = 0.6931471805599453f;

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
  float *partial;     // what blocks leave of units that are cut: two pieces each
  struct Cut *cuts;   // one for each block
  int blocks;
  int page_shift;  // log2 of the slots of a page, or -1
  int q_pairs;     // two 16-bit values of q lie at a multiple of 4 bytes
};

// A request's tokens beyond these are not looked at: places are 32-bit numbers in the kernels.
constexpr int MOST_TOKENS = 0x7fff0000;

// Keys [lo, hi) of a request that are attended; its pages are crd[entry] onward.  Tiles begin at `origin`, lo rounded down to a
// multiple of 16, so that 16 keys of a tile lie in one page where that has a multiple of 16 slots.
struct Span {
  int lo, hi, origin;
  int64_t entry;
};
__device__ __forceinline__ Span span_of(const AttendArgs &a, int request) {
  // A list ends where the lists do, whatever pos says: no walk is longer than they are.
  const int64_t first = load_index(a.lists.d_pos, request, a.lists.idx_bytes), last = min(load_index(a.lists.d_pos, request + 1, a.lists.idx_bytes), a.lists.entries);
  const int64_t room = first < 0 || last <= first ? 0 : (last - first) * a.cache.page_size, n = load_index(a.length, request, a.lists.idx_bytes);
  Span s;
  s.hi = (int)max((int64_t)0, min(min(n, room), (int64_t)MOST_TOKENS));
  s.lo = a.window > 0 && a.window < s.hi ? s.hi - (int)a.window : 0;
  s.origin = s.lo & ~15;
  s.entry = first;
  return s;
}
// Tiles of a unit of a request; a request without tokens has one, which writes its zeros.
__device__ __forceinline__ int tiles_of(const Span &s, int tile) { return max(1, (s.hi - s.origin + tile - 1) / tile); }

// n * all / shares: where share n of the work begins.
__device__ __forceinline__ int64_t share_start(int n, int64_t all, int shares) {
  if (all < (1 << 22) && shares < (1 << 10)) return (uint32_t)n * (uint32_t)all / (uint32_t)shares;
  return n * all / shares;
}

// A block's way through its share.  The work of a unit is UNIT_COST, for its queries and its result, and one for each tile, in
// this order; all units lie one behind the other, and a share is a stretch of that line.  A unit's tile belongs to the share
// that it lies in.
struct Walk {
  int request, unit, tile, end, tiles;  // of this unit: the next tile, the first one that is not this share's, and how many it has
  int64_t left;                         // from the unit's beginning to the share's end
  Span span;
  bool done;

  __device__ __forceinline__ void enter(int tile_keys) {
    tiles = tiles_of(span, tile_keys);
    end = (int)min((int64_t)tiles, left - UNIT_COST);
    done = end <= tile;
  }
  __device__ __forceinline__ void next_unit(const AttendArgs &a, int units, int tile_keys) {
    left -= UNIT_COST + tiles;
    tile = 0;
    done = left <= UNIT_COST;
    if (done) return;
    if (++unit == units) {
      unit = 0;
      if (++request == a.requests) {
        done = true;
        return;
      }
      span = span_of(a, request);
    }
    enter(tile_keys);
  }
  __device__ __forceinline__ void next_tile(const AttendArgs &a, int units, int tile_keys) {
    if (++tile == end) next_unit(a, units, tile_keys);
  }
};

// A unit that is cut: its shares, where the first of them leaves its part (0: its first piece, 1: its last; the others' parts are
// their first), and which it is.  last = 0: there is none.
struct CutUnit {
  int first, last, slot, request, unit;
};
// What a block leaves for the join: the unit that begins in its share and goes on, and the one that its share goes on with.
struct Cut {
  CutUnit begins, goes_on;
};

struct Share {
  int64_t all, to;  // all work, and where this share ends
  int shares;
  // The share of position x: the largest n with n * all / shares < x + 1.
  __device__ __forceinline__ int of(int64_t x) const {
    if (all < (1 << 22) && shares < (1 << 10)) return (int)(((uint32_t)(x + 1) * (uint32_t)shares + (uint32_t)all - 1) / (uint32_t)all) - 1;
    return (int)(((x + 1) * shares + all - 1) / all) - 1;
  }
  // The unit of a walk.
  __device__ __forceinline__ CutUnit cut(const Walk &w) const {
    const int64_t at = to - w.left;  // where it begins
    const int first = of(at + UNIT_COST);
    return {first, of(at + UNIT_COST + w.tiles - 1), share_start(first, all, shares) < at ? 1 : 0, w.request, w.unit};
  }
};
// Notes what is cut of the piece [began, w.end) of a unit.
__device__ __forceinline__ void note_cut(const AttendArgs &a, const Share &share, const Walk &w, int began) {
  if (threadIdx.x != 0 || (began == 0 && w.end == w.tiles)) return;
  const CutUnit c = share.cut(w);
  if (began == 0) a.cuts[blockIdx.x].begins = c;
  else a.cuts[blockIdx.x].goes_on = c;
}
__device__ __forceinline__ void note_none(const AttendArgs &a) {
  if (threadIdx.x == 0 && a.cuts != nullptr) a.cuts[blockIdx.x].begins.last = a.cuts[blockIdx.x].goes_on.last = 0;
}

// Sums the work of all requests (a thread takes a run of them) and finds where this block's share begins; all threads return the
// same.  Where units are few and none is much longer than a share would be, every unit is a share, and nothing has to be
// joined; otherwise the shares are equal and cut units anywhere.
__device__ __forceinline__ Share find_share(const AttendArgs &a, int tile_keys, Walk &w) {
  __shared__ int64_t warp_sums[ATT_THREADS / 32], found_left;
  __shared__ int warp_longest[ATT_THREADS / 32], found_request, found_unit;
  __shared__ Span found_span;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, units = (int)a.cache.heads * a.head_blocks, me = blockIdx.x;
  const int64_t all_units = (int64_t)a.requests * units;
  Share s = {};
  w.tile = 0;
  w.request = me / units;  // if units are shares
  w.unit = me - w.request * units;
  w.left = UNIT_COST + MOST_TOKENS;
  if (w.request < a.requests) w.span = span_of(a, w.request);
  bool whole = a.cuts == nullptr;
  if (!whole) {
    const int run = (a.requests + ATT_THREADS - 1) / ATT_THREADS, first = threadIdx.x * run;
    int64_t sum = 0;
    int longest = 0;
    Span last;
    for (int b = first; b < min(first + run, a.requests); ++b) {
      last = span_of(a, b);
      const int n = UNIT_COST + tiles_of(last, tile_keys);
      sum += (int64_t)n * units;
      longest = max(longest, n);
    }
    int64_t upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t below = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += below;
      longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, d));
    }
    if (lane == 31) {
      warp_sums[warp] = upto;
      warp_longest[warp] = longest;
    }
    __syncthreads();
    for (int v = 0; v < ATT_THREADS / 32; ++v) {
      if (v < warp) upto += warp_sums[v];
      s.all += warp_sums[v];
      longest = max(longest, warp_longest[v]);
    }
    s.shares = (int)max((int64_t)1, min((int64_t)a.blocks, s.all / MIN_WORK));
    whole = all_units <= a.blocks && (longest - UNIT_COST - WHOLE_TILES) * (int64_t)s.shares <= s.all;
    const int64_t from = share_start(min(me, s.shares - 1), s.all, s.shares);
    s.to = share_start(min(me, s.shares - 1) + 1, s.all, s.shares);
    if (!whole && from >= upto - sum && from < upto) {
      int64_t into = from - (upto - sum);
      int b = first;
      while (run > 1) {
        last = span_of(a, b);
        const int64_t n = (int64_t)(UNIT_COST + tiles_of(last, tile_keys)) * units;
        if (into < n) break;
        into -= n;
        ++b;
      }
      const int n = UNIT_COST + tiles_of(last, tile_keys);
      found_request = b;
      found_unit = (int)(into / n);
      found_left = into % n;
      found_span = last;
    }
    __syncthreads();
    if (!whole) {
      w.request = found_request;
      w.unit = found_unit;
      w.tile = (int)max((int64_t)0, found_left - UNIT_COST);
      w.left = s.to - from + found_left;
      w.span = found_span;
    }
  }
  w.done = whole ? me >= all_units : me >= s.shares;
  if (w.done) return s;
  if (whole) w.left = UNIT_COST + tiles_of(w.span, tile_keys);
  w.enter(tile_keys);
  return s;
}

// ---- any type, width, stride and alignment --------------------------------------

constexpr int ANY_HEADS = 8, ANY_TILE = 32;

__host__ __device__ constexpr int any_smem(int dim) { return (ANY_HEADS * dim + 2 * ANY_TILE * (dim + 1) + ANY_HEADS * ANY_TILE + 2 * ANY_HEADS) * 4; }

// Right for everything, and for heads of odd widths the only one: 32 requests of up to 8192 tokens, 8 key heads of 30 bf16 values,
// 64 query heads take 1146 us (114 GB/s), heads of 64 by attend_mma_kernel 53.  Bound by its loads of single values and by
// shared memory.  A block walks its tiles of 32 keys: keys and values to shared memory in 32 bits, a thread a key and two heads for the
// scores, a thread a dimension or two for the sums.
template <typename T>
__global__ void __launch_bounds__(ATT_THREADS) attend_any_kernel(const __grid_constant__ AttendArgs a) {
  extern __shared__ float smem[];
  const int dim = a.dim, pitch = dim + 1;
  float *const qs = smem, *const ks = qs + ANY_HEADS * dim, *const vs = ks + ANY_TILE * pitch, *const ps = vs + ANY_TILE * pitch;
  float *const factor = ps + ANY_HEADS * ANY_TILE, *const total = factor + ANY_HEADS;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  pdl_wait();
  Walk w;
  const Share share = find_share(a, ANY_TILE, w);
  pdl_release();
  note_none(a);
  const int units = (int)a.cache.heads * a.head_blocks;
  for (bool first_piece = true; !w.done; first_piece = false) {
    const int kv_head = w.unit / a.head_blocks, head0 = (w.unit % a.head_blocks) * ANY_HEADS, heads = min(ANY_HEADS, a.group - head0);
    const int request = w.request;
    const Span span = w.span;
    __syncthreads();
    for (int i = threadIdx.x; i < heads * dim; i += ATT_THREADS)
      qs[i] = to_f32(static_cast<const T *>(a.q)[request * a.q_token_stride + (int64_t)(kv_head * a.group + head0 + i / dim) * a.q_head_stride + i % dim]);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, acc[2][ANY_HEADS] = {};
    for (int t = w.tile; t < w.end; ++t) {
      const int key0 = span.origin + t * ANY_TILE;
      __syncthreads();
      for (int j = warp; j < ANY_TILE; j += ATT_THREADS / 32) {
        const bool in = key0 + j >= span.lo && key0 + j < span.hi;
        const int64_t row0 = in ? cache_row(a.cache, a.lists, request, key0 + j, a.page_shift) : -1, row = row0 + kv_head * a.cache.page_size;
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
        score = key0 + lane >= span.lo && key0 + lane < span.hi ? score * a.scale2 : -INFINITY;
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
    const bool whole = w.tile == 0 && w.end == w.tiles;
    float *const slot = a.partial + ((int64_t)blockIdx.x * 2 + (first_piece ? 0 : 1)) * ANY_HEADS * (dim + 2);
    note_cut(a, share, w, w.tile);
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
        a.lse[(int64_t)request * a.q_heads + kv_head * a.group + head0 + h] = sum == 0.0f ? -INFINITY : m[u] * LN2 + logf(sum);
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
          static_cast<T *>(a.out)[((int64_t)request * a.q_heads + kv_head * a.group + head0 + h) * dim + i] = from_f32<T>(total[h] == 0.0f ? 0.0f : acc[e][h] / total[h]);
        else
          slot[h * (dim + 2) + 2 + i] = acc[e][h];
      }
    }
    w.next_unit(a, units, ANY_TILE);
  }
}

// Adds up what the blocks left of the units that were cut, in their order: block (share where the unit begins, head), a thread a
// dimension or two.
template <typename T>
__global__ void __launch_bounds__(ATT_THREADS) join_any_kernel(const __grid_constant__ AttendArgs a, int heads_of_unit) {
  pdl_wait();
  const CutUnit cut = a.cuts[blockIdx.x].begins;
  const int first = blockIdx.x, h = blockIdx.y, dim = a.dim;
  const int head0 = (cut.unit % a.head_blocks) * heads_of_unit;
  if (cut.last == 0 || head0 + h >= a.group) return;
  auto slot = [&](int i) { return a.partial + ((int64_t)(i * 2 + (i > first ? 0 : cut.slot)) * ANY_HEADS + h) * (dim + 2); };
  float most = -INFINITY, sum = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int i = first; i <= cut.last; ++i) most = fmaxf(most, slot(i)[0]);
  const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll 4
  for (int i = first; i <= cut.last; ++i) {
    const float *p = slot(i);
    const float f = exp2f(p[0] - base);
    sum = fmaf(p[1], f, sum);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = threadIdx.x + e * ATT_THREADS;
      if (d < dim) acc[e] = fmaf(p[2 + d], f, acc[e]);
    }
  }
  const int64_t head = (int64_t)cut.request * a.q_heads + cut.unit / a.head_blocks * a.group + head0 + h;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int d = threadIdx.x + e * ATT_THREADS;
    if (d < dim) static_cast<T *>(a.out)[head * dim + d] = from_f32<T>(sum == 0.0f ? 0.0f : acc[e] / sum);
  }
  if (threadIdx.x == 0 && a.lse != nullptr) a.lse[head] = sum == 0.0f ? -INFINITY : most * LN2 + logf(sum);
}

// Whether the lists cannot hold more than what find_share leaves whole: then nothing is cut, and there is nothing to join (a short
// request of one user: 1 x 129 tokens take 10.3 us without, 14.4 with the join's launch).
static bool always_whole(const AttendArgs &a, int tile) {
  const int64_t most_tokens = a.lists.entries > MOST_TOKENS / a.cache.page_size ? MOST_TOKENS : a.lists.entries * a.cache.page_size;
  return (int64_t)a.requests * a.cache.heads * a.head_blocks <= a.blocks && most_tokens <= WHOLE_TILES * tile - 16;
}

// The workspace of a call: `floats` for the pieces of each block, and the cuts behind them.
static int make_workspace(AttendArgs &a, PoolBuf &work, size_t floats, cudaStream_t st) {
  const size_t pieces = ((size_t)a.blocks * floats * sizeof(float) + 15) / 16 * 16;
  LAPIS_TRY(work.alloc(pieces + a.blocks * sizeof(Cut), st));
  a.partial = static_cast<float *>(work.p);
  a.cuts = reinterpret_cast<Cut *>(static_cast<char *>(work.p) + pieces);
  return LAPIS_OK;
}

template <typename T>
static int launch_any(AttendArgs a, int dev, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};  // devices on which this kernel may use its shared memory
  if ((allowed.load(std::memory_order_relaxed) >> dev & 1) == 0) {
    LAPIS_CUDA_TRY(cudaFuncSetAttribute(attend_any_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, any_smem(KV_MAX_DIM)));
    allowed.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  a.head_blocks = (a.group + ANY_HEADS - 1) / ANY_HEADS;
  a.blocks = std::min(2 * sm_count(), MOST_BLOCKS);
  PoolBuf work;
  const bool whole = always_whole(a, ANY_TILE);
  if (!whole) LAPIS_TRY(make_workspace(a, work, 2 * ANY_HEADS * (a.dim + 2), st));
  LAPIS_CUDA_TRY(launch_pdl(attend_any_kernel<T>, dim3(a.blocks), ATT_THREADS, any_smem(a.dim), st, a));
  if (whole) return LAPIS_OK;
  LAPIS_CUDA_TRY(launch_pdl(join_any_kernel<T>, dim3(a.blocks, ANY_HEADS), ATT_THREADS, 0, st, a, ANY_HEADS));
  return LAPIS_OK;
}

// ---- a warp's pipeline --------------------------------------------------------------
//
// Keys and values come by cp.async into a ring that one warp uses for itself, STAGES deep: KEYS keys of a tile at a time, the
// part of it that is this warp's.  C: the configuration of a kernel.

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool real) {  // zeros where it is not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0));
}
__device__ __forceinline__ void copy8(uint32_t to, const void *from, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(real ? 8 : 0));
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(real ? 4 : 0));
}
__device__ __forceinline__ uint4 load16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ uint2 load8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at));
  return r;
}
__device__ __forceinline__ float load4(uint32_t at) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(at));
  return r;
}
// 2^x to 2 units in the last place; what is below 2^-126 is zero.
__device__ __forceinline__ float power2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename C>
struct Feed {
  static constexpr int KEYS = C::KEYS, GROUP = C::GROUP, GROUPS = KEYS / GROUP, ROWS = 32 / C::CHUNKS > 0 ? 32 / C::CHUNKS : 1;
  static constexpr int PASSES = C::CHUNKS > 32 ? C::CHUNKS / 32 : 1;  // copies of a row
  Walk in;
  uint32_t ring;
  // Pages of the next steps to copy.  `grouped`: pages have a multiple of GROUP slots; lane n then has the page of the n-th GROUP
  // keys of this warp from tile `looked` on, 32 / GROUPS steps of a unit by one look.  Otherwise lane n has that of key n of the
  // next step.
  int64_t page;
  int slot_in_page, looked;
  uint32_t page_rows, head_row;
  bool grouped;

  __device__ __forceinline__ int of_lane() const { return threadIdx.x % KEYS; }  // the key of a step that is this lane's
  __device__ __forceinline__ int first_key() const { return in.span.origin + in.tile * C::TILE + threadIdx.x / 32 * KEYS; }
  __device__ __forceinline__ void look_up(const AttendArgs &a) {
    const int lane = threadIdx.x % 32, page_size = (int)a.cache.page_size;
    looked = in.tile;
    head_row = (uint32_t)(in.unit / a.head_blocks * page_size);
    const int key = first_key() + (grouped ? lane / GROUPS * C::TILE + lane % GROUPS * GROUP : of_lane());
    page = -1;
    if (key < in.span.hi) {
      const int nth = a.page_shift >= 0 ? key >> a.page_shift : (int)((uint32_t)key / (uint32_t)page_size);
      slot_in_page = key - nth * page_size;
      const int64_t entry = in.span.entry + nth;
      if (entry >= 0 && entry < a.lists.entries) page = load_index(a.lists.d_crd, entry, a.lists.idx_bytes);
    }
  }
  __device__ __forceinline__ void begin(const AttendArgs &a, uint32_t ring_) {
    ring = ring_;
    grouped = a.cache.page_size % GROUP == 0;
    page_rows = (uint32_t)(a.cache.heads * a.cache.page_size);
    slot_in_page = 0;
    look_up(a);
  }
  // Where piece ch of 16 bytes of row r goes: the rows are swizzled so that neither the reads of K nor those of V meet in a bank.
  static __device__ __forceinline__ int k_at(int r, int ch) { return r * C::ROW + (ch ^ C::k_swizzle(r)) * 16; }
  static __device__ __forceinline__ int v_at(int r, int ch) { return KEYS * C::ROW + r * C::ROW + (ch ^ C::v_swizzle(r)) * 16; }
  static constexpr int SCALES = 2 * KEYS * C::ROW;

  // Sends the next step to a stage of the ring.  A key that is not attended is zeros there, whatever its slot holds.
  __device__ __forceinline__ void fetch(const AttendArgs &a, int stage, int units) {
    const int lane = threadIdx.x % 32, ch0 = lane % C::CHUNKS, low = C::CHUNKS > 32 ? 0 : lane / C::CHUNKS, row_bytes = a.dim * C::ELEMENT;
    const uint32_t to = ring + stage * C::STAGE;
    const int key = first_key() + of_lane();
    const bool listed = page >= 0 && page < a.cache.pages;
    const uint32_t looked_row = (uint32_t)page * page_rows + head_row + (uint32_t)slot_in_page;
    const int at = grouped ? (in.tile - looked) * GROUPS + of_lane() / GROUP : of_lane();  // the lane that looked this one's key up
    const bool found = __shfl_sync(0xffffffffu, listed, at);
    uint32_t row = __shfl_sync(0xffffffffu, looked_row, at) + (grouped ? of_lane() % GROUP : 0);  // of this lane's key
    const bool there = found && key >= in.span.lo && key < in.span.hi;
    if (!there) row = 0;
    if (grouped && row_bytes % 16 == 0 && __all_sync(0xffffffffu, there)) {
#pragma unroll
      for (int n = 0; n < GROUPS; ++n) {
        const int64_t offset = (int64_t)__shfl_sync(0xffffffffu, row, n * GROUP) * row_bytes + low * row_bytes;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          const int ch = ch0 + p * 32;
          const char *const kp = static_cast<const char *>(a.cache.d_k) + ch * 16 + offset, *const vp = static_cast<const char *>(a.cache.d_v) + ch * 16 + offset;
          if (ch * 16 < row_bytes) {
#pragma unroll
            for (int i = 0; i < GROUP / ROWS; ++i) {
              const int r = n * GROUP + i * ROWS + low;
              copy16(to + k_at(r, ch), kp + i * ROWS * row_bytes, true);
              copy16(to + v_at(r, ch), vp + i * ROWS * row_bytes, true);
            }
          }
        }
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < KEYS / ROWS; ++i) {
        const int r = i * ROWS + low;
        const int64_t offset = (int64_t)__shfl_sync(0xffffffffu, row, r) * row_bytes;
        const bool real = __shfl_sync(0xffffffffu, there, r);
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          const int ch = ch0 + p * 32;
          const char *const kp = static_cast<const char *>(a.cache.d_k) + ch * 16 + offset, *const vp = static_cast<const char *>(a.cache.d_v) + ch * 16 + offset;
          if (ch * 16 >= row_bytes) continue;
          if (row_bytes % 16 == 0) {
            copy16(to + k_at(r, ch), kp, real);
            copy16(to + v_at(r, ch), vp, real);
          } else {  // rows begin at multiples of 8 bytes
            copy8(to + k_at(r, ch), kp, real);
            copy8(to + v_at(r, ch), vp, real);
            if (ch * 16 + 8 < row_bytes) {
              copy8(to + k_at(r, ch) + 8, kp + 8, real);
              copy8(to + v_at(r, ch) + 8, vp + 8, real);
            }
          }
        }
      }
    }
    if (C::CODES && lane < KEYS) {
      copy4(to + SCALES + lane * 4, a.cache.d_k_scale + row, there);
      copy4(to + SCALES + KEYS * 4 + lane * 4, a.cache.d_v_scale + row, there);
    }
    const int unit = in.unit, request = in.request;
    in.next_tile(a, units, C::TILE);
    if (!in.done && (!grouped || in.unit != unit || in.request != request || in.tile - looked == 32 / GROUPS)) look_up(a);
  }
};

// ---- 32-bit queries and caches ----------------------------------------------------
//
// Products and sums in 32 bits on the CUDA cores: bound by the cache for a query head or two a key head, and with eight by
// shared memory and the products, about even with it.  A warp's KEYS keys of a step: four lanes share a key, a quarter of its
// pieces each, and add up their parts of HEADS scores so that lane c of the four ends with heads c * HEADS / 4 onward; the
// weights go through shared memory, and then a lane owns four dimensions (of every SPLIT-th key, where heads are narrow).
// 16 requests of up to 2047 tokens, 8 heads of 72: 17 us alone (5.2 TB/s; a block's first data comes after 5 us) and 25 in all,
// 182 by attend_any_kernel.  32 of up to 8192, 8 key heads of 128: 6.3 TB/s with 2 query heads each, 5.2 with 8.

template <int DP_, int HEADS_>
struct F32Config {
  static constexpr int DP = DP_, HEADS = HEADS_;            // padded head; query heads of a unit
  static constexpr bool CODES = false;
  static constexpr int ELEMENT = 4, ROW = DP * 4, CHUNKS = DP / 4;
  static constexpr int KEYS = DP == 64 ? 16 : 8, GROUP = 8, TILE = KEYS * (ATT_THREADS / 32);
  static constexpr int STAGE = 2 * KEYS * ROW;
  static constexpr int OWN = HEADS >= 4 ? HEADS / 4 : 1;    // heads of a lane while there are scores
  static constexpr int SPLIT = DP == 64 ? 2 : 1, OWNED = DP == 256 ? 2 : 1;  // keys side by side; fours of dimensions of a lane
  static constexpr int PART = HEADS * DP + 2 * HEADS;       // floats of a warp's sums: O, then m and l
  static constexpr int WEIGHTS = KEYS * HEADS + HEADS;      // floats of a warp's weights, and of the factors for older sums
  static constexpr int EXTRA = (HEADS * DP + ATT_THREADS / 32 * WEIGHTS) * 4;
  // As many as shared memory holds with two stages each: three, of heads of 256 one (with three).
  static constexpr int BLOCKS = DP == 256 ? 1 : 3;
  static constexpr int STAGES = (227 * 1024 / BLOCKS - 2048 - EXTRA) / (ATT_THREADS / 32 * STAGE);
  static constexpr int SMEM = ATT_THREADS / 32 * STAGES * STAGE + EXTRA;
  static_assert(STAGES >= 2, "one is copied while another is read");
  static_assert(PART * 4 <= STAGE, "a warp's sums fit where its last keys were");
  static __device__ __forceinline__ int k_swizzle(int r) { return (r & 1) << 2; }
  static __device__ __forceinline__ int v_swizzle(int) { return 0; }
};

__device__ __forceinline__ float4 load_float4(uint32_t at) {
  const uint4 x = load16(at);
  return make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w));
}

template <typename C>
__global__ void __launch_bounds__(ATT_THREADS, C::BLOCKS) attend_f32_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int WARPS = ATT_THREADS / 32, KEYS = C::KEYS, HEADS = C::HEADS, OWN = C::OWN, STAGES = C::STAGES, ROUNDS = KEYS / 8;
  extern __shared__ __align__(128) unsigned char stages[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c = lane % 4;
  unsigned char *const mine = stages + warp * STAGES * C::STAGE;
  float *const qs = reinterpret_cast<float *>(stages + WARPS * STAGES * C::STAGE), *const weights = qs + HEADS * C::DP + warp * C::WEIGHTS;
  float *const factors = weights + KEYS * HEADS;
  const int units = (int)a.cache.heads * a.head_blocks;
  pdl_wait();
  Feed<C> feed;
  const Share share = find_share(a, C::TILE, feed.in);
  pdl_release();
  note_none(a);
  if (feed.in.done) return;
  Walk out = feed.in;
  for (int i = lane; i < STAGES * C::STAGE / 16; i += 32) reinterpret_cast<uint4 *>(mine)[i] = make_uint4(0, 0, 0, 0);  // beyond the head
  __syncwarp();
  feed.begin(a, shared_address(mine));

  // The queries of a unit are fetched while the one in front is given out.
  constexpr int MINE = HEADS * C::DP / ATT_THREADS > 0 ? HEADS * C::DP / ATT_THREADS : 1;
  float raw[MINE];
  auto load_q = [&]() {
    const int head0 = (out.unit % a.head_blocks) * HEADS;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int at = i * ATT_THREADS + threadIdx.x, h = at / C::DP, d = at % C::DP;
      raw[i] = at < HEADS * C::DP && d < a.dim && head0 + h < a.group
                   ? static_cast<const float *>(a.q)[out.request * a.q_token_stride + (int64_t)(out.unit / a.head_blocks * a.group + head0 + h) * a.q_head_stride + d]
                   : 0.0f;
    }
  };
  auto take_q = [&]() {
#pragma unroll
    for (int i = 0; i < MINE; ++i)
      if (i * ATT_THREADS + threadIdx.x < HEADS * C::DP) qs[i * ATT_THREADS + threadIdx.x] = raw[i];
    __syncthreads();
  };
  float4 acc[HEADS][C::OWNED];
  float m[OWN], l[OWN];
  auto clear = [&]() {
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
#pragma unroll
      for (int o = 0; o < C::OWNED; ++o) acc[h][o] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
  };
  load_q();
  int began = out.tile, stage = 0, stage_in = 0;
  bool first_piece = true;
  const int rounds = (a.dim + 15) / 16;  // pieces of a key that a lane multiplies
#pragma unroll 1
  for (int ahead = 1 - STAGES;; ahead = min(ahead + 1, 0)) {  // below 0: there are not enough copies on their way
    if (ahead == 0) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();
    if (!feed.in.done) feed.fetch(a, stage_in, units);
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
    if (ahead < 0) {
      if (ahead == -1) {
        take_q();
        clear();
      }
      continue;
    }

    const uint32_t ks = feed.ring + stage * C::STAGE, vs = ks + KEYS * C::ROW, q_at = shared_address(qs);
    const int key0 = out.span.origin + out.tile * C::TILE + warp * KEYS;
    float score[ROUNDS][OWN];
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
      const int r = u * 8 + g;
      float2 part[HEADS];
#pragma unroll
      for (int h = 0; h < HEADS; ++h) part[h] = make_float2(0.0f, 0.0f);
#pragma unroll 2
      for (int i = 0; i < rounds; ++i) {
        const float4 k = load_float4(ks + r * C::ROW + (((c + 4 * i) ^ C::k_swizzle(r)) * 16));
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
          const float4 x = load_float4(q_at + (h * C::DP + (c + 4 * i) * 4) * 4);
          part[h] = fma2({k.x, k.y}, {x.x, x.y}, part[h]);
          part[h] = fma2({k.z, k.w}, {x.z, x.w}, part[h]);
        }
      }
      float sum[HEADS];
#pragma unroll
      for (int h = 0; h < HEADS; ++h) sum[h] = part[h].x + part[h].y;
      if constexpr (HEADS == 1) {
        sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 1);
        sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 2);
        score[u][0] = sum[0];
      } else {
        float half[HEADS / 2];
#pragma unroll
        for (int h = 0; h < HEADS / 2; ++h) {
          const float keep = c & 2 ? sum[HEADS / 2 + h] : sum[h], send = c & 2 ? sum[h] : sum[HEADS / 2 + h];
          half[h] = keep + __shfl_xor_sync(0xffffffffu, send, 2);
        }
#pragma unroll
        for (int h = 0; h < OWN; ++h) {
          const float keep = c & 1 ? half[OWN + h] : half[h], send = c & 1 ? half[h] : half[OWN + h];
          score[u][h] = keep + __shfl_xor_sync(0xffffffffu, send, 1);
        }
      }
      const bool seen = key0 + r >= out.span.lo && key0 + r < out.span.hi;
#pragma unroll
      for (int i = 0; i < OWN; ++i) score[u][i] = seen ? score[u][i] * a.scale2 : -INFINITY;
    }
    bool grows = false;
    float base[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      float x = m[i];
#pragma unroll
      for (int u = 0; u < ROUNDS; ++u) x = fmaxf(x, score[u][i]);
#pragma unroll
      for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
      base[i] = x == -INFINITY ? 0.0f : x;
      grows |= x > m[i];
      const float f = exp2f(m[i] - base[i]);
      l[i] *= f;
      m[i] = x;
      if (g == 0) factors[(HEADS == 1 ? 0 : c * OWN) + i] = f;
#pragma unroll
      for (int u = 0; u < ROUNDS; ++u) {
        const float p = exp2f(score[u][i] - base[i]);
        l[i] += p;
        weights[(u * 8 + g) * HEADS + (HEADS == 1 ? 0 : c * OWN) + i] = p;
      }
    }
    grows = __any_sync(0xffffffffu, grows);
    __syncwarp();
    if (grows) {
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        const float f = factors[h];
#pragma unroll
        for (int o = 0; o < C::OWNED; ++o) {
          acc[h][o].x *= f;
          acc[h][o].y *= f;
          acc[h][o].z *= f;
          acc[h][o].w *= f;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < KEYS; j += C::SPLIT) {
      const int r = j + (C::SPLIT == 2 ? lane / 16 : 0), ch = C::SPLIT == 2 ? lane % 16 : lane;
      float p[HEADS];
      if constexpr (HEADS >= 4) {
#pragma unroll
        for (int h = 0; h < HEADS; h += 4) {
          const float4 x = *reinterpret_cast<const float4 *>(weights + r * HEADS + h);
          p[h] = x.x;
          p[h + 1] = x.y;
          p[h + 2] = x.z;
          p[h + 3] = x.w;
        }
      } else {
        p[0] = weights[r];
      }
#pragma unroll
      for (int o = 0; o < C::OWNED; ++o) {
        const float4 v = load_float4(vs + r * C::ROW + (ch + 32 * o) * 16);
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
          const float2 lo = fma2({v.x, v.y}, {p[h], p[h]}, {acc[h][o].x, acc[h][o].y}), hi = fma2({v.z, v.w}, {p[h], p[h]}, {acc[h][o].z, acc[h][o].w});
          acc[h][o] = make_float4(lo.x, lo.y, hi.x, hi.y);
        }
      }
    }
    __syncwarp();  // the weights have been read

    const int used = stage;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if (out.tile + 1 < out.end) {
      ++out.tile;
      continue;
    }
    const int request = out.request, head0 = (out.unit % a.head_blocks) * HEADS, heads = min(HEADS, a.group - head0);
    const int64_t first_head = (int64_t)request * a.q_heads + out.unit / a.head_blocks * a.group + head0;
    const bool whole = began == 0 && out.end == out.tiles;
    note_cut(a, share, out, began);
    out.next_unit(a, units, C::TILE);
    if (!out.done) load_q();
    // the warps' sums meet where their last keys were
    float *const sums = reinterpret_cast<float *>(mine + used * C::STAGE);
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
      if (g == 0) {
        const int h = (HEADS == 1 ? 0 : c * OWN) + i;
        sums[HEADS * C::DP + 2 * h] = m[i];
        sums[HEADS * C::DP + 2 * h + 1] = l[i];
      }
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
#pragma unroll
      for (int o = 0; o < C::OWNED; ++o) {
        float4 x = acc[h][o];
        if constexpr (C::SPLIT == 2) {
          x.x += __shfl_xor_sync(0xffffffffu, x.x, 16);
          x.y += __shfl_xor_sync(0xffffffffu, x.y, 16);
          x.z += __shfl_xor_sync(0xffffffffu, x.z, 16);
          x.w += __shfl_xor_sync(0xffffffffu, x.w, 16);
        }
        if (C::SPLIT == 1 || lane < 16) *reinterpret_cast<float4 *>(sums + h * C::DP + (lane % C::CHUNKS + 32 * o) * 4) = x;
      }
    __syncthreads();
    auto of_warp = [&](int w) { return reinterpret_cast<const float *>(stages + (w * STAGES + used) * C::STAGE); };
    float *const slot = a.partial + ((int64_t)blockIdx.x * 2 + (first_piece ? 0 : 1)) * ANY_HEADS * (a.dim + 2);
    for (int at = threadIdx.x; at < heads * C::DP; at += ATT_THREADS) {
      const int h = at / C::DP, d = at % C::DP;
      float most = -INFINITY, total = 0.0f, x = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) most = fmaxf(most, of_warp(w)[HEADS * C::DP + 2 * h]);
      const float shift = most == -INFINITY ? 0.0f : most;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = exp2f(of_warp(w)[HEADS * C::DP + 2 * h] - shift);
        total = fmaf(of_warp(w)[HEADS * C::DP + 2 * h + 1], f, total);
        x = fmaf(of_warp(w)[at], f, x);
      }
      if (d >= a.dim) continue;
      if (whole) {
        static_cast<float *>(a.out)[(first_head + h) * a.dim + d] = total == 0.0f ? 0.0f : x / total;
        if (d == 0 && a.lse != nullptr) a.lse[first_head + h] = total == 0.0f ? -INFINITY : most * LN2 + logf(total);
      } else {
        slot[h * (a.dim + 2) + 2 + d] = x;
        if (d == 0) {
          slot[h * (a.dim + 2)] = most;
          slot[h * (a.dim + 2) + 1] = total;
        }
      }
    }
    __syncthreads();
    if (out.done) return;
    if (a.dim != C::DP) {
      for (int i = lane; i < C::STAGE / 16; i += 32) reinterpret_cast<uint4 *>(sums)[i] = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    first_piece = false;
    began = 0;
    take_q();
    clear();
  }
}

template <typename C>
static int launch_f32(AttendArgs a, int dev, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};  // devices on which this kernel may use its shared memory
  if ((allowed.load(std::memory_order_relaxed) >> dev & 1) == 0) {
    LAPIS_CUDA_TRY(cudaFuncSetAttribute(attend_f32_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    allowed.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  a.head_blocks = (a.group + C::HEADS - 1) / C::HEADS;
  a.blocks = std::min(C::BLOCKS * sm_count(), MOST_BLOCKS);
  PoolBuf work;
  const bool whole = always_whole(a, C::TILE);
  if (!whole) LAPIS_TRY(make_workspace(a, work, 2 * ANY_HEADS * (a.dim + 2), st));
  LAPIS_CUDA_TRY(launch_pdl(attend_f32_kernel<C>, dim3(whole ? a.requests * (int)a.cache.heads * a.head_blocks : a.blocks), ATT_THREADS, C::SMEM, st, a));
  if (whole) return LAPIS_OK;
  LAPIS_CUDA_TRY(launch_pdl(join_any_kernel<float>, dim3(a.blocks, C::HEADS), ATT_THREADS, 0, st, a, C::HEADS));
  return LAPIS_OK;
}

template <int HEADS>
static int launch_f32_of(const AttendArgs &a, int dev, cudaStream_t st) {
  if (a.dim <= 64) return launch_f32<F32Config<64, HEADS>>(a, dev, st);
  if (a.dim <= 128) return launch_f32<F32Config<128, HEADS>>(a, dev, st);
  return launch_f32<F32Config<256, HEADS>>(a, dev, st);
}

// ---- 16-bit queries: products on the tensor cores ----------------------------------
//
// Bound by the cache coming from memory, so the products only have to keep out of its way: mma.sync of 16 keys by 8 heads by
// 16 values, whose smallest shape fits the few query heads of a key head (tcgen05 has 64 or 128 rows, of which one to sixteen
// would be heads or, turned round, needs the weights to go through shared memory once more).  S^T = K Q^T has the keys in rows
// and the heads in columns, O^T = V^T P^T the values in rows: keys and values are the A operands, which shared memory gives
// by ldmatrix without a copy, and P^T is S^T's accumulator after a movmatrix.
// A warp is a pipeline of its own: it copies the KEYS keys that are its part of a tile by cp.async, STAGES deep, keeps its own
// m, l and O, and meets the other three only where a unit ends.
// Weights go into the product with the values as a 16-bit number, and where that would show in the result (all but bf16
// results from a quantised cache, whose own 8 bits are 2^-8 and the weights' 11 here) as two, high and low part, whose sum has
// at least 16 bits.  Quantised caches: codes are exact in fp16, so are queries after a power of two is taken out of each; a
// key's scale is multiplied to its score in 32 bits, a value's scale to its weight, and the product is taken relative to the largest
// one that the head has seen, carried along as the softmax's maximum is: a large scale counts for no more than its token's weight.
// What fp16 leaves of weight * scale is off by at most 2^-38 of that largest one beside the rounding to its bits.
// Measured, kernel alone: 1 x 131,072 tokens, 8 key heads of 128 in bf16, 32 query heads: 82 to 87 us, 6.2 to 6.5 TB/s, the rate of a copy; 128
// requests of up to 8192, 64 query heads, int8: 197 us, 6.0 TB/s of DRAM, 881 instructions a step at 2.5 a cycle; called again and
// again it falls to 215 to 235 us, as the power cap takes the clock.  Scores of int8 by whole-number products of three digits of the
// queries (no conversion of the keys, 14 % fewer instructions) took 229 us where this took 231, and 62 where this took 59 on 32
// requests.  Four warps of 168 registers, three blocks an SM: two blocks of 250 registers took 274 us of the second where three took
// 244.

constexpr int MMA_WARPS = ATT_THREADS / 32;

template <typename T_, int STORE_, int DP_, int NT_>
struct MmaConfig {
  using T = T_;                                             // type of q and of the result
  static constexpr int STORE = STORE_;                      // LAPIS_I8, LAPIS_E4M3, or anything else: T
  static constexpr bool CODES = STORE == LAPIS_I8 || STORE == LAPIS_E4M3;
  static constexpr bool HALF = CODES || std::is_same<T, __half>::value;  // fp16 products, or bf16
  static constexpr bool TWO_PARTS = !(CODES && std::is_same<T, __nv_bfloat16>::value);  // of the weights
  static constexpr int QP = std::is_same<T, float>::value ? 2 : 1;                      // parts of the queries
  static constexpr int DP = DP_, NT = NT_;                  // padded head, and eights of query heads
  static constexpr int ELEMENT = CODES ? 1 : 2, ROW = DP * ELEMENT;  // bytes of a key in shared memory
  static constexpr int KEYS = ROW <= 128 ? 32 : 16, TILE = KEYS * MMA_WARPS, MT = KEYS / 16;
  // Keys that are looked up together.  32 requests of up to 8192 tokens in int8: with 8, pages of 24 or 8 slots take 60 us (72 to 75
  // with 16), those of 16 or 64 also 60 (59); with 16 query heads, or 16-bit caches, where copies count for less, 16.
  static constexpr int GROUP = CODES && NT == 1 ? 8 : 16;
  static constexpr int CHUNKS = ROW / 16;
  static constexpr int STAGE = 2 * KEYS * ROW + (CODES ? 2 * KEYS * 4 : 0);
  static constexpr int DT = DP / 16, PART = DT * 128 + 16;  // floats of eight heads' sums: O, then m and l
  // Wide heads of codes: one block an SM takes 168 us of 32 requests of up to 8192, two 119.
  static constexpr int BLOCKS = DP == 256 ? (CODES ? 2 : 1) : DP * NT * QP >= 256 ? 2 : 3;  // an SM, by registers and shared memory
  static constexpr int STAGES = (227 * 1024 / BLOCKS - 2048) / (MMA_WARPS * STAGE);
  static constexpr int SMEM = MMA_WARPS * STAGES * STAGE;
  static_assert(STAGES >= 2, "one is copied while another is read");
  static_assert(PART * 4 <= STAGE, "a warp's sums fit where its last keys were");
  // Weights in fp16 are times 2^14, so that they are subnormal only below 2^-28; the sums are without it.
  static constexpr float OFFSET = HALF ? 0x1p14f : 1.0f;
  static constexpr uint32_t LEAST_UNIT = 0x07800000;  // 2^-112: OFFSET / it is a number
  static __device__ __forceinline__ int k_swizzle(int r) { return !CODES ? r & 7 : DP == 64 ? 0 : r & 4; }
  static __device__ __forceinline__ int v_swizzle(int r) { return !CODES ? r & 7 : DP == 64 ? r & 2 : (r & 3) << 1; }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d += a (low + high), for results in 32 bits: the tensor cores cut what lies below the last place of the largest term, and over
// long sums that adds up to 1 to 4e-6 of a result; two products at a time, added by rounding, are as near as a sum in 32 bits.
__device__ __forceinline__ void mma_apart(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&low)[2], const uint32_t (&high)[2]) {
  float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  mma<true>(part, a, low[0], low[1]);
  mma<true>(part, a, high[0], high[1]);
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] += part[i];
}
// Two numbers of 32 bits as two of 16, the first in the low half; `back`: the 16-bit numbers in 32 bits.
template <bool HALF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <bool HALF>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if (HALF) return __half22float2(*reinterpret_cast<const __half2 *>(&x));
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
// Two codes, in the low or the high half of x, as two fp16 numbers.  int8: 0x6400 + (code + 128) is 1024 + 128 + code.
template <int STORE, bool HIGH>
__device__ __forceinline__ uint32_t codes2(uint32_t x) {
  if (STORE == LAPIS_I8) {
    const uint32_t biased = __byte_perm(x, 0x64646464u, HIGH ? 0x4342 : 0x4140);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&r);
  }
  uint32_t r;
  const uint16_t two = (uint16_t)(HIGH ? x >> 16 : x);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
  return r;
}

// What a warp has summed of eight heads: lane (g, c), g = lane / 4, c = lane % 4, holds dimensions by g of heads 2c and 2c + 1.
template <int DT>
struct Sums {
  float o[DT][4], m[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.0f;
  }
};

// Dimension of o[t][0] of group g; that of o[t][2] is the one 8 further (16-bit caches) or the next (codes).
template <typename C>
__device__ __forceinline__ int dimension(int t, int g) {
  if (!C::CODES) return t * 16 + g;
  return C::DP == 64 ? g * 8 + 2 * t : (g + 8 * (t / 8)) * 16 + 2 * (t % 8);
}

// Adds up the warps of the block and gives eight heads out: as results, or to `part` where the unit was cut.  The warps' sums meet
// where their last keys were (`mine`, and warp w's `apart` bytes times w behind the first one's); each adds up a quarter.
template <typename C>
__device__ __forceinline__ void give(const AttendArgs &a, const Sums<C::DT> &s, unsigned char *mine, int apart, int request, int first_head, int heads, float *part) {
  using T = typename C::T;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  float4 *const to = reinterpret_cast<float4 *>(mine);
  const unsigned char *const all = mine - warp * apart;
#pragma unroll
  for (int t = 0; t < C::DT; ++t) to[t * 32 + lane] = make_float4(s.o[t][0], s.o[t][1], s.o[t][2], s.o[t][3]);
  if (g == 0) to[C::DT * 32 + c] = make_float4(s.m[0], s.m[1], s.l[0], s.l[1]);
  __syncthreads();
  float4 ml[MMA_WARPS];
  float2 f[MMA_WARPS];
#pragma unroll
  for (int w = 0; w < MMA_WARPS; ++w) ml[w] = reinterpret_cast<const float4 *>(all + w * apart)[C::DT * 32 + c];
  float m[2] = {ml[0].x, ml[0].y}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int w = 1; w < MMA_WARPS; ++w) {
    m[0] = fmaxf(m[0], ml[w].x);
    m[1] = fmaxf(m[1], ml[w].y);
  }
#pragma unroll
  for (int w = 0; w < MMA_WARPS; ++w) {
    f[w] = make_float2(power2(ml[w].x - (m[0] == -INFINITY ? 0.0f : m[0])), power2(ml[w].y - (m[1] == -INFINITY ? 0.0f : m[1])));
    l[0] = fmaf(ml[w].z, f[w].x, l[0]);
    l[1] = fmaf(ml[w].w, f[w].y, l[1]);
  }
  if (warp == 0 && g == 0) {
    if (part != nullptr) reinterpret_cast<float4 *>(part)[C::DT * 32 + c] = make_float4(m[0], m[1], l[0], l[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (part == nullptr && a.lse != nullptr && 2 * c + i < heads)
        a.lse[(int64_t)request * a.q_heads + first_head + 2 * c + i] = l[i] == 0.0f ? -INFINITY : m[i] * LN2 + logf(l[i]);
  }
  const float by[2] = {l[0] == 0.0f ? 0.0f : 1.0f / l[0], l[1] == 0.0f ? 0.0f : 1.0f / l[1]};
  T *const out = static_cast<T *>(a.out) + ((int64_t)request * a.q_heads + first_head + 2 * c) * a.dim;
#pragma unroll 1
  for (int t = warp; t < C::DT; t += MMA_WARPS) {
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < MMA_WARPS; ++w) {
      const float4 y = reinterpret_cast<const float4 *>(all + w * apart)[t * 32 + lane];
      x.x = fmaf(y.x, f[w].x, x.x);
      x.y = fmaf(y.y, f[w].y, x.y);
      x.z = fmaf(y.z, f[w].x, x.z);
      x.w = fmaf(y.w, f[w].y, x.w);
    }
    if (part != nullptr) {
      reinterpret_cast<float4 *>(part)[t * 32 + lane] = x;
      continue;
    }
    const int d0 = dimension<C>(t, g), d1 = C::CODES ? d0 + 1 : d0 + 8;
    if (2 * c < heads) {
      if (d0 < a.dim) out[d0] = from_f32<T>(x.x * by[0]);
      if (d1 < a.dim) out[d1] = from_f32<T>(x.z * by[0]);
    }
    if (2 * c + 1 < heads) {
      if (d0 < a.dim) out[a.dim + d0] = from_f32<T>(x.y * by[1]);
      if (d1 < a.dim) out[a.dim + d1] = from_f32<T>(x.w * by[1]);
    }
  }
  __syncthreads();
}

template <typename C>
__global__ void __launch_bounds__(ATT_THREADS, C::BLOCKS) attend_mma_kernel(const __grid_constant__ AttendArgs a) {
  using T = typename C::T;
  constexpr int KEYS = C::KEYS, MT = C::MT, NT = C::NT, DT = C::DT, STAGES = C::STAGES;
  extern __shared__ __align__(128) unsigned char stages[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c = lane % 4;
  unsigned char *const mine = stages + warp * STAGES * C::STAGE;
  const uint32_t ring = shared_address(mine);
  const int units = (int)a.cache.heads * a.head_blocks;
  pdl_wait();
  Feed<C> feed;
  const Share share = find_share(a, C::TILE, feed.in);
  pdl_release();
  note_none(a);
  if (feed.in.done) return;
  Walk out = feed.in;  // of the products; that of the copies is ahead
  auto clear_stage = [&](int stage) {  // what is beyond the head is never copied
    for (int i = lane; i < C::STAGE / 16; i += 32) reinterpret_cast<uint4 *>(mine + stage * C::STAGE)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  };
  if (a.dim != C::DP)
    for (int i = 0; i < STAGES; ++i) clear_stage(i);
  feed.begin(a, ring);

  uint32_t q[C::QP][NT][DT][2];
  float score_by[NT][2];     // scale of the scores of heads 2c, 2c + 1
  // Codes: the largest |weight * value's scale| of a head so far, relative to m, and the bits of the power of two above it that the
  // sums of its values are relative to.  Both go down where m goes up, so that keys count by what they add to the result.
  float peak[NT][2];
  uint32_t unit[NT][2];
  Sums<DT> sums[NT];
  // The queries of unit `out` as they are; q takes them once the unit in front has been given out.  Four values of a lane: for
  // codes they are neighbours.
  uint2 raw[C::QP][NT][DT];
  auto load_q = [&]() {
    const int kv_head = out.unit / a.head_blocks, head0 = (out.unit % a.head_blocks) * 8 * NT;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool real = head0 + n * 8 + g < a.group;
      const T *const from = static_cast<const T *>(a.q) + (int64_t)out.request * a.q_token_stride +
                            (int64_t)(kv_head * a.group + (real ? head0 + n * 8 + g : 0)) * a.q_head_stride;
#pragma unroll
      for (int k = 0; k < DT; ++k) {
        const int d = C::CODES ? (k / 4) * 64 + c * 16 + (k % 4) * 4 : k * 16 + c * 2, e = C::CODES ? d + 2 : d + 8;
        if constexpr (C::QP == 2) {
          raw[0][n][k] = raw[1][n][k] = make_uint2(0, 0);
          if (real && d < a.dim) {
            raw[0][n][k] = make_uint2(__float_as_uint(from[d]), __float_as_uint(from[d + 1]));
            raw[1][n][k] = make_uint2(__float_as_uint(from[e]), __float_as_uint(from[e + 1]));
          }
        } else {
          const uint16_t *const at = reinterpret_cast<const uint16_t *>(from);
          uint2 x = make_uint2(0, 0);
          if (a.q_pairs) {
            if (real && d < a.dim) x.x = *reinterpret_cast<const uint32_t *>(at + d);
            if (real && e < a.dim) x.y = *reinterpret_cast<const uint32_t *>(at + e);
          } else {
            if (real && d < a.dim) x.x = at[d] | (uint32_t)at[d + 1] << 16;
            if (real && e < a.dim) x.y = at[e] | (uint32_t)at[e + 1] << 16;
          }
          raw[0][n][k] = x;
        }
      }
    }
  };
  auto take_q = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      sums[n].clear();
      peak[n][0] = peak[n][1] = 0.0f;
      unit[n][0] = unit[n][1] = C::LEAST_UNIT;
      if constexpr (!C::CODES) {
        score_by[n][0] = score_by[n][1] = a.scale2;
#pragma unroll
        for (int k = 0; k < DT; ++k) {
          q[0][n][k][0] = raw[0][n][k].x;
          q[0][n][k][1] = raw[0][n][k].y;
        }
      } else {  // to [2^13, 2^14), by a power of two for each head
        constexpr bool IS_HALF = std::is_same<T, __half>::value;
        float most = 0.0f;
        auto value = [&](int k) {
          if constexpr (C::QP == 2) {
            return make_float4(__uint_as_float(raw[0][n][k].x), __uint_as_float(raw[0][n][k].y), __uint_as_float(raw[1][n][k].x), __uint_as_float(raw[1][n][k].y));
          } else {
            const float2 x = unpack2<IS_HALF>(raw[0][n][k].x), y = unpack2<IS_HALF>(raw[0][n][k].y);
            return make_float4(x.x, x.y, y.x, y.y);
          }
        };
#pragma unroll
        for (int k = 0; k < DT; ++k) {
          const float4 x = value(k);
          most = fmaxf(most, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int exponent = min(max((int)(__float_as_uint(most) >> 23), 14), 254);
        const float by = __uint_as_float((uint32_t)(267 - exponent) << 23);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int e = __shfl_sync(0xffffffffu, exponent, (2 * c + i) * 4);
          score_by[n][i] = a.scale2 * __uint_as_float((uint32_t)(e - 13) << 23);
        }
#pragma unroll
        for (int k = 0; k < DT; ++k) {
          const float4 x = value(k);
          q[0][n][k][0] = pack2<true>(x.x * by, x.y * by);
          q[0][n][k][1] = pack2<true>(x.z * by, x.w * by);
          if constexpr (C::QP == 2) {
            const float2 h0 = unpack2<true>(q[0][n][k][0]), h1 = unpack2<true>(q[0][n][k][1]);
            q[1][n][k][0] = pack2<true>(x.x * by - h0.x, x.y * by - h0.y);
            q[1][n][k][1] = pack2<true>(x.z * by - h1.x, x.w * by - h1.y);
          }
        }
      }
    }
  };
  load_q();
  int began = out.tile, stage = 0, stage_in = 0;
  bool first_piece = true;
#pragma unroll 1
  for (int ahead = 1 - STAGES;; ahead = min(ahead + 1, 0)) {  // below 0: there are not enough copies on their way
    if (ahead == 0) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();
    if (!feed.in.done) feed.fetch(a, stage_in, units);
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
    if (ahead < 0) {
      if (ahead == -1) take_q();
      continue;
    }

    const uint32_t ks = ring + stage * C::STAGE, vs = ks + KEYS * C::ROW, scales = vs + KEYS * C::ROW;
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[mt][n][0] = s[mt][n][1] = s[mt][n][2] = s[mt][n][3] = 0.0f;
      if (!C::CODES) {
        const int r = mt * 16 + (lane & 8) + (lane & 7), half = lane >> 4;
#pragma unroll
        for (int k = 0; k < DT; ++k) {
          uint32_t x[4];
          ldmatrix4(x, ks + r * C::ROW + (((2 * k + half) ^ (r & 7)) * 16));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma<C::HALF>(s[mt][n], x, q[0][n][k][0], q[0][n][k][1]);
        }
      } else {
        const int r = mt * 16 + (g >> 1) + 4 * (g & 1), swizzle = C::DP == 64 ? 0 : r & 4;
#pragma unroll
        for (int k = 0; k < DT / 4; ++k) {
          const uint4 top = load16(ks + r * C::ROW + (((k * 4 + c) ^ swizzle) * 16)), low = load16(ks + (r + 8) * C::ROW + (((k * 4 + c) ^ swizzle) * 16));
          const uint32_t tw[4] = {top.x, top.y, top.z, top.w}, lw[4] = {low.x, low.y, low.z, low.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t flip = C::STORE == LAPIS_I8 ? 0x80808080u : 0, t = tw[j] ^ flip, l = lw[j] ^ flip;
            const uint32_t x[4] = {codes2<C::STORE, false>(t), codes2<C::STORE, false>(l), codes2<C::STORE, true>(t), codes2<C::STORE, true>(l)};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (C::QP == 1) {
                mma<C::HALF>(s[mt][n], x, q[0][n][k * 4 + j][0], q[0][n][k * 4 + j][1]);
              } else {
                mma_apart(s[mt][n], x, q[1][n][k * 4 + j], q[0][n][k * 4 + j]);
              }
            }
          }
        }
      }
    }

    // scores of keys (row g, row g + 8 of the tile) and heads (2c, 2c + 1)
    const int key0 = out.span.origin + out.tile * C::TILE + warp * KEYS;
    const bool all_seen = key0 >= out.span.lo && key0 + KEYS <= out.span.hi;
    float value_scale[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = mt * 16 + e * 8 + (C::CODES ? (g >> 1) + 4 * (g & 1) : g);
        const bool seen = all_seen || (key0 + r >= out.span.lo && key0 + r < out.span.hi);
        float by = 1.0f;
        value_scale[mt][e] = 1.0f;
        if (C::CODES) {
          by = load4(scales + r * 4);
          value_scale[mt][e] = load4(scales + (KEYS + r) * 4);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          s[mt][n][2 * e] = seen ? s[mt][n][2 * e] * (score_by[n][0] * by) : -INFINITY;
          s[mt][n][2 * e + 1] = seen ? s[mt][n][2 * e + 1] * (score_by[n][1] * by) : -INFINITY;
        }
      }
    }
    float most[NT][2], base[NT][2];
    bool grows = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = sums[n].m[i];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) x = fmaxf(x, fmaxf(s[mt][n][i], s[mt][n][2 + i]));
#pragma unroll
        for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
        most[n][i] = x;
        base[n][i] = x == -INFINITY ? 0.0f : x;
        grows |= x > sums[n].m[i];
      }
    }
    // s becomes the weights, of codes times their scales
    float added[NT][2], largest[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        added[n][i] = largest[n][i] = 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float &p = s[mt][n][2 * e + i];
            p = power2(p - base[n][i]);
            added[n][i] += p;
            if (C::CODES) {
              p *= value_scale[mt][e];
              largest[n][i] = fmaxf(largest[n][i], fabsf(p));  // a caller's own scales may be negative
            }
          }
        }
        if (C::CODES) grows |= largest[n][i] > __uint_as_float(unit[n][i]);
      }
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f[i] = power2(sums[n].m[i] - base[n][i]);
          sums[n].l[i] *= f[i];
          sums[n].m[i] = most[n][i];
          if (C::CODES) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) largest[n][i] = fmaxf(largest[n][i], __shfl_xor_sync(0xffffffffu, largest[n][i], d));
            peak[n][i] = fmaxf(peak[n][i] * f[i], largest[n][i]);
            const uint32_t now = min(max((__float_as_uint(peak[n][i]) & 0x7f800000u) + 0x800000u, C::LEAST_UNIT), 0x7f000000u);
            // times unit / now, which is above 2^127 only where f is 0
            f[i] *= __uint_as_float((uint32_t)min(max((int)(unit[n][i] >> 23) - (int)(now >> 23) + 127, 0), 254) << 23);
            unit[n][i] = now;
          }
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          sums[n].o[t][0] *= f[0];
          sums[n].o[t][1] *= f[1];
          sums[n].o[t][2] *= f[0];
          sums[n].o[t][3] *= f[1];
        }
      }
    }
    float weight_by[NT][2];  // OFFSET, of codes over the unit
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sums[n].l[i] += added[n][i];
        weight_by[n][i] = C::CODES ? __uint_as_float(__float_as_uint(C::OFFSET) + 0x3f800000u - unit[n][i]) : C::OFFSET;
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t high[NT][2], low[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float p0 = s[mt][n][2 * e], p1 = s[mt][n][2 * e + 1];
          if (C::HALF) {
            p0 *= weight_by[n][0];
            p1 *= weight_by[n][1];
          }
          const uint32_t h = pack2<C::HALF>(p0, p1);
          high[n][e] = transposed(h);
          if (C::TWO_PARTS) {
            const float2 back = unpack2<C::HALF>(h);
            low[n][e] = transposed(pack2<C::HALF>(p0 - back.x, p1 - back.y));
          }
        }
      }
      if (!C::CODES) {
        const int r = mt * 16 + ((lane & 16) >> 1) + (lane & 7), half = (lane >> 3) & 1;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          uint32_t x[4];
          ldmatrix4_trans(x, vs + r * C::ROW + (((2 * t + half) ^ (r & 7)) * 16));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma<C::HALF>(sums[n].o[t], x, high[n][0], high[n][1]);
            if (C::TWO_PARTS) mma<C::HALF>(sums[n].o[t], x, low[n][0], low[n][1]);
          }
        }
      } else {
        constexpr int WORDS = C::DP == 64 ? 2 : 4;
#pragma unroll
        for (int j = 0; j < (C::DP + 127) / 128; ++j) {
          uint32_t w[4][WORDS];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = mt * 16 + 4 * i + c;
            if (C::DP == 64) {
              const uint2 x = load8(vs + r * C::ROW + (((g >> 1) ^ (r & 2)) * 16) + (g & 1) * 8);
              w[i][0] = x.x;
              w[i][1] = x.y;
            } else {
              const uint4 x = load16(vs + r * C::ROW + (((g + 8 * j) ^ ((r & 3) << 1)) * 16));
              w[i][0] = x.x;
              w[i][1] = x.y;
              w[i][WORDS - 2] = x.z;
              w[i][WORDS - 1] = x.w;
            }
          }
#pragma unroll
          for (int k = 0; k < WORDS; ++k) {
            const uint32_t flip = C::STORE == LAPIS_I8 ? 0x80808080u : 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // dimensions 4k, 4k + 1 and 4k + 2, 4k + 3: rows g and g + 8 of a tile
              const uint32_t ab = __byte_perm(w[0][k], w[1][k], h == 0 ? 0x5140 : 0x7362) ^ flip;
              const uint32_t cd = __byte_perm(w[2][k], w[3][k], h == 0 ? 0x5140 : 0x7362) ^ flip;
              const uint32_t x[4] = {codes2<C::STORE, false>(ab), codes2<C::STORE, true>(ab), codes2<C::STORE, false>(cd), codes2<C::STORE, true>(cd)};
              const int t = j * 8 + 2 * k + h;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if constexpr (C::QP == 2) {
                  mma_apart(sums[n].o[t], x, low[n], high[n]);
                } else {
                  mma<C::HALF>(sums[n].o[t], x, high[n][0], high[n][1]);
                  if (C::TWO_PARTS) mma<C::HALF>(sums[n].o[t], x, low[n][0], low[n][1]);
                }
              }
            }
          }
        }
      }
    }
    const int used = stage;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if (out.tile + 1 < out.end) {
      ++out.tile;
      continue;
    }
    const int request = out.request, head0 = (out.unit % a.head_blocks) * 8 * NT, first_head = out.unit / a.head_blocks * a.group + head0;
    const bool whole = began == 0 && out.end == out.tiles;
    note_cut(a, share, out, began);
    out.next_unit(a, units, C::TILE);
    if (!out.done) load_q();  // on its way while the sums are given out
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int d = 4; d < 32; d *= 2) sums[n].l[i] += __shfl_xor_sync(0xffffffffu, sums[n].l[i], d);
      if (C::HALF) {
        const float by[2] = {C::CODES ? __uint_as_float(unit[n][0]) / C::OFFSET : 1.0f / C::OFFSET, C::CODES ? __uint_as_float(unit[n][1]) / C::OFFSET : 1.0f / C::OFFSET};
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) sums[n].o[t][i] *= by[i & 1];
      }
      float *const part = a.partial + (((int64_t)blockIdx.x * 2 + (first_piece ? 0 : 1)) * NT + n) * C::PART;
      __syncwarp();
      give<C>(a, sums[n], mine + used * C::STAGE, STAGES * C::STAGE, request, first_head + n * 8, a.group - head0 - n * 8, whole ? nullptr : part);
    }
    if (out.done) return;
    if (a.dim != C::DP) clear_stage(used);
    first_piece = false;
    began = 0;
    take_q();
  }
}

// Adds up what the blocks left of the units that were cut: the blocks of a unit's first shares take some of its sixteens of
// dimensions each, a thread four sums of every parts-th share.  Bound by the time of its loads: the record of the cut, then the
// shares' sums, BATCH at a time.  5.5 us for units of two shares, 7 for eight units of 55; one block a unit took 15 for the latter,
// eight blocks for every unit 7.7 for the former.  512 threads join 157 shares in two trips where 256 take four (1 x 30,000: 14.7 us
// of attention and 20.5).
constexpr int JOIN_THREADS = 512;
template <typename C>
__device__ __forceinline__ void join_unit(const AttendArgs &a, const CutUnit &cut, int n, float4 (&others)[2][JOIN_THREADS]) {
  using T = typename C::T;
  constexpr int BATCH = 4;
  const int shares = cut.last - cut.first + 1, members = shares <= 8 ? 1 : min(shares, C::DT), member = (int)blockIdx.x - cut.first;
  if (cut.last == 0 || member >= members) return;
  const int each = (C::DT + members - 1) / members, parts = max(1, JOIN_THREADS / 32 / each), rounds = (each * 32 + JOIN_THREADS - 1) / JOIN_THREADS;
  const int first_head = cut.unit / a.head_blocks * a.group, head0 = (cut.unit % a.head_blocks) * 8 * C::NT + n * 8, heads = a.group - head0;
  const float4 nothing = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f);
  for (int round = 0; round < rounds; ++round) {
    const int in = round * JOIN_THREADS + (int)threadIdx.x, part = in / 32 / each % parts, t = member * each + in / 32 % each;
    const int lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
    const bool real = t < C::DT && in / 32 < each * parts;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f), ml = nothing;
    auto add = [&](const float4 &x, const float4 &xml) {
      const float m0 = fmaxf(ml.x, xml.x), m1 = fmaxf(ml.y, xml.y), b0 = m0 == -INFINITY ? 0.0f : m0, b1 = m1 == -INFINITY ? 0.0f : m1;
      const float f0 = power2(ml.x - b0), f1 = power2(ml.y - b1), e0 = power2(xml.x - b0), e1 = power2(xml.y - b1);
      acc = make_float4(acc.x * f0 + x.x * e0, acc.y * f1 + x.y * e1, acc.z * f0 + x.z * e0, acc.w * f1 + x.w * e1);
      ml = make_float4(m0, m1, ml.z * f0 + xml.z * e0, ml.w * f1 + xml.w * e1);
    };
    for (int from = part; real && from < shares; from += BATCH * parts) {
      float4 x[BATCH], xml[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int share = from + i * parts;
        const float4 *const slot = reinterpret_cast<const float4 *>(a.partial + ((int64_t)((cut.first + share) * 2 + (share > 0 ? 0 : cut.slot)) * C::NT + n) * C::PART);
        x[i] = share < shares ? slot[t * 32 + lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        xml[i] = share < shares ? slot[C::DT * 32 + c] : nothing;
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) add(x[i], xml[i]);
    }
    if (parts > 1) {
      __syncthreads();
      others[0][threadIdx.x] = acc;
      others[1][threadIdx.x] = ml;
      __syncthreads();
      if (part == 0 && real)
        for (int i = 1; i < parts; ++i) add(others[0][threadIdx.x + i * each * 32], others[1][threadIdx.x + i * each * 32]);
    }
    if (part > 0 || !real) continue;
    const int d0 = dimension<C>(t, g), d1 = C::CODES ? d0 + 1 : d0 + 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (2 * c + i >= heads) continue;
      const int64_t head = (int64_t)cut.request * a.q_heads + first_head + head0 + 2 * c + i;
      const float m = i == 0 ? ml.x : ml.y, l = i == 0 ? ml.z : ml.w, by = l == 0.0f ? 0.0f : 1.0f / l;
      if (t == 0 && g == 0 && a.lse != nullptr) a.lse[head] = l == 0.0f ? -INFINITY : m * LN2 + logf(l);
      T *const out = static_cast<T *>(a.out) + head * a.dim;
      if (d0 < a.dim) out[d0] = from_f32<T>((i == 0 ? acc.x : acc.y) * by);
      if (d1 < a.dim) out[d1] = from_f32<T>((i == 0 ? acc.z : acc.w) * by);
    }
  }
}
template <typename C>
__global__ void __launch_bounds__(JOIN_THREADS) join_mma_kernel(const __grid_constant__ AttendArgs a) {
  __shared__ float4 others[2][JOIN_THREADS];
  pdl_wait();
  const Cut cut = a.cuts[blockIdx.x];
  join_unit<C>(a, cut.begins, blockIdx.y, others);
  join_unit<C>(a, cut.goes_on, blockIdx.y, others);
}

template <typename C>
static int launch_mma(AttendArgs a, int dev, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};  // devices on which this kernel may use its shared memory
  if ((allowed.load(std::memory_order_relaxed) >> dev & 1) == 0) {
    LAPIS_CUDA_TRY(cudaFuncSetAttribute(attend_mma_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    allowed.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  a.head_blocks = (a.group + 8 * C::NT - 1) / (8 * C::NT);
  a.blocks = std::min(C::BLOCKS * sm_count(), MOST_BLOCKS);
  PoolBuf work;
  const bool whole = always_whole(a, C::TILE);
  if (!whole) LAPIS_TRY(make_workspace(a, work, 2 * C::NT * C::PART, st));
  LAPIS_CUDA_TRY(launch_pdl(attend_mma_kernel<C>, dim3(whole ? a.requests * (int)a.cache.heads * a.head_blocks : a.blocks), ATT_THREADS, C::SMEM, st, a));
  if (whole) return LAPIS_OK;
  LAPIS_CUDA_TRY(launch_pdl(join_mma_kernel<C>, dim3(a.blocks, C::NT), JOIN_THREADS, 0, st, a));
  return LAPIS_OK;
}

// Units of 8 query heads, or of 16 where more than 8 share a key head: 32 requests of up to 4096, 16 heads a key head, bf16 66 us
// (by eights, the cache read twice, 89), int8 56 (67), e4m3 of 64 41 (45).
template <typename T, int STORE>
static int launch_mma_of(const AttendArgs &a, int dev, cudaStream_t st) {
  if (a.dim <= 64) return a.group <= 8 ? launch_mma<MmaConfig<T, STORE, 64, 1>>(a, dev, st) : launch_mma<MmaConfig<T, STORE, 64, 2>>(a, dev, st);
  if (a.dim > 128) return launch_mma<MmaConfig<T, STORE, 256, 1>>(a, dev, st);
  if constexpr (!std::is_same<T, float>::value)
    if (a.group > 8) return launch_mma<MmaConfig<T, STORE, 128, 2>>(a, dev, st);
  return launch_mma<MmaConfig<T, STORE, 128, 1>>(a, dev, st);
}

// Rows of whole 8 bytes (of 32-bit numbers: of 16) from 16-byte addresses.
static bool pieces_fit(const AttendArgs &a) {
  const int64_t row = a.dim * type_bytes(a.cache.type);
  return row % (a.cache.type == LAPIS_F32 ? 16 : 8) == 0 && reinterpret_cast<uintptr_t>(a.cache.d_k) % 16 == 0 && reinterpret_cast<uintptr_t>(a.cache.d_v) % 16 == 0;
}

// 32 bits: units of 1, 4 or 8 query heads.  32 requests of up to 4096, 8 key heads of 128, 1, 4 and 8 query heads each: 99, 101 and
// 128 us; all by eights 125, 126 and 128.
template <typename T>
static int launch_type(const AttendArgs &a, int dev, cudaStream_t st) {
  if (!pieces_fit(a)) return launch_any<T>(a, dev, st);
  if (a.cache.type == LAPIS_I8) return launch_mma_of<T, LAPIS_I8>(a, dev, st);
  if (a.cache.type == LAPIS_E4M3) return launch_mma_of<T, LAPIS_E4M3>(a, dev, st);
  if constexpr (!std::is_same<T, float>::value) return launch_mma_of<T, LAPIS_F32>(a, dev, st);
  else return a.group == 1 ? launch_f32_of<1>(a, dev, st) : a.group <= 4 ? launch_f32_of<4>(a, dev, st) : launch_f32_of<8>(a, dev, st);
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
  const float scale2 = (float)(scale * 1.4426950408889634);
  if (!std::isfinite(scale2)) return fail(LAPIS_EBADARG, "%s: scale must be finite, in 32 bits", what);
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
  a.scale2 = scale2;
  a.window = window;
  a.cache = *cache;
  a.lists = *lists;
  if (cache->pages == 0) {  // nothing is read, but zeros are copied from somewhere
    a.cache.d_k = a.cache.d_v = const_cast<void *>(q->d);
    a.cache.d_k_scale = a.cache.d_v_scale = static_cast<float *>(a.cache.d_k);
  }
  a.length = d_length;
  a.out = d_out;
  a.lse = d_lse;
  cudaStream_t st = as_stream(stream);
  a.page_shift = page_shift_of(cache->page_size);
  a.q_pairs = reinterpret_cast<uintptr_t>(a.q) % 4 == 0 && a.q_token_stride % 2 == 0 && a.q_head_stride % 2 == 0;
  if (type == LAPIS_F32) return launch_type<float>(a, dev, st);
  if (type == LAPIS_F16) return launch_type<__half>(a, dev, st);
  return launch_type<__nv_bfloat16>(a, dev, st);
}

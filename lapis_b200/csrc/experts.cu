// A layer of experts: the router, the slots of each expert as CSR rows, tokens copied into that order and summed back.
//
//   route     the k largest logits of a token and their softmax, w_j = exp(l_j - m) / sum exp(l_i - m), and the logits' gradient:
//             over the chosen ones dl_e = w_e (g_e - sum_i w_i g_i), over all dl_i = [i chosen] w_i g_i - p_i sum_j w_j g_j
//   lists     a stable counting sort of the slots (token * k + j) by expert
//   gather    rows[place[t, j]] = x[t]
//   combine   out[t] = sum_j w[t, j] rows[place[t, j]]; backward: drows[place[t, j]] = w[t, j] dout[t], dw[t, j] = rows[..] . dout[t]
//
// Everything is computed in 32 bits and rounded once, sums in a fixed order.  Places, offsets and experts are looked at before
// they are followed.
//
// Kernels wait for the launch in front of them before anything else, and let the next one in as their blocks end.  Released at the top, in a stream of
// their like, the gradient of 8191 x 130 logits takes 7.4 us instead of 6.6, lists of 131,072 slots of 1024 experts 40 instead of 35, one row x 4096 x 4096
// (int4_few.cu) 6.4 instead of 5.0; lists of 160 slots 1.85 instead of 2.05, of 16,384 5.8 instead of 6.05; the others are within 1 %.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "experts.h"

namespace lapis_b200 {

// ---- router ---------------------------------------------------------------------

constexpr int ROUTE_THREADS = 128;

struct RouteArgs {
  const void *logits;
  int64_t tokens, token_stride;
  int experts, k, normalise;
  float *weights;
  int32_t *expert;
  const float *dweights;
  void *dlogits;
};

// Numbers in the order of the logits: NaN above all, -0 as 0.  0 is below all of them: no logit.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = x != x ? 0x7fffffffu : __float_as_uint(x + 0.0f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
template <typename T>
__device__ __forceinline__ uint32_t key16_of(T x) {
  if (x != x) return 0xffffu;
  const uint32_t u = *reinterpret_cast<const uint16_t *>(&x) == 0x8000u ? 0 : *reinterpret_cast<const uint16_t *>(&x);
  return u & 0x8000u ? u ^ 0xffffu : u | 0x8000u;
}
// The logit of a key (of 16-bit ones the upper half), and whether it is one that may be chosen: above -infinity.
template <typename T>
__device__ __forceinline__ float logit_of(uint32_t key) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
  } else {
    const uint32_t k = key >> 16;
    const uint16_t u = (uint16_t)(k & 0x8000u ? k ^ 0x8000u : k ^ 0xffffu);
    return to_f32(*reinterpret_cast<const T *>(&u));
  }
}
template <typename T>
__device__ __forceinline__ bool is_logit(uint32_t key) {
  constexpr uint32_t NEVER = sizeof(T) == 4 ? 0x007fffffu : std::is_same<T, __half>::value ? 0x03ffffffu : 0x007fffffu;  // of -infinity, with any number
  return key > NEVER;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}

// The two largest keys of a lane that follow the last one taken from it, and their places i (of logits lane + 32 i); of equal keys the
// lower place comes first.  16-bit logits and their numbers make one key of 32 bits, no two of which are equal.
template <bool PACKED, int R>
struct Largest {
  uint32_t key[2];
  int at[2];
  // Those of `all` behind key `last` at place `last_at`, packed ones up to `last`; 0 where there are no more.
  template <bool FROM_START>
  __device__ __forceinline__ void find(const uint32_t (&all)[R], uint32_t last, int last_at) {
    key[0] = key[1] = 0;
    at[0] = at[1] = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      uint32_t x = all[i];
      if (!FROM_START && (PACKED ? x > last : x > last || (x == last && i <= last_at))) x = 0;
      if constexpr (!PACKED) {
        const bool first = x > key[0], second = x > key[1];
        at[1] = first ? at[0] : second ? i : at[1];
        at[0] = first ? i : at[0];
      }
      key[1] = max(key[1], min(key[0], x));
      key[0] = max(key[0], x);
    }
  }
};

// A warp a token; lane l holds logits l, l + 32, ... (32 R of them at most).  A turn takes the largest key of the warp; its lane goes on to
// its second, and only when that is taken too looks through its logits again, which of 8 among 256 happens about once a token.
// Bound by the instructions on 32 bits, one every two cycles: 16,384 x 256 with a look in every turn took 15.4 us.
template <typename T, int R>
__global__ void __launch_bounds__(ROUTE_THREADS) route_kernel(const __grid_constant__ RouteArgs a) {
  constexpr bool PACKED = sizeof(T) == 2;
  const int lane = threadIdx.x % 32;
  const int64_t token = (int64_t)blockIdx.x * (ROUTE_THREADS / 32) + threadIdx.x / 32;
  pdl_wait();
  if (token >= a.tokens) return;
  const T *const logits = static_cast<const T *>(a.logits) + token * a.token_stride;
  T given[R];
#pragma unroll
  for (int i = 0; i < R; ++i) given[i] = lane + 32 * i < a.experts ? logits[lane + 32 * i] : from_f32<T>(0.0f);
  uint32_t key[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if constexpr (PACKED) key[i] = key16_of<T>(given[i]) << 16 | (0xffffu - (lane + 32 * i));
    else key[i] = key_of(given[i]);
    if (lane + 32 * i >= a.experts) key[i] = 0;
  }
  Largest<PACKED, R> mine;
  mine.template find<true>(key, 0, 0);
  int left = 2;  // of `mine`
  uint32_t most = __reduce_max_sync(0xffffffffu, mine.key[0]);
  const float top = logit_of<T>(most);
  float total = 0.0f;
  if (!a.normalise) {
#pragma unroll
    for (int i = 0; i < R; ++i) total += is_logit<T>(key[i]) ? expf(to_f32(given[i]) - top) : 0.0f;
    total = warp_sum(total);
  }
  uint32_t taken = 0;  // the key of the lane's choice, the lane-th largest
  int expert = -1;
  for (int j = 0; j < a.k && is_logit<T>(most); ++j) {
    int number;
    if constexpr (PACKED) {
      number = 0xffff - (int)(most & 0xffffu);
    } else {
      const uint32_t lanes = __ballot_sync(0xffffffffu, mine.key[0] == most);
      const int here = lane + 32 * mine.at[0];
      number = (lanes & (lanes - 1)) == 0 ? __shfl_sync(0xffffffffu, here, __ffs(lanes) - 1) : __reduce_min_sync(0xffffffffu, mine.key[0] == most ? here : 32 * R);
    }
    if (lane == j) {
      taken = most;
      expert = number;
    }
    const bool won = number % 32 == lane;
    if (won) --left;
    if (__any_sync(0xffffffffu, left == 0)) {
      if (left == 0) {
        mine.template find<false>(key, PACKED ? most - 1 : most, number / 32);
        left = 2;
      }
    } else if (won) {
      mine.key[0] = mine.key[1];
      mine.at[0] = mine.at[1];
    }
    most = __reduce_max_sync(0xffffffffu, mine.key[0]);
  }
  const float weight = expert < 0 ? 0.0f : expf(logit_of<T>(taken) - top);
  if (a.normalise) total = warp_sum(weight);
  if (lane < a.k) {
    a.weights[token * a.k + lane] = expert < 0 ? 0.0f : weight / total;
    a.expert[token * a.k + lane] = expert;
  }
}

// A warp a token: its row is written as it would be without the chosen ones, and then theirs.
template <typename T, int R>
__global__ void __launch_bounds__(ROUTE_THREADS) route_backward_kernel(const __grid_constant__ RouteArgs a) {
  const int lane = threadIdx.x % 32;
  const int64_t token = (int64_t)blockIdx.x * (ROUTE_THREADS / 32) + threadIdx.x / 32;
  pdl_wait();
  if (token >= a.tokens) return;
  const T *const logits = static_cast<const T *>(a.logits) + token * a.token_stride;
  T *const out = static_cast<T *>(a.dlogits) + token * a.experts;
  int expert = -1;
  float mine = -INFINITY, g = 0.0f;
  if (lane < a.k) {
    expert = a.expert[token * a.k + lane];
    if ((uint32_t)expert >= (uint32_t)a.experts) expert = -1;
    if (expert >= 0) {
      mine = to_f32(logits[expert]);
      g = a.dweights[token * a.k + lane];
    }
  }
  float l[R], most, total;
  if (a.normalise) {
    most = warp_max(mine);
    if (most == -INFINITY) most = 0.0f;
    mine = expf(mine - most);
    total = warp_sum(mine);
  } else {
    most = -INFINITY;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      l[i] = lane + 32 * i < a.experts ? to_f32(logits[lane + 32 * i]) : -INFINITY;
      most = fmaxf(most, l[i]);
    }
    most = warp_max(most);
    if (most == -INFINITY) most = 0.0f;
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) total += l[i] = expf(l[i] - most);
    total = warp_sum(total);
    mine = expf(mine - most);
  }
  if (total == 0.0f) total = 1.0f;
  const float w = mine / total, inner = warp_sum(expert >= 0 ? w * g : 0.0f);
  const float own = a.normalise ? w * (g - inner) : w * g;
  float sum = a.normalise ? 0.0f : -(w * inner);  // of the lane's expert, which a caller may name twice
  for (int j = 0; j < a.k; ++j) {
    const int e = __shfl_sync(0xffffffffu, expert, j);
    const float x = __shfl_sync(0xffffffffu, own, j);
    if (e == expert) sum += x;
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (lane + 32 * i < a.experts) out[lane + 32 * i] = from_f32<T>(a.normalise ? 0.0f : -(l[i] / total * inner));
  __syncwarp();
  if (expert >= 0) out[expert] = from_f32<T>(sum);
}

template <typename T, int R>
static int launch_route_as(const RouteArgs &a, cudaStream_t st) {
  const dim3 grid((unsigned)((a.tokens + ROUTE_THREADS / 32 - 1) / (ROUTE_THREADS / 32)));
  LAPIS_CUDA_TRY(a.dlogits != nullptr ? launch_pdl(route_backward_kernel<T, R>, grid, ROUTE_THREADS, 0, st, a)
                                      : launch_pdl(route_kernel<T, R>, grid, ROUTE_THREADS, 0, st, a));
  return LAPIS_OK;
}
template <typename T>
static int launch_route_of(const RouteArgs &a, cudaStream_t st) {
  if (a.experts <= 32) return launch_route_as<T, 1>(a, st);
  if (a.experts <= 64) return launch_route_as<T, 2>(a, st);
  if (a.experts <= 128) return launch_route_as<T, 4>(a, st);
  if (a.experts <= 256) return launch_route_as<T, 8>(a, st);
  if (a.experts <= 512) return launch_route_as<T, 16>(a, st);
  return launch_route_as<T, 32>(a, st);
}
static int launch_route(int type, const RouteArgs &a, cudaStream_t st) {
  switch (type) {
    case LAPIS_F32: return launch_route_of<float>(a, st);
    case LAPIS_F16: return launch_route_of<__half>(a, st);
    default: return launch_route_of<__nv_bfloat16>(a, st);
  }
}

// ---- lists ----------------------------------------------------------------------

constexpr int LIST_THREADS = 512, LIST_WARPS = LIST_THREADS / 32, LIST_MOST = 32;  // LIST_MOST: slots of a thread, where there are more rounds than one

struct ListArgs {
  const void *expert;
  int idx_bytes, experts, blocks;
  int64_t slots;
  int rounds;        // of 512 S slots for each block, one behind the other
  template <int S>
  __device__ __forceinline__ int rounds_of() const { return S < LIST_MOST ? 1 : rounds; }
  uint32_t *counts;  // [blocks, experts + 1], or null for one block
  int32_t *pos, *crd, *place;
};
// The list of a slot; `experts` for those that are no one's.
__device__ __forceinline__ int bucket_of(const ListArgs &a, int64_t slot) {
  const int64_t e = load_index(a.expert, slot, a.idx_bytes);
  return (uint64_t)e < (uint64_t)a.experts ? (int)e : a.experts;
}

// What each block's slots add to each list.
template <int S>
__global__ void __launch_bounds__(LIST_THREADS) list_count_kernel(const __grid_constant__ ListArgs a) {
  extern __shared__ uint32_t hist[];
  const int buckets = a.experts + 1;
  for (int b = threadIdx.x; b < buckets; b += LIST_THREADS) hist[b] = 0;
  pdl_wait();
  __syncthreads();
  for (int round = 0; round < a.rounds_of<S>(); ++round) {
    const int64_t first = ((int64_t)blockIdx.x * a.rounds_of<S>() + round) * LIST_THREADS * S;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int64_t slot = first + s * LIST_THREADS + threadIdx.x;
      if (slot < a.slots) atomicAdd(&hist[bucket_of(a, slot)], 1u);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < buckets; b += LIST_THREADS) a.counts[(int64_t)blockIdx.x * buckets + b] = hist[b];
}

// Every warp numbers its slots within each list (peers in a step of 32 by match), the block adds up its warps and the blocks in
// front of it, and the lists' beginnings are a scan over all lists' lengths.  Further rounds go on where the one in front ended.
template <int S>
__global__ void __launch_bounds__(LIST_THREADS) list_place_kernel(const __grid_constant__ ListArgs a) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t warp_sums[LIST_WARPS];
  const int buckets = a.experts + 1, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint32_t *const of_warp = smem, *const length = smem + LIST_WARPS * buckets, *const in_front = length + buckets, *const of_round = in_front + buckets;
  for (int i = threadIdx.x; i < (LIST_WARPS + 2) * buckets; i += LIST_THREADS) smem[i] = 0;
  pdl_wait();
  uint32_t *const mine = of_warp + warp * buckets;
  for (int round = 0; round < a.rounds_of<S>(); ++round) {
    const int64_t first = (((int64_t)blockIdx.x * a.rounds_of<S>() + round) * LIST_WARPS + warp) * 32 * S;
    int bucket[S];
    uint32_t rank[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int64_t slot = first + s * 32 + lane;
      bucket[s] = slot < a.slots ? bucket_of(a, slot) : -1;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint32_t peers = __match_any_sync(0xffffffffu, bucket[s]);
      const uint32_t before = bucket[s] >= 0 ? mine[bucket[s]] : 0;
      rank[s] = before + __popc(peers & ((1u << lane) - 1));
      __syncwarp();
      if (bucket[s] >= 0 && lane == __ffs(peers) - 1) mine[bucket[s]] = before + __popc(peers);
      __syncwarp();
    }
    if (round == 0 && a.counts != nullptr) {
      const int share = max(1, LIST_THREADS / buckets);  // threads that add up one list's counts
      for (int i = threadIdx.x; i < share * buckets; i += LIST_THREADS) {
        const int b = i % buckets;
        uint32_t all = 0, before = 0;
#pragma unroll 8
        for (int n = i / buckets; n < a.blocks; n += share) {
          const uint32_t c = a.counts[(int64_t)n * buckets + b];
          all += c;
          before += n < (int)blockIdx.x ? c : 0;
        }
        atomicAdd(&length[b], all);
        atomicAdd(&in_front[b], before);
      }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < buckets; b += LIST_THREADS) {
      uint32_t upto = 0;
#pragma unroll
      for (int w = 0; w < LIST_WARPS; ++w) {
        const uint32_t n = of_warp[w * buckets + b];
        of_warp[w * buckets + b] = upto;
        upto += n;
      }
      if constexpr (S == LIST_MOST) of_round[b] = upto;
      if (a.counts == nullptr) length[b] = upto;
    }
    __syncthreads();
    if (round == 0) {
      // Where the lists begin: a thread takes `run` lists that lie next to one another.
      const int run = (buckets + LIST_THREADS - 1) / LIST_THREADS, from = threadIdx.x * run;
      uint32_t sum = 0;
      for (int b = from; b < min(from + run, buckets); ++b) sum += length[b];
      uint32_t upto = sum;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const uint32_t below = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += below;
      }
      if (lane == 31) warp_sums[warp] = upto;
      __syncthreads();
      uint32_t begin = upto - sum;
      for (int w = 0; w < warp; ++w) begin += warp_sums[w];
      for (int b = from; b < min(from + run, buckets); ++b) {
        if (blockIdx.x == 0) a.pos[b] = (int32_t)begin;
        in_front[b] += begin;
        begin += length[b];
      }
      __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (bucket[s] < 0) continue;
      const int64_t slot = first + s * 32 + lane;
      const uint32_t at = in_front[bucket[s]] + mine[bucket[s]] + rank[s];
      a.place[slot] = (int32_t)at;
      if (at < a.slots) a.crd[at] = (int32_t)slot;  // not so only where somebody writes the experts meanwhile, which are read twice
    }
    if (round + 1 == a.rounds_of<S>()) break;
    __syncthreads();
    if constexpr (S == LIST_MOST)
      for (int b = threadIdx.x; b < buckets; b += LIST_THREADS) in_front[b] += of_round[b];
    for (int i = threadIdx.x; i < LIST_WARPS * buckets; i += LIST_THREADS) of_warp[i] = 0;
  }
}

template <int S>
static int launch_lists_as(ListArgs &a, cudaStream_t st) {
  const int buckets = a.experts + 1;
  // Every block reads the counts of all, so there are not more of them than fill the GPU: 2^27 slots of 256 experts took 42.6 ms with a block
  // for each 16,384, 4.2 ms like this.
  const int64_t chunks = std::max<int64_t>(1, (a.slots + LIST_THREADS * S - 1) / (LIST_THREADS * S));
  a.rounds = S < LIST_MOST ? 1 : (int)((chunks + 2 * sm_count() - 1) / (2 * sm_count()));
  a.blocks = (int)((chunks + a.rounds - 1) / a.rounds);
  CallBuf counts;
  if (a.blocks > 1) {
    LAPIS_TRY(scratch(&counts, (size_t)a.blocks * buckets * sizeof(uint32_t), st));
    a.counts = static_cast<uint32_t *>(counts.p);
    LAPIS_CUDA_TRY(launch_pdl(list_count_kernel<S>, dim3(a.blocks), LIST_THREADS, buckets * sizeof(uint32_t), st, a));
  }
  const size_t smem = (LIST_WARPS + 3) * buckets * sizeof(uint32_t);
  LAPIS_TRY(allow_smem<list_place_kernel<S>>((int)((LIST_WARPS + 3) * (MAX_EXPERTS + 1) * sizeof(uint32_t))));
  LAPIS_CUDA_TRY(launch_pdl(list_place_kernel<S>, dim3(a.blocks), LIST_THREADS, smem, st, a));
  return LAPIS_OK;
}
static int launch_lists(ListArgs &a, cudaStream_t st) {
  // One block, where its turns take less than a second launch.
  if (a.slots <= LIST_THREADS) return launch_lists_as<1>(a, st);
  if (a.slots <= 2 * LIST_THREADS) return launch_lists_as<2>(a, st);
  if (a.slots <= 4 * LIST_THREADS) return launch_lists_as<4>(a, st);
  if (a.slots <= 8 * LIST_THREADS) return launch_lists_as<8>(a, st);
  const int64_t all = a.slots / sm_count();
  if (all <= LIST_THREADS) return launch_lists_as<1>(a, st);
  if (all <= 2 * LIST_THREADS) return launch_lists_as<2>(a, st);
  if (all <= 4 * LIST_THREADS) return launch_lists_as<4>(a, st);
  if (all <= 8 * LIST_THREADS) return launch_lists_as<8>(a, st);
  return launch_lists_as<LIST_MOST>(a, st);
}

// ---- rows there and back ----------------------------------------------------------

constexpr int ROWS_THREADS = 256;

struct RowsArgs {
  const void *x, *rows;
  int64_t x_stride, row_stride, dim;  // strides in elements
  int64_t tokens, slots;
  int k, experts;
  int64_t items;
  uint32_t chunks;  // items of a row
  int run;          // of combine: what an item has of them, in turns of its loop
  const int32_t *pos, *place;
  const float *weights;
  void *out;
  float *dweights;
};
// A slot's place, or -1 where the list names none, and whether there is an expert at it.
struct Place {
  int32_t at;
  bool here;
};
__device__ __forceinline__ Place place_of(const RowsArgs &a, int64_t slot, int32_t end) {
  const int32_t at = a.place[slot];
  return {(uint32_t)at < (uint64_t)a.slots ? at : -1, (uint32_t)at < (uint64_t)a.slots && at < end};
}
__device__ __forceinline__ int64_t divided(int64_t item, uint32_t by, int64_t items) {
  return items <= 0xffffffffll ? (int64_t)((uint32_t)item / by) : item / by;
}

// A piece of a row: V elements, 16 bytes where rows allow it.
template <typename T, int V>
struct alignas(sizeof(T) * V) Piece {
  T v[V];
};

// A warp an item: GATHER_PIECES pieces a lane of a token's row, read once and written k times.
constexpr int GATHER_PIECES = 2;  // 16,384 x 8 rows of 2048 106.9 us, with 4 108.5, with 8 108.8; 40 x 4 rows 2.7 us, 3.3, 4.3
template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS) gather_kernel(const __grid_constant__ RowsArgs a) {
  using P = Piece<T, V>;
  const int lane = threadIdx.x % 32;
  const int64_t item = (int64_t)blockIdx.x * (ROWS_THREADS / 32) + threadIdx.x / 32;
  pdl_wait();
  if (item >= a.items) return;
  const int64_t token = divided(item, a.chunks, a.items);
  const int64_t first = (item - token * a.chunks) * (32 * GATHER_PIECES) + lane, pieces = a.dim / V;
  const P *const from = reinterpret_cast<const P *>(static_cast<const T *>(a.x) + token * a.x_stride);
  const int32_t end = a.pos[a.experts];
  P got[GATHER_PIECES] = {};
#pragma unroll
  for (int u = 0; u < GATHER_PIECES; ++u)
    if (first + u * 32 < pieces) got[u] = from[first + u * 32];
  for (int j0 = 0; j0 < a.k; j0 += 32) {
    const Place p = j0 + lane < a.k ? place_of(a, token * a.k + j0 + lane, end) : Place{-1, false};
    for (int j = 0; j < min(32, a.k - j0); ++j) {
      const int32_t at = __shfl_sync(0xffffffffu, p.at, j);
      const bool here = __shfl_sync(0xffffffffu, p.here, j);
      if (at < 0) continue;
      P *const to = reinterpret_cast<P *>(static_cast<T *>(a.out) + at * a.dim);
#pragma unroll
      for (int u = 0; u < GATHER_PIECES; ++u)
        if (first + u * 32 < pieces) to[first + u * 32] = here ? got[u] : P{};
    }
  }
}

__device__ __forceinline__ float2 pair_of(uint32_t word, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&word)); }
__device__ __forceinline__ float2 pair_of(uint32_t word, __nv_bfloat16) { return make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u)); }

// Rows of 16-byte pieces.  A warp takes (token, chunk) after (token, chunk); for each it needs J rows at a time, C pieces a lane of each,
// which come by cp.async into a ring of its own: every lane copies what it will add, so that nothing but its own copies is waited for.
// Bound by memory.  What it takes is bytes in flight: rows of eight places a token, 16 warps an SM with 8 KB each on their way.
constexpr int RING_STAGES = 3, RING_WARPS = 8;
template <typename T, int J>
__global__ void __launch_bounds__(32 * RING_WARPS, 2) combine_ring_kernel(const __grid_constant__ RowsArgs a) {
  constexpr int C = 8 / J, V = 16 / sizeof(T), STAGE = 32 * 8 * 16;
  extern __shared__ __align__(16) uint8_t rings[];
  __shared__ float weight_of[RING_WARPS][RING_STAGES][J];
  __shared__ uint32_t here_of[RING_WARPS][RING_STAGES];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint8_t *const ring = rings + warp * RING_STAGES * STAGE + lane * 16;
  const int64_t step = (int64_t)gridDim.x * RING_WARPS;
  const int pieces = (int)(a.dim / V);
  pdl_wait();
  const int32_t end = a.pos[a.experts];

  struct Unit {  // rows j0 to j0 + J - 1 of a token's chunk
    int64_t item, token;
    int j0, first;
  };
  const auto place = [&](Unit &u) {
    if (u.item >= a.items) return;
    u.token = divided(u.item, a.chunks, a.items);
    u.first = (int)(u.item - u.token * a.chunks) * (32 * C) + lane;
  };
  const auto advance = [&](Unit &u) {
    u.j0 += J;
    if (u.j0 < a.k) return;
    u.j0 = 0;
    u.item += step;
    place(u);
  };
  Unit next = {(int64_t)blockIdx.x * RING_WARPS + warp, 0, 0, 0}, now = next;
  place(next);
  now = next;
  int32_t at = -1;  // of the next unit: the lane's row, or -1, and its weight
  float w = 1.0f;
  const auto look = [&] {
    at = -1;
    if (next.item >= a.items || lane >= J || next.j0 + lane >= a.k) return;
    const int64_t slot = next.token * a.k + next.j0 + lane;
    const Place p = place_of(a, slot, end);
    at = p.here ? p.at : -1;
    if (a.weights != nullptr) w = a.weights[slot];
  };
  const auto ask = [&](int stage) {
    if (next.item < a.items) {
      const uint32_t here = __ballot_sync(0xffffffffu, at >= 0);
      if (lane < J) weight_of[warp][stage][lane] = w;
      if (lane == 0) here_of[warp][stage] = here;
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + stage * STAGE);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int32_t row = __shfl_sync(0xffffffffu, at, j);
        const uint4 *const from = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.rows) + row * a.row_stride) + next.first;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (row >= 0 && next.first + c * 32 < pieces)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (j * C + c) * 512), "l"(from + c * 32) : "memory");
      }
      advance(next);
      look();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look();
#pragma unroll
  for (int s = 0; s < RING_STAGES - 1; ++s) ask(s);
  float2 sum[C][V / 2] = {};
  for (int stage = 0; now.item < a.items; stage = stage == RING_STAGES - 1 ? 0 : stage + 1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(RING_STAGES - 2) : "memory");
    __syncwarp();
    const uint32_t here = here_of[warp][stage];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (!(here >> j & 1)) continue;
      const float wj = weight_of[warp][stage][j];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint4 v = *reinterpret_cast<const uint4 *>(ring + stage * STAGE + (j * C + c) * 512);
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          float2 x;
          if constexpr (sizeof(T) == 2) x = pair_of(words[i], T());
          else x = make_float2(__uint_as_float(words[2 * i]), __uint_as_float(words[2 * i + 1]));
          sum[c][i] = fma2(make_float2(wj, wj), x, sum[c][i]);
        }
      }
    }
    if (now.j0 + J >= a.k) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        Piece<T, V> done;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          done.v[2 * i] = from_f32<T>(sum[c][i].x);
          done.v[2 * i + 1] = from_f32<T>(sum[c][i].y);
          sum[c][i] = make_float2(0.0f, 0.0f);
        }
        if (now.first + c * 32 < pieces) reinterpret_cast<Piece<T, V> *>(static_cast<T *>(a.out) + now.token * a.dim)[now.first + c * 32] = done;
      }
    }
    advance(now);
    __syncwarp();  // here_of and weight_of of the stage in front, which is asked into now, have been read
    ask(stage == 0 ? RING_STAGES - 1 : stage - 1);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Rows of any alignment.  A warp an item: `run` chunks of 32 U elements of a token's row, J rows asked for at a time.
template <typename T, int U, int J>
__global__ void __launch_bounds__(ROWS_THREADS, 4) combine_kernel(const __grid_constant__ RowsArgs a) {
  const int lane = threadIdx.x % 32;
  const int64_t item = (int64_t)blockIdx.x * (ROWS_THREADS / 32) + threadIdx.x / 32;
  pdl_wait();
  if (item >= a.items) return;
  const int64_t token = divided(item, a.chunks, a.items);
  const int chunk = (int)(item - token * a.chunks), dim = (int)a.dim;
  const int32_t end = a.pos[a.experts];
  const uint32_t upto = min((uint32_t)dim, (uint32_t)(chunk + 1) * a.run * 32 * U);
  for (uint32_t from = (uint32_t)chunk * a.run * 32 * U; from < upto; from += 32 * U) {
    const int first = (int)from + lane;
    float sum[U] = {};
    for (int j0 = 0; j0 < a.k; j0 += 32) {
      const Place p = j0 + lane < a.k ? place_of(a, token * a.k + j0 + lane, end) : Place{-1, false};
      const int32_t mine = p.here ? p.at : -1;
      const float weight = a.weights != nullptr && p.here ? a.weights[token * a.k + j0 + lane] : 1.0f;
      for (int j1 = 0; j1 < min(32, a.k - j0); j1 += J) {
        T got[J][U];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int32_t at = __shfl_sync(0xffffffffu, mine, j1 + j);
          const T *const row = static_cast<const T *>(a.rows) + at * a.row_stride;
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (at >= 0 && first + u * 32 < dim) got[j][u] = row[first + u * 32];
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const bool here = __shfl_sync(0xffffffffu, mine, j1 + j) >= 0;
          const float w = __shfl_sync(0xffffffffu, weight, j1 + j);
          if (!here) continue;
#pragma unroll
          for (int u = 0; u < U; ++u) sum[u] = fmaf(w, to_f32(got[j][u]), sum[u]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * 32 < dim) static_cast<T *>(a.out)[token * a.dim + first + u * 32] = from_f32<T>(sum[u]);
  }
}

__device__ __forceinline__ uint32_t word_of(float2 x, __half) {
  const __half2 h = __float22half2_rn(x);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t word_of(float2 x, __nv_bfloat16) {
  const __nv_bfloat162 h = __float22bfloat162_rn(x);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// A warp a slot: its row's product with dout of its token, and its weight times dout.  16-bit pieces stay words until they are used: as
// arrays of elements they took 89 registers, and the warps that memory needs did not fit.
constexpr int BACK_PIECES = 4, BACK_BLOCKS = 4;  // 8192 x 6 rows of 5120 164 us; 5 blocks an SM (spills) 169, 2 pieces 167
template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS, BACK_BLOCKS) combine_backward_kernel(const __grid_constant__ RowsArgs a) {
  using P = typename std::conditional<V == 1, T, uint4>::type;
  const int lane = threadIdx.x % 32;
  const int64_t slot = (int64_t)blockIdx.x * (ROWS_THREADS / 32) + threadIdx.x / 32;
  pdl_wait();
  if (slot >= a.slots) return;
  const int64_t token = divided(slot, a.k, a.slots);
  const int pieces = (int)(a.dim / V);
  const Place p = place_of(a, slot, a.pos[a.experts]);
  P *const to = reinterpret_cast<P *>(static_cast<T *>(a.out) + max(p.at, 0) * a.dim);
  float2 dot = make_float2(0.0f, 0.0f);
  if (p.here) {
    const P *const dout = reinterpret_cast<const P *>(static_cast<const T *>(a.x) + token * a.x_stride);
    const P *const row = reinterpret_cast<const P *>(static_cast<const T *>(a.rows) + p.at * a.row_stride);
    const float w = a.weights[slot];
    for (int first = lane; first < pieces; first += 32 * BACK_PIECES) {
      P d[BACK_PIECES], r[BACK_PIECES];
#pragma unroll
      for (int u = 0; u < BACK_PIECES; ++u)
        if (first + u * 32 < pieces) {
          d[u] = dout[first + u * 32];
          r[u] = row[first + u * 32];
        }
#pragma unroll
      for (int u = 0; u < BACK_PIECES; ++u) {
        if (first + u * 32 >= pieces) continue;
        if constexpr (V == 1) {
          dot.x = fmaf(to_f32(d[u]), to_f32(r[u]), dot.x);
          to[first + u * 32] = from_f32<T>(w * to_f32(d[u]));
        } else {
          const uint32_t dw[4] = {d[u].x, d[u].y, d[u].z, d[u].w}, rw[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
          uint32_t out[4];
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 x = pair_of(dw[i], T());
              dot = fma2(x, pair_of(rw[i], T()), dot);
              out[i] = word_of(mul2(make_float2(w, w), x), T());
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float2 x = make_float2(__uint_as_float(dw[i]), __uint_as_float(dw[i + 1]));
              dot = fma2(x, make_float2(__uint_as_float(rw[i]), __uint_as_float(rw[i + 1])), dot);
              const float2 y = mul2(make_float2(w, w), x);
              out[i] = __float_as_uint(y.x), out[i + 1] = __float_as_uint(y.y);
            }
          }
          to[first + u * 32] = make_uint4(out[0], out[1], out[2], out[3]);
        }
      }
    }
  } else if (p.at >= 0) {
    for (int i = lane; i < pieces; i += 32) to[i] = P{};
  }
  const float all = warp_sum(dot.x + dot.y);
  if (lane == 0) a.dweights[slot] = all;
}

// ---- the same for narrow rows -----------------------------------------------------

// Rows of up to so many pieces leave lanes of a warp without work where a warp takes a row: there a thread takes a piece.  38,933 x 4 rows of
// bf16, us, a warp a row and a thread a piece: combined 128 wide 29.7 and 12.2, 256 wide 31.9 and 23.9; gradients 70 and 25, 76 and 51;
// copied 128 wide 25.5 and 24.4 with the lists, 256 wide 27.2 and 38.8, as a thread reads its piece for every slot.
constexpr int NARROW = 32, NARROW_GATHER = 16;

template <typename T, int V>
__device__ __forceinline__ void to_floats(float (&x)[V], const Piece<T, V> &p) {
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = to_f32(p.v[v]);
}

template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS) gather_narrow_kernel(const __grid_constant__ RowsArgs a) {
  using P = Piece<T, V>;
  const int64_t item = (int64_t)blockIdx.x * ROWS_THREADS + threadIdx.x;
  pdl_wait();
  if (item >= a.items) return;
  const int64_t slot = divided(item, a.chunks, a.items), token = divided(slot, a.k, a.slots);
  const int piece = (int)(item - slot * a.chunks);
  const Place p = place_of(a, slot, a.pos[a.experts]);
  if (p.at < 0) return;
  P got = {};
  if (p.here) got = reinterpret_cast<const P *>(static_cast<const T *>(a.x) + token * a.x_stride)[piece];
  reinterpret_cast<P *>(static_cast<T *>(a.out) + p.at * a.dim)[piece] = got;
}

template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS) combine_narrow_kernel(const __grid_constant__ RowsArgs a) {
  using P = Piece<T, V>;
  constexpr int J = 4;  // rows asked for at a time
  const int64_t item = (int64_t)blockIdx.x * ROWS_THREADS + threadIdx.x;
  pdl_wait();
  if (item >= a.items) return;
  const int64_t token = divided(item, a.chunks, a.items);
  const int piece = (int)(item - token * a.chunks);
  const int32_t end = a.pos[a.experts];
  float sum[V] = {};
  for (int j0 = 0; j0 < a.k; j0 += J) {
    Place p[J];
    P got[J];
#pragma unroll
    for (int j = 0; j < J; ++j) p[j] = j0 + j < a.k ? place_of(a, token * a.k + j0 + j, end) : Place{-1, false};
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (p[j].here) got[j] = reinterpret_cast<const P *>(static_cast<const T *>(a.rows) + p[j].at * a.row_stride)[piece];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (!p[j].here) continue;
      const float w = a.weights != nullptr ? a.weights[token * a.k + j0 + j] : 1.0f;
      float x[V];
      to_floats<T, V>(x, got[j]);
#pragma unroll
      for (int v = 0; v < V; ++v) sum[v] = fmaf(w, x[v], sum[v]);
    }
  }
  P done;
#pragma unroll
  for (int v = 0; v < V; ++v) done.v[v] = from_f32<T>(sum[v]);
  reinterpret_cast<P *>(static_cast<T *>(a.out) + token * a.dim)[piece] = done;
}

// a.run lanes, a power of two, take a slot.
template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS) combine_backward_narrow_kernel(const __grid_constant__ RowsArgs a) {
  using P = Piece<T, V>;
  const int64_t slot = ((int64_t)blockIdx.x * ROWS_THREADS + threadIdx.x) / a.run;
  const int piece = threadIdx.x & (a.run - 1);
  pdl_wait();
  float dot = 0.0f;
  if (slot < a.slots) {
    const Place p = place_of(a, slot, a.pos[a.experts]);
    if (piece < (int)a.chunks && p.at >= 0) {
      P done = {};
      if (p.here) {
        const float w = a.weights[slot];
        float d[V], r[V];
        to_floats<T, V>(d, reinterpret_cast<const P *>(static_cast<const T *>(a.x) + divided(slot, a.k, a.slots) * a.x_stride)[piece]);
        to_floats<T, V>(r, reinterpret_cast<const P *>(static_cast<const T *>(a.rows) + p.at * a.row_stride)[piece]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          dot = fmaf(d[v], r[v], dot);
          done.v[v] = from_f32<T>(w * d[v]);
        }
      }
      reinterpret_cast<P *>(static_cast<T *>(a.out) + p.at * a.dim)[piece] = done;
    }
  }
  for (int d = a.run / 2; d > 0; d /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
  if (slot < a.slots && piece == 0) a.dweights[slot] = dot;
}

enum RowsOp { GATHER, COMBINE, COMBINE_BACKWARD };

template <typename T, int J>
static int launch_ring(RowsArgs &a, cudaStream_t st) {
  const int64_t lanes = (a.dim * (int)sizeof(T) / 16 + 31) / 32;
  a.chunks = (uint32_t)((lanes + 8 / J - 1) / (8 / J));
  a.items = a.tokens * a.chunks;
  const int smem = RING_WARPS * RING_STAGES * 32 * 8 * 16;
  LAPIS_TRY((allow_smem<combine_ring_kernel<T, J>>(smem)));
  const int64_t blocks = std::min<int64_t>(2 * sm_count(), (a.items + RING_WARPS - 1) / RING_WARPS);
  LAPIS_CUDA_TRY(launch_pdl(combine_ring_kernel<T, J>, dim3((unsigned)blocks), 32 * RING_WARPS, smem, st, a));
  return LAPIS_OK;
}
template <typename T, int V>
static int launch_combine(RowsArgs &a, cudaStream_t st) {
  if constexpr (V > 1) {
    return a.k <= 1 ? launch_ring<T, 1>(a, st) : a.k <= 2 ? launch_ring<T, 2>(a, st) : launch_ring<T, 4>(a, st);
  } else {
    constexpr int WARPS = ROWS_THREADS / 32, U = 8;
    // A warp looks up a token's places once for several pieces, where there are warps enough for that.
    const int64_t turns = (a.dim + 32 * U - 1) / (32 * U), warps = (int64_t)sm_count() * 128;
    a.run = (int)std::min<int64_t>(turns, std::max<int64_t>(1, a.tokens * turns / warps));
    a.chunks = (uint32_t)((turns + a.run - 1) / a.run);
    a.items = a.tokens * a.chunks;
    const int64_t blocks = (a.items + WARPS - 1) / WARPS;
    if (blocks > 0x7fffffff) return fail(LAPIS_ETOOBIG, "experts: rows beyond 2^31 blocks");
    LAPIS_CUDA_TRY(launch_pdl(combine_kernel<T, U, 2>, dim3((unsigned)blocks), ROWS_THREADS, 0, st, a));
    return LAPIS_OK;
  }
}
template <typename T, int V>
static int launch_narrow(RowsOp op, RowsArgs &a, cudaStream_t st) {
  a.chunks = (uint32_t)(a.dim / V);  // pieces
  for (a.run = 1; a.run < (int)a.chunks;) a.run *= 2;
  a.items = op == GATHER ? a.slots * a.chunks : op == COMBINE ? a.tokens * a.chunks : a.slots * a.run;
  const int64_t blocks = (a.items + ROWS_THREADS - 1) / ROWS_THREADS;
  if (blocks > 0x7fffffff) return fail(LAPIS_ETOOBIG, "experts: rows beyond 2^31 blocks");
  LAPIS_CUDA_TRY(op == GATHER ? launch_pdl(gather_narrow_kernel<T, V>, dim3((unsigned)blocks), ROWS_THREADS, 0, st, a)
                 : op == COMBINE ? launch_pdl(combine_narrow_kernel<T, V>, dim3((unsigned)blocks), ROWS_THREADS, 0, st, a)
                                 : launch_pdl(combine_backward_narrow_kernel<T, V>, dim3((unsigned)blocks), ROWS_THREADS, 0, st, a));
  return LAPIS_OK;
}
template <typename T, int V>
static int launch_rows_as(RowsOp op, RowsArgs &a, cudaStream_t st) {
  constexpr int WARPS = ROWS_THREADS / 32;
  if (a.dim / V <= (op == GATHER ? NARROW_GATHER : NARROW)) return launch_narrow<T, V>(op, a, st);
  if (op == COMBINE) return launch_combine<T, V>(a, st);
  const int64_t lanes = (a.dim / V + 31) / 32;
  a.chunks = (uint32_t)((lanes + GATHER_PIECES - 1) / GATHER_PIECES);
  a.items = op == COMBINE_BACKWARD ? a.slots : a.tokens * a.chunks;
  const int64_t blocks = (a.items + WARPS - 1) / WARPS;
  if (blocks > 0x7fffffff) return fail(LAPIS_ETOOBIG, "experts: rows beyond 2^31 blocks");
  LAPIS_CUDA_TRY(op == GATHER ? launch_pdl(gather_kernel<T, V>, dim3((unsigned)blocks), ROWS_THREADS, 0, st, a)
                              : launch_pdl(combine_backward_kernel<T, V>, dim3((unsigned)blocks), ROWS_THREADS, 0, st, a));
  return LAPIS_OK;
}
static bool fits(const void *p, int64_t stride, int bytes, int align) { return reinterpret_cast<uintptr_t>(p) % align == 0 && stride * bytes % align == 0; }
template <typename T>
static int launch_rows_of(RowsOp op, RowsArgs &a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = fits(a.x, a.x_stride, sizeof(T), 16) && fits(a.rows, a.row_stride, sizeof(T), 16) && fits(a.out, a.dim, sizeof(T), 16);
  return wide ? launch_rows_as<T, V>(op, a, st) : launch_rows_as<T, 1>(op, a, st);
}
static int launch_rows(int type, RowsOp op, RowsArgs &a, cudaStream_t st) {
  switch (type) {
    case LAPIS_F32: return launch_rows_of<float>(op, a, st);
    case LAPIS_F16: return launch_rows_of<__half>(op, a, st);
    default: return launch_rows_of<__nv_bfloat16>(op, a, st);
  }
}

// ---- checks -----------------------------------------------------------------------

int check_expert_lists(const char *what, const lapis_b200_expert_lists *l) {
  if (l == nullptr) return fail(LAPIS_EBADARG, "%s: null lists", what);
  if (l->tokens < 0 || l->k < 0 || l->experts < 0) return fail(LAPIS_EBADSHAPE, "%s: negative size", what);
  if (l->experts > MAX_EXPERTS) return fail(LAPIS_ETOOBIG, "%s: more than %d experts", what, MAX_EXPERTS);
  if (l->k > 0 && l->tokens > 0x7fffffff / l->k) return fail(LAPIS_ETOOBIG, "%s: 2^31 slots or more", what);
  if (l->d_pos == nullptr || (l->tokens * l->k > 0 && (l->d_crd == nullptr || l->d_place == nullptr))) return fail(LAPIS_EBADARG, "%s: null list", what);
  return LAPIS_OK;
}
static int check_rows(const char *what, int type, int64_t dim, const lapis_b200_expert_lists *lists) {
  if (!is_float_type(type)) return fail(LAPIS_EBADARG, "%s: type must be LAPIS_F32, LAPIS_F16 or LAPIS_BF16", what);
  LAPIS_TRY(check_expert_lists(what, lists));
  if (dim < 0) return fail(LAPIS_EBADSHAPE, "%s: negative size", what);
  if (dim > 1 << 30) return fail(LAPIS_ETOOBIG, "%s: rows of more than 2^30 elements", what);
  return LAPIS_OK;
}
static RowsArgs rows_args(int64_t dim, const lapis_b200_expert_lists *l) {
  RowsArgs a = {};
  a.dim = dim;
  a.tokens = l->tokens;
  a.slots = l->tokens * l->k;
  a.k = (int)l->k;
  a.experts = (int)l->experts;
  a.pos = l->d_pos;
  a.place = l->d_place;
  return a;
}
static int check_route(const char *what, int type, int64_t tokens, int64_t experts, const void *d_logits, int64_t k) {
  if (!is_float_type(type)) return fail(LAPIS_EBADARG, "%s: type must be LAPIS_F32, LAPIS_F16 or LAPIS_BF16", what);
  if (tokens < 0 || experts < 0 || k < 0) return fail(LAPIS_EBADSHAPE, "%s: negative size", what);
  if (k > experts) return fail(LAPIS_EBADSHAPE, "%s: more choices than experts", what);
  if (experts > MAX_EXPERTS) return fail(LAPIS_ETOOBIG, "%s: more than %d experts", what, MAX_EXPERTS);
  if (k > MAX_CHOSEN) return fail(LAPIS_ETOOBIG, "%s: more than %d choices", what, MAX_CHOSEN);
  if (tokens > 0x7fffffff) return fail(LAPIS_ETOOBIG, "%s: 2^31 tokens or more", what);
  if (tokens > 0 && experts > 0 && d_logits == nullptr) return fail(LAPIS_EBADARG, "%s: null operand", what);
  return LAPIS_OK;
}

}  // namespace lapis_b200

using namespace lapis_b200;

extern "C" int lapis_b200_route(int type, int64_t tokens, int64_t experts, const void *d_logits, int64_t token_stride, int64_t k, int normalise,
                                float *d_weights, int32_t *d_expert, void *stream) {
  clear_error();
  const char *what = "route";
  LAPIS_TRY(check_route(what, type, tokens, experts, d_logits, k));
  if (tokens == 0 || k == 0) return LAPIS_OK;
  if (d_weights == nullptr || d_expert == nullptr) return fail(LAPIS_EBADARG, "%s: null operand", what);
  RouteArgs a = {};
  a.logits = d_logits;
  a.tokens = tokens;
  a.token_stride = token_stride;
  a.experts = (int)experts;
  a.k = (int)k;
  a.normalise = normalise != 0;
  a.weights = d_weights;
  a.expert = d_expert;
  return launch_route(type, a, as_stream(stream));
}

extern "C" int lapis_b200_route_backward(int type, int64_t tokens, int64_t experts, const void *d_logits, int64_t token_stride, int64_t k, int normalise,
                                         const int32_t *d_expert, const float *d_dweights, void *d_dlogits, void *stream) {
  clear_error();
  const char *what = "route_backward";
  LAPIS_TRY(check_route(what, type, tokens, experts, d_logits, k));
  if (tokens == 0 || experts == 0) return LAPIS_OK;
  if (d_dlogits == nullptr || (k > 0 && (d_expert == nullptr || d_dweights == nullptr))) return fail(LAPIS_EBADARG, "%s: null operand", what);
  RouteArgs a = {};
  a.logits = d_logits;
  a.tokens = tokens;
  a.token_stride = token_stride;
  a.experts = (int)experts;
  a.k = (int)k;
  a.normalise = normalise != 0;
  a.expert = const_cast<int32_t *>(d_expert);
  a.dweights = d_dweights;
  a.dlogits = d_dlogits;
  return launch_route(type, a, as_stream(stream));
}

extern "C" int lapis_b200_expert_lists_make(int idx_bytes, int64_t tokens, int64_t k, int64_t experts, const void *d_expert, int32_t *d_pos, int32_t *d_crd,
                                            int32_t *d_place, void *stream) {
  clear_error();
  const char *what = "expert_lists";
  const lapis_b200_expert_lists l = {tokens, k, experts, d_pos, d_crd, d_place};
  if (idx_bytes != 4 && idx_bytes != 8) return fail(LAPIS_EBADARG, "%s: idx_bytes must be 4 or 8", what);
  LAPIS_TRY(check_expert_lists(what, &l));
  if (tokens * k > 0 && d_expert == nullptr) return fail(LAPIS_EBADARG, "%s: null operand", what);
  ListArgs a = {};
  a.expert = d_expert;
  a.idx_bytes = idx_bytes;
  a.experts = (int)experts;
  a.slots = tokens * k;
  a.pos = d_pos;
  a.crd = d_crd;
  a.place = d_place;
  return launch_lists(a, as_stream(stream));
}

extern "C" int lapis_b200_expert_gather(int type, int64_t dim, const void *d_x, int64_t x_stride, const lapis_b200_expert_lists *lists, void *d_rows,
                                        void *stream) {
  clear_error();
  const char *what = "expert_gather";
  LAPIS_TRY(check_rows(what, type, dim, lists));
  RowsArgs a = rows_args(dim, lists);
  if (a.slots == 0 || dim == 0) return LAPIS_OK;
  if (d_x == nullptr || d_rows == nullptr) return fail(LAPIS_EBADARG, "%s: null operand", what);
  a.x = d_x;
  a.x_stride = x_stride;
  a.out = d_rows;
  return launch_rows(type, GATHER, a, as_stream(stream));
}

extern "C" int lapis_b200_expert_combine(int type, int64_t dim, const void *d_rows, int64_t row_stride, const lapis_b200_expert_lists *lists,
                                         const float *d_weights, void *d_out, void *stream) {
  clear_error();
  const char *what = "expert_combine";
  LAPIS_TRY(check_rows(what, type, dim, lists));
  RowsArgs a = rows_args(dim, lists);
  if (a.tokens == 0 || dim == 0) return LAPIS_OK;
  if (d_out == nullptr || (a.slots > 0 && d_rows == nullptr)) return fail(LAPIS_EBADARG, "%s: null operand", what);
  a.rows = d_rows;
  a.row_stride = row_stride;
  a.weights = d_weights;
  a.out = d_out;
  return launch_rows(type, COMBINE, a, as_stream(stream));
}

extern "C" int lapis_b200_expert_combine_backward(int type, int64_t dim, const void *d_dout, int64_t dout_stride, const void *d_rows, int64_t row_stride,
                                                  const lapis_b200_expert_lists *lists, const float *d_weights, void *d_drows, float *d_dweights,
                                                  void *stream) {
  clear_error();
  const char *what = "expert_combine_backward";
  LAPIS_TRY(check_rows(what, type, dim, lists));
  RowsArgs a = rows_args(dim, lists);
  if (a.slots == 0) return LAPIS_OK;
  if (d_weights == nullptr || d_dweights == nullptr || (dim > 0 && (d_dout == nullptr || d_rows == nullptr || d_drows == nullptr)))
    return fail(LAPIS_EBADARG, "%s: null operand", what);
  a.x = d_dout;
  a.x_stride = dout_stride;
  a.rows = d_rows;
  a.row_stride = row_stride;
  a.weights = d_weights;
  a.out = d_drows;
  a.dweights = d_dweights;
  return launch_rows(type, COMBINE_BACKWARD, a, as_stream(stream));
}

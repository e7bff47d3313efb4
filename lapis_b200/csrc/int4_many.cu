// Products of many rows with 4-bit weights (int4.cu) on tcgen05: 128 outputs a tile, up to 128 columns of the product at a time.
//
// mma.sync reads the rows x from shared memory once for every 16 outputs, and takes 8 cycles for 16 x 8 x 16: from 16 columns on the two take
// longer than the weights (64 rows x 14,336 x 4096: 84 us).  Here a tile's codes become numbers in tensor memory, as the A operand of
// 128 x N x 16, and the rows x lie in shared memory as its B operand, so that a byte of either is handled once for 128 outputs.  A
// group's sum is read from tensor memory, scaled and added in registers.
//
// Two launches.  arrange_kernel lays the rows out as the blocks of 64 columns that lie in shared memory (swizzled, 32-bit values in three
// parts, rows fetched by lists, zeros behind the last column), once for all tiles; a tile has such a block by one bulk copy.  In
// int4_many_kernel eight warps convert codes, a strip each, and add the groups' sums, one thread copies blocks and one issues the
// products.  Where a matrix has few tiles, the CTAs of a cluster share a tile's columns, and their sums meet in distributed shared
// memory.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "int4.h"
#include "tcgen05.h"

namespace lapis_b200 {

constexpr int MANY_WARPS = 8, MANY_THREADS = 32 * (MANY_WARPS + 2);  // a warp copies, a warp issues
constexpr int X_STAGES = 4;  // of x, of two blocks at most: a copy takes about 1 us
constexpr int MANY_TILE = 128, MANY_STRIPS = MANY_TILE / STRIP;

// Blocks of a stage, and columns of tensor memory: sums of two stages and their codes, a power of two.
__host__ __device__ constexpr int stage_blocks(int group) { return group == 32 ? 1 : 2; }
__host__ __device__ constexpr int many_tmem(int group, int nc) {
  return 2 * stage_blocks(group) * BLOCK / group * nc + 64 * stage_blocks(group) <= 256 ? 256 : 512;
}
// Shared memory: the stages of x, or the sums of a tile as [column][output] with a float between columns.  A cluster asks for more than that,
// in proportion to tensor memory: its CTAs wait for one another, so none may be resident whose tensor memory a CTA of another such
// cluster holds, of a launch on another stream, that waits in the same way.  Two of 76 KB fit an SM, or one of 152.  CTAs that share
// nothing end by themselves, and the next launch's may come in beside them (64 rows x 14,336 x 4096 in groups of 64: 30 us, else 37).
constexpr int MANY_SUM_PITCH = MANY_TILE + 1;
constexpr int many_smem(int nc) { return 1024 + std::max(X_STAGES * 2 * nc * 128, nc * MANY_SUM_PITCH * 4); }
constexpr int many_cluster_smem(int group, int nc) { return std::max(many_tmem(group, nc) == 256 ? 76 << 10 : 152 << 10, many_smem(nc)); }

__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
               "r"(r[15])
               : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[N]) {
  static_assert(N % 16 == 0, "columns");
#pragma unroll
  for (int i = 0; i < N; i += 16)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7]), "=r"(r[i + 8]), "=r"(r[i + 9]),
          "=r"(r[i + 10]), "=r"(r[i + 11]), "=r"(r[i + 12]), "=r"(r[i + 13]), "=r"(r[i + 14]), "=r"(r[i + 15])
        : "r"(at + i));
}
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {  // r is not touched before
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void many_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
// D [+]= A (tensor memory, K-major) times B (shared memory, K-major).
template <bool ADD>
__device__ __forceinline__ void many_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
               "n"(ADD ? 1 : 0)
               : "memory");
}
// K-major rows of 128 bytes, groups of 8 rows 1024 bytes apart, 128-byte swizzle.
__device__ __forceinline__ uint64_t rows_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// One lane of the warp, the same every time.
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void workers_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * MANY_WARPS) : "memory"); }
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of the shared memory of the cluster's CTA `rank`, at this CTA's address.
__device__ __forceinline__ float peer_float(const float *p, int rank) {
  uint32_t at;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(tc::smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// Where an expert's rows lie as they are laid out, in groups of 8 columns of the product (times a.blocks, of 1024 bytes): pass p of it begins
// p * NC / 8 groups behind arranged_at(pos[e], e), and its blocks of 64 columns of x follow one another, each with the groups that the pass
// has rows for.  No two experts overlap: n rows take less than n * (NC / 8) / ROWS + 1 groups, and from pos[e] to pos[e] + n and the next expert
// there are more than n * (NC / 8) / ROWS of them.
template <int NC, int ROWS>
__host__ __device__ constexpr int64_t arranged_at(int64_t begin, int expert) { return begin * (NC / 8) / ROWS + expert; }
// Bytes of a block of 64 columns for `rows` rows of a pass.
template <int A_ROW>
__device__ __forceinline__ int block_bytes(int rows) { return (rows * A_ROW + 7) / 8 * 1024; }

// A thread half a row's block: 32 columns, of which lane c's operand has 8 c to 8 c + 7.  The columns of the product come in the order of the
// codes in tensor memory, pair p of lane c at 4 p + c, so that pair p of the four lanes makes 16 bytes.
template <typename X, int NC>
__global__ void __launch_bounds__(256) arrange_kernel(const __grid_constant__ ProductArgs a) {
  constexpr bool PARTS = std::is_same<X, float>::value;
  constexpr int A_ROW = PARTS ? 3 : 1, ROWS = NC / A_ROW, V = 16 / sizeof(X);
  pdl_wait();
  const int expert = blockIdx.y, columns = (int)a.columns;
  int64_t begin = 0, end = a.rows;
  if (a.pos != nullptr) {
    begin = min((int64_t)max(a.pos[expert], 0), a.rows);
    end = min((int64_t)a.pos[expert + 1], a.rows);
  }
  uint8_t *const passes = a.arranged + arranged_at<NC, ROWS>(begin, expert) * a.blocks * 1024;
  const int halves = 2 * a.blocks;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (end - begin) * halves; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / halves;
    const int half = (int)(i - row * halves), c0 = half * 32, r = (int)(row % ROWS);
    int64_t from = begin + row;
    if (a.fetch) from = a.crd[from] / a.k;
    const bool there = (uint64_t)from < (uint64_t)a.x_rows;
    const X *const x = static_cast<const X *>(a.x) + from * a.x_stride;
    alignas(16) X v[32];
    if (there && a.wide && c0 + 32 <= columns) {
#pragma unroll
      for (int k = 0; k < 32 / V; ++k) reinterpret_cast<uint4 *>(v)[k] = reinterpret_cast<const uint4 *>(x + c0)[k];
    } else {
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = there && c0 + k < columns ? x[c0 + k] : from_f32<X>(0.0f);
    }
    uint8_t *const block = passes + (row / ROWS) * a.blocks * (NC * 128) + (int64_t)(half / 2) * block_bytes<A_ROW>((int)min((int64_t)ROWS, end - begin - (row - r)));
#pragma unroll
    for (int p = 0; p < A_ROW; ++p) {
      uint32_t word[16];  // pair by pair
      if constexpr (!PARTS) {
#pragma unroll
        for (int k = 0; k < 16; ++k) word[k] = reinterpret_cast<const uint32_t *>(v)[k];
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) {  // 8 bits each: cut, not rounded, as the largest numbers would become infinite; what is not finite has one part
          uint32_t got[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float &left = v[2 * k + e];
            got[e] = left != left ? 0x7fc00000u : __float_as_uint(left) & 0xffff0000u;
            left = (got[e] & 0x7f800000u) == 0x7f800000u ? 0.0f : left - __uint_as_float(got[e]);
          }
          word[k] = __byte_perm(got[0], got[1], 0x7632);
        }
      }
      const int n = r * A_ROW + p;
#pragma unroll
      for (int pair = 0; pair < 4; ++pair)
        *reinterpret_cast<uint4 *>(block + n * 128 + ((half % 2 * 4 + pair) ^ (n & 7)) * 16) = make_uint4(word[pair], word[4 + pair], word[8 + pair], word[12 + pair]);
    }
  }
}

// What a lane of a converting warp has of a batch beside its codes: the zeros of rows r and r + 8 of its strip, and the scales of the output
// whose sums it adds, asked for a batch ahead.
template <int GROUPS, bool ZEROS>
struct Record {
  uint32_t zero[2] = {0x88888888u, 0x88888888u}, scale[GROUPS];  // 16-bit scales two in a word

  __device__ __forceinline__ void ask(const uint8_t *zeros, const uint8_t *at, int type) {
    if constexpr (ZEROS) {
      if constexpr (GROUPS == 8) zero[0] = reinterpret_cast<const uint32_t *>(zeros)[0], zero[1] = reinterpret_cast<const uint32_t *>(zeros)[1];
      else if constexpr (GROUPS == 4) zero[0] = reinterpret_cast<const uint32_t *>(zeros)[0];
      else zero[0] = reinterpret_cast<const uint16_t *>(zeros)[0];
    }
    if (type == LAPIS_F32) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) scale[g] = reinterpret_cast<const uint32_t *>(at)[g];
    } else {
#pragma unroll
      for (int g = 0; g < GROUPS / 2; ++g) scale[g] = reinterpret_cast<const uint32_t *>(at)[g];
    }
  }
  __device__ __forceinline__ void scales(float (&to)[GROUPS], int type) const {
    if (type == LAPIS_F32) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) to[g] = __uint_as_float(scale[g]);
    } else if (type == LAPIS_BF16) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) to[g] = __uint_as_float(g % 2 ? scale[g / 2] & 0xffff0000u : scale[g / 2] << 16);
    } else {
#pragma unroll
      for (int g = 0; g < GROUPS; g += 2) {
        const float2 s = __half22float2(*reinterpret_cast<const __half2 *>(&scale[g / 2]));
        to[g] = s.x, to[g + 1] = s.y;
      }
    }
  }
};

// NC: columns of the product of a pass over the weights.  The tensor core's work comes in stages of 128 columns of x (64 where groups are of
// 32).  A stage has half of the codes' room and of the sums' room in tensor memory, and one barrier says that its products are done and
// both are free again: what bounds the kernel are the hand-overs between converting and issuing warps, 280 cycles for a wait and 100 for a
// commit.  64 rows x 14,336 x 4096, gated, groups of 64: 30 us (1.1 TB/s, 250 TFLOP/s); with a commit for every block and group 38.  Two CTAs an SM have
// 96 registers a thread: with 64 columns in groups of 128 a thread spills 68 to 120 bytes, with 32 up to 100.
template <typename X, int GROUP, int NC, bool ZEROS>
__global__ void __launch_bounds__(MANY_THREADS, many_tmem(GROUP, NC) == 256 ? 2 : 1) int4_many_kernel(const __grid_constant__ ProductArgs a) {
  using T = typename std::conditional<std::is_same<X, float>::value, __nv_bfloat16, X>::type;
  constexpr int A_ROW = std::is_same<X, float>::value ? 3 : 1, ROWS = NC / A_ROW, GROUPS = BATCH / GROUP;
  constexpr int SB = stage_blocks(GROUP), SG = SB * BLOCK / GROUP, SUMS = 2 * SG * NC;  // blocks and groups of a stage, columns of sums in tensor memory
  constexpr int TMEM = many_tmem(GROUP, NC);
  constexpr uint32_t IDESC = (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(NC >> 3) << 17) | ((uint32_t)(MANY_TILE >> 4) << 24);
  extern __shared__ uint8_t many_shared[];
  __shared__ uint64_t ready[2], done[2], copied[X_STAGES];
  __shared__ uint32_t tmem_slot;
  uint8_t *const smem = many_shared + (1024 - (tc::smem_u32(many_shared) & 1023)) % 1024;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int shares = 1 << a.shares_log, my_share = blockIdx.x & (shares - 1), tile = blockIdx.x >> a.shares_log;
  const int outs = a.gated ? MANY_TILE / 2 : MANY_TILE, first_out = tile * outs, expert = blockIdx.y;
  X *const y = static_cast<X *>(a.y);
  pdl_wait();
  int64_t begin = 0, end = a.rows;
  if (a.pos != nullptr) {
    begin = min((int64_t)max(a.pos[expert], 0), a.rows);
    end = expert < a.experts ? min((int64_t)a.pos[expert + 1], a.rows) : a.rows;
    if (expert == a.experts || begin >= end) {  // rows of no expert (with lists the grid has one layer)
      pdl_release();
      const int n = min(outs, a.outputs - first_out);
      if (expert == a.experts && my_share == 0)
        for (int64_t r = begin; r < end; ++r)
          for (int i = threadIdx.x; i < n; i += MANY_THREADS) y[r * a.outputs + first_out + i] = from_f32<X>(0.0f);
      return;  // all CTAs of the cluster
    }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&ready[s], MANY_WARPS + 1);
      tc::mbar_init(&done[s], 1);
    }
    for (int s = 0; s < X_STAGES; ++s) tc::mbar_init(&copied[s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MANY_WARPS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "n"(TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  pdl_release();  // no CTA of the next kernel takes tensor memory that one of this kernel still waits for
  const uint32_t tmem = tmem_slot;
  // This CTA's batches of the tile's columns.
  const int per = (a.batches + shares - 1) >> a.shares_log, batch0 = min(my_share * per, a.batches), batches = min(per, a.batches - batch0);
  const int blocks = min(batches * (BATCH / BLOCK), a.blocks - batch0 * (BATCH / BLOCK)), stages = (blocks + SB - 1) / SB;
  bool ok = true;
  uint32_t parity = 0, x_turn = 0;  // of the next wait for each half's barrier; stages of x so far, of all passes

  for (int64_t row0 = begin + (int64_t)blockIdx.z * ROWS; row0 < end; row0 += (int64_t)gridDim.z * ROWS) {  // every CTA has a pass at least
    const int rows = (int)min((int64_t)ROWS, end - row0), block_size = block_bytes<A_ROW>(rows);
    if (warp == MANY_WARPS + 1) {
      // Copies X_STAGES stages of x ahead, and says of each that it is there: what else is ready is said by the converting warps.
      if (lane == 0) {
        asm volatile("fence.proxy.async;" ::: "memory");  // blocks, and the sums where they come, were written by ordinary stores
        const uint8_t *const from = a.arranged + (arranged_at<NC, ROWS>(begin, expert) + (row0 - begin) / ROWS * (NC / 8)) * a.blocks * 1024 +
                                    (int64_t)batch0 * (BATCH / BLOCK) * block_size;
        const auto copy = [&](int i) {
          const uint32_t s = (x_turn + i) % X_STAGES, bytes = min(SB, blocks - i * SB) * block_size;
          tc::mbar_expect_tx(&copied[s], bytes);
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(smem) + s * SB * NC * 128),
                       "l"(from + (int64_t)i * SB * block_size), "r"(bytes), "r"(tc::smem_u32(&copied[s]))
                       : "memory");
        };
        const auto arrived = [&](int i) { return tc::mbar_wait(&copied[(x_turn + i) % X_STAGES], (x_turn + i) / X_STAGES & 1); };
        int asked = min(stages, X_STAGES), there = 0;
        for (int i = 0; i < asked; ++i) copy(i);
        for (int i = 0; i < stages + 2 && ok; ++i) {
          if (i >= 2 && i - 2 < stages) {  // what stage i - 2 had is free
            ok = tc::mbar_wait(&done[i & 1], parity >> (i & 1) & 1);
            parity ^= 1u << (i & 1);
            if (ok && asked < stages) copy(asked++);
          }
          if (ok && i < stages) {
            ok = arrived(there++);
            tc::mbar_arrive(&ready[i & 1]);
          }
        }
        while (there < asked) arrived(there++);  // a wait gave up: no copy comes behind the end of the CTA
        x_turn += stages;
      }
      __syncwarp();
    } else if (warp == MANY_WARPS) {
      // All lanes go through the stages, and one issues: what the products are given is then computed once for the warp, in uniform registers.
      // By a thread of its own a product took 100 cycles.
      const bool leader = elected();
      const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t x0 = rows_desc(__shfl_sync(0xffffffffu, tc::smem_u32(smem), 0));
      // A stage's second block lies right behind the first.  Columns of the product beyond the rows are whatever lies in the rest of the
      // stage: nobody looks at their sums.
      const uint32_t block_step = __shfl_sync(0xffffffffu, block_size / 16, 0);
      for (int i = 0; i < stages && ok; ++i) {
        const uint32_t s = i & 1;
        ok = __all_sync(0xffffffffu, tc::mbar_wait(&ready[s], parity >> s & 1));
        parity ^= 1u << s;
        fence_after();
        const uint64_t x = x0 + x_turn++ % X_STAGES * (SB * NC * 128 / 16);
        const uint32_t d = d0 + s * SG * NC, codes = d0 + SUMS + s * SB * 32;
        const int here = ok ? blocks - i * SB : 0;
        if (leader) {
#pragma unroll
          for (int b = 0; b < SB; ++b) {
            if (b >= here) break;
#pragma unroll
            for (int ks = 0; ks < BLOCK / 16; ++ks) {
              const int at = b * BLOCK + ks * 16;
              if (at % GROUP != 0) many_mma<true>(d + at / GROUP * NC, codes + b * 32 + ks * 8, x + b * block_step + ks * 2, IDESC);
              else many_mma<false>(d + at / GROUP * NC, codes + b * 32 + ks * 8, x + b * block_step + ks * 2, IDESC);
            }
          }
          if (here > 0) many_commit(&done[s]);
        }
        __syncwarp();
      }
    } else {
      // A warp converts the strip that lies in its half of its quarter of tensor memory, and adds half of the columns of that quarter.
      const int quarter = warp % 4, half = warp / 4;
      const auto strip_of = [&](int s) { return (int64_t)expert * a.strips + min(tile * MANY_STRIPS + s, a.strips - 1); };
      const uint4 *codes = reinterpret_cast<const uint4 *>(a.codes) + (strip_of(2 * quarter + half) * a.blocks + batch0 * (BATCH / BLOCK)) * 32 + lane;
      const uint8_t *zeros = a.records + (strip_of(2 * quarter + half) * a.batches + batch0) * a.record_bytes + a.zeros_at + lane / 4 * GROUPS;
      const int scale_bytes = a.scale_type == LAPIS_F32 ? 4 : 2;
      Record<GROUPS, ZEROS> record;
      const uint8_t *scales = a.records + (strip_of(2 * quarter + lane / 16) * a.batches + batch0) * a.record_bytes + (lane % 8 * 2 + lane % 16 / 8) * GROUPS * scale_bytes;
      const uint32_t a_at = tmem + SUMS + ((uint32_t)(32 * quarter + 16 * half) << 16);
      const uint32_t sum_at = tmem + half * (NC / 2) + ((uint32_t)(32 * quarter) << 16);
      uint4 code[BATCH / BLOCK];
      if (blocks > 0) record.ask(zeros, scales, a.scale_type);
#pragma unroll
      for (int b = 0; b < BATCH / BLOCK; ++b)
        if (b < blocks) code[b] = codes[b * 32];
      float2 sum[NC / 4] = {};
      float behind[2][SG];  // of the stage that each half has: its groups' scales, and how many groups it has (0: none)
      int behind_groups[2] = {0, 0};
      // Waits for the products of the stage that has this half, and adds their sums.
      const auto free_half = [&](int s) {
        if (behind_groups[s] == 0) return;
        if (ok) ok = tc::mbar_wait(&done[s], parity >> s & 1);
        parity ^= 1u << s;
        __syncwarp();
        fence_after();
        constexpr int STEP = NC / 2 < 32 ? NC / 2 : 32;
#pragma unroll
        for (int g = 0; g < SG; ++g) {
          if (g >= behind_groups[s]) break;
#pragma unroll
          for (int c = 0; c < NC / 2; c += STEP) {
            uint32_t got[STEP];
            tmem_load(sum_at + (s * SG + g) * NC + c, got);
            tmem_wait(got);
#pragma unroll
            for (int i = 0; i < STEP; i += 2)
              sum[(c + i) / 2] = fma2(make_float2(behind[s][g], behind[s][g]), make_float2(__uint_as_float(got[i]), __uint_as_float(got[i + 1])), sum[(c + i) / 2]);
          }
        }
        behind_groups[s] = 0;
      };
      for (int i0 = 0; i0 < blocks; i0 += BATCH / BLOCK) {
        float scale[GROUPS];
        record.scales(scale, a.scale_type);
        const uint32_t zero[2] = {record.zero[0], ZEROS && GROUPS < 8 ? record.zero[0] >> 4 * GROUPS : record.zero[1]};
        zeros += a.record_bytes;
        scales += a.record_bytes;
        if (i0 + BATCH / BLOCK < blocks) record.ask(zeros, scales, a.scale_type);
        codes += BATCH / BLOCK * 32;
#pragma unroll
        for (int st = 0; st < BATCH / BLOCK / SB; ++st) {
          if (i0 + st * SB >= blocks) break;
          constexpr int EVEN = BATCH / BLOCK / SB;  // an even number of stages a batch: a stage's half is known here
          static_assert(EVEN % 2 == 0, "halves");
          const int s = st & 1;
#pragma unroll
          for (int u = 0; u < SB; ++u) {
            const int b = st * SB + u;
            if (i0 + b >= blocks) break;
            uint32_t number[16];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              Zero<T> z0, z1;
              z0.set(ZEROS ? zero[0] >> 4 * ((b * 64 + h * 32) / GROUP) & 15 : 8);
              z1.set(ZEROS ? zero[1] >> 4 * ((b * 64 + h * 32) / GROUP) & 15 : 8);
              uint32_t p0[4], p1[4];
              pairs_of(p0, h ? code[b].y : code[b].x, z0);
              pairs_of(p1, h ? code[b].w : code[b].z, z1);
#pragma unroll
              for (int p = 0; p < 4; ++p) number[8 * h + 2 * p] = p0[p], number[8 * h + 2 * p + 1] = p1[p];
            }
            if (i0 + b + BATCH / BLOCK < blocks) code[b] = codes[b * 32];
            if (u == 0) free_half(s);  // the first block's numbers are there before it has to be
            tmem_store(a_at + (s * SB + u) * 32, number);
          }
#pragma unroll
          for (int g = 0; g < SG; ++g) behind[s][g] = scale[st * SG + g];
          behind_groups[s] = (min(SB, blocks - i0 - st * SB) * BLOCK + GROUP - 1) / GROUP;
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&ready[s]);
        }
      }
      if (stages % 2 == 1) free_half(1);
      free_half(0);
      if (stages % 2 == 0) free_half(1);
      // Every product has been waited for: the blocks' memory takes the sums.
      workers_barrier();
      float *const sums = reinterpret_cast<float *>(smem);
#pragma unroll
      for (int c = 0; c < NC / 4; ++c) {
        sums[(half * (NC / 2) + 2 * c) * MANY_SUM_PITCH + 32 * quarter + lane] = sum[c].x;
        sums[(half * (NC / 2) + 2 * c + 1) * MANY_SUM_PITCH + 32 * quarter + lane] = sum[c].y;
      }
    }
    if (shares > 1) cluster_barrier();
    else __syncthreads();
    // A share's part of the result: outputs from every CTA's sums, in the order of the shares.
    if (warp < MANY_WARPS) {
      const float *const sums = reinterpret_cast<const float *>(smem);
      const auto total = [&](int r, int n) {
        float v = 0.0f;
#pragma unroll
        for (int p = A_ROW - 1; p >= 0; --p) {  // the small parts first
          const float *const at = sums + (r * A_ROW + p) * MANY_SUM_PITCH + n;
          if (shares == 1) v += *at;
          else
            for (int q = 0; q < shares; ++q) v += peer_float(at, q);
        }
        return v;
      };
      const int outs_log = a.gated ? 6 : 7;
      for (int i = threadIdx.x + my_share * 32 * MANY_WARPS; i < rows << outs_log; i += shares * 32 * MANY_WARPS) {
        const int n = i & (outs - 1), r = i >> outs_log;
        if (first_out + n >= a.outputs) continue;
        const int in = a.gated ? n / 8 * STRIP + n % 8 : n;
        float v = total(r, in);
        if (a.gated) v = v / (1.0f + expf(-v)) * total(r, in + 8);
        y[(row0 + r) * a.outputs + first_out + n] = from_f32<X>(v);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next pass's copies come where the sums are
    }
    if (shares > 1) cluster_barrier();  // the others have read this CTA's sums
    else __syncthreads();
  }
  if (!ok) atomicExch(a.error_flag, 9);
  fence_before();
  __syncthreads();
  if (warp == MANY_WARPS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
}

template <typename X, int GROUP, int NC>
static int launch_many_as(ProductArgs &a, int matrices, cudaStream_t st) {
  const int tiles = (a.strips + MANY_STRIPS - 1) / MANY_STRIPS;
  // As many CTAs to a tile as keep all of them resident, two an SM where tensor memory has room for two.  Measured (with a slower issuing
  // thread): 14,336 x 4096 (112 tiles), 64 rows, groups of 128 33.7 us with one CTA a tile, 31.0 with two, 35.9 with four; 4096 x 4096 (32
  // tiles), 32 rows 28.7, 19.6 with two, 13.9 with four, 14.1 with eight.
  const int64_t slots = (int64_t)sm_count() * (512 / many_tmem(GROUP, NC));
  // Passes of one matrix come before that: they need no join (126 rows of 32 bits x 256 x 1536, groups of 32: six passes one after the other 60 us, at once 16).
  constexpr int ROWS = NC / (std::is_same<X, float>::value ? 3 : 1);
  const int64_t passes = a.pos != nullptr ? 1 : std::max<int64_t>(1, std::min({(a.rows + ROWS - 1) / ROWS, slots / tiles, (int64_t)65535}));
  a.shares_log = 0;
  while (a.shares_log < 3 && (2 << a.shares_log) <= a.batches && (tiles * passes << (a.shares_log + 1)) * a.experts <= slots) ++a.shares_log;
  // All passes of all experts (arranged_at): the rows, up to 8 columns of the product more for each expert.
  CallBuf arranged;
  LAPIS_TRY(scratch(&arranged, (size_t)arranged_at<NC, ROWS>(a.rows, a.experts) * a.blocks * 1024, st));
  a.arranged = static_cast<uint8_t *>(arranged.p);
  const int64_t each = (a.rows + a.experts - 1) / a.experts * 2 * a.blocks;
  LAPIS_CUDA_TRY(launch_pdl(arrange_kernel<X, NC>, dim3((unsigned)std::min<int64_t>(4 * sm_count(), (each + 255) / 256), a.experts), 256, 0, st, a));
  const auto kernel = a.zeros_at ? int4_many_kernel<X, GROUP, NC, true> : int4_many_kernel<X, GROUP, NC, false>;
  LAPIS_TRY(a.zeros_at ? (allow_smem<int4_many_kernel<X, GROUP, NC, true>>(many_cluster_smem(GROUP, NC))) : (allow_smem<int4_many_kernel<X, GROUP, NC, false>>(many_cluster_smem(GROUP, NC))));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles << a.shares_log, matrices, (unsigned)passes);
  cfg.blockDim = dim3(MANY_THREADS);
  cfg.dynamicSmemBytes = a.shares_log > 0 ? many_cluster_smem(GROUP, NC) : many_smem(NC);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1 << a.shares_log;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.shares_log > 0 ? 2 : 1;
  LAPIS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, (const ProductArgs)a));
  return LAPIS_OK;
}
template <typename X, int GROUP>
static int launch_many_of(ProductArgs &a, int matrices, int64_t expected, cudaStream_t st) {
  const int64_t columns = expected * (std::is_same<X, float>::value ? 3 : 1);
  if (columns <= 32) return launch_many_as<X, GROUP, 32>(a, matrices, st);
  if constexpr (GROUP == 128)
    if (columns > 64) return launch_many_as<X, GROUP, 128>(a, matrices, st);
  return launch_many_as<X, GROUP, 64>(a, matrices, st);
}
template <typename X>
static int launch_many_of(ProductArgs &a, int group, int matrices, int64_t expected, cudaStream_t st) {
  switch (group) {
    case 32: return launch_many_of<X, 32>(a, matrices, expected, st);
    case 64: return launch_many_of<X, 64>(a, matrices, expected, st);
    default: return launch_many_of<X, 128>(a, matrices, expected, st);
  }
}
int launch_many(int type, ProductArgs &a, int group, int matrices, int64_t expected, cudaStream_t st) {
  int dev = 0;
  LAPIS_CUDA_TRY(cudaGetDevice(&dev));
  a.error_flag = bgemm_error_flag(dev);
  if (a.error_flag == nullptr) return lapis_last_error();
  switch (type) {
    case LAPIS_F32: return launch_many_of<float>(a, group, matrices, expected, st);
    case LAPIS_F16: return launch_many_of<__half>(a, group, matrices, expected, st);
    default: return launch_many_of<__nv_bfloat16>(a, group, matrices, expected, st);
  }
}

}  // namespace lapis_b200

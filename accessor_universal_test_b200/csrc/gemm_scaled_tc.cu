// gemm_scaled_tc.cu -- the product of block-scaled 8-bit codes on the
// fifth-generation tensor cores.
//
// out = sum over the blocks b of 128 of k: (a_b . b_b^T) * a_scale[b, row] *
// b_scale[b, column / 128].  The scales are FP32, so they cannot go into the
// instruction: each block's product is made in tensor memory by itself (four
// instructions of 32 codes, the first without an addend) and added, times its
// scales, to the sums in the epilogue warps' registers, while the next blocks'
// products are made elsewhere in tensor memory.
//
// Roles: the first warps scale and add and, at the end of a tile, store; of the
// last warpgroup, one warp loads the operands' tiles, one brings the scales and
// two issue the products.
#include "gemm_scaled.cuh"

#include <cuda.h>

#include <algorithm>
#include <atomic>

namespace aut::scaled {
namespace {

constexpr int kMaxDevices = 16;
constexpr int kTileM = 128;
// Blocks of k whose scales are brought at a time, and how many such batches
// there is room for.
constexpr int kScaleBatch = 4, kScaleSlots = 4;
// Results that do not go out in 16-byte stores are turned, 16 rows of 16 words at
// a time, so that a warp writes whole lines of rows.
constexpr int kTurnPitch = 17;
// A load takes a few thousand cycles at most: a pair's pause for them once one
// of its waits has given up (about half a millisecond).
constexpr long long kPairDrainCycles = 1000000;

struct tile_params {
  gemm_params g;
  uint32_t idesc;
  uint32_t tiles_m, tiles_n;
  uint32_t parts;  // of k, for the split kernels
  uint32_t a_rows; // of a tile that are loaded: no more than a has, by eights
  uint32_t stages;      // of the ring, each the operands of a step
  uint32_t block_bytes; // of one block of k: a_rows of a, then b's rows
  bool wide_out; // out rows take 16-byte stores
  unsigned int *status;
  long long wait_cycles;
  uint64_t stall_tile;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count)
               : "memory");
}

__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)),
               "r"(bytes)
               : "memory");
}

__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ bool bar_try(uint32_t addr, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\t"
               "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
               "selp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done)
               : "r"(addr), "r"(parity)
               : "memory");
  return done != 0;
}

// Waits at most `limit` clock cycles, and no longer than until another role of
// the block has given up.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, long long limit,
                                         volatile int *gave_up) {
  const uint32_t addr = smem_addr(bar);
  if (bar_try(addr, parity)) return true;
  const long long start = clock64();
  for (uint32_t i = 1;; ++i) {
    if (bar_try(addr, parity)) return true;
    if ((i & 31u) == 0u && (*gave_up != 0 || clock64() - start > limit)) return false;
  }
}

// Address, in the cluster's shared memory, of what stands at `p` in its first block.
__device__ __forceinline__ uint32_t leader_addr(const void *p) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
  return a;
}

// Four floats of shared memory of the cluster's block `rank`.
__device__ __forceinline__ float4 cluster_load_four(const float *p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// Arrives on a barrier of the pair's first block.  Relaxed: what the arrival
// hands over is tensor memory that has been read (tcgen05.wait::ld and the
// fence before it order that); a release over the cluster waits for all of the
// thread's memory operations, about a thousand cycles.
__device__ __forceinline__ void bar_arrive_leader(uint64_t *bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                   leader_addr(bar))
               : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elected() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\t"
               "elect.sync _|p, 0xffffffff;\n\t"
               "selp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(one));
  return one != 0;
}

// The loads of both blocks of a pair are counted on its first block's barrier.
template <bool Pair>
__device__ __forceinline__ void load_tile(void *dst, const CUtensorMap *map, int column, int row,
                                          uint32_t bar) {
  if constexpr (Pair)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile"
                 ".mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst)),
                 "l"(map), "r"(column), "r"(row), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile"
                 ".mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst)),
                 "l"(map), "r"(column), "r"(row), "r"(bar)
                 : "memory");
}

// Shared-memory descriptor of a tile of rows of 128 bytes with the 128-byte
// swizzle (eight rows make an atom of 1024 bytes, the stride between atoms): the
// low word holds the address in units of 16 bytes, the high word is constant.
__device__ __forceinline__ uint32_t descriptor_low(uint32_t addr) {
  return ((addr & 0x3ffffu) >> 4) | 1u << 16;
}
constexpr uint32_t kDescriptorHigh = (1024 >> 4) | 1u << 14 | 2u << 29;

// One thread issues all products, so it must not compute between them: the
// descriptors differ by a constant in the low word, and whether the product is
// added is known at compile time.
template <bool Pair, bool Add>
__device__ __forceinline__ void mma_f8(uint32_t tmem, uint32_t a, uint32_t b, uint32_t idesc) {
#define AUT_MMA_F8(group)                                                                  \
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"                                 \
               "setp.ne.b32 p, %4, 0;\n\t"                                                 \
               "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"                          \
               "tcgen05.mma.cta_group::" group ".kind::f8f6f4 [%0], a, b, %3, p;\n\t}" ::   \
                   "r"(tmem),                                                              \
               "r"(a), "r"(b), "r"(idesc), "n"(Add ? 1 : 0), "r"(kDescriptorHigh)          \
               : "memory")
  if constexpr (Pair) AUT_MMA_F8("2");
  else AUT_MMA_F8("1");
#undef AUT_MMA_F8
}

// The product of a block of 128 codes: four instructions of 32.
template <bool Pair>
__device__ __forceinline__ void mma_block(uint32_t tmem, uint32_t a, uint32_t b, uint32_t idesc) {
  mma_f8<Pair, false>(tmem, a, b, idesc);
  mma_f8<Pair, true>(tmem, a + 2, b + 2, idesc);
  mma_f8<Pair, true>(tmem, a + 4, b + 4, idesc);
  mma_f8<Pair, true>(tmem, a + 6, b + 6, idesc);
}

// Arrives on the barrier, of both blocks where it is a pair, once the
// instructions issued so far are done.
template <bool Pair> __device__ __forceinline__ void mma_commit(uint64_t *bar) {
  if constexpr (Pair)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster"
                 ".multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::
                     "r"(smem_addr(bar))
                 : "memory");
}

template <bool Pair, int Columns> __device__ __forceinline__ void tmem_alloc(uint32_t *base) {
  if constexpr (Pair) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(base)),
                 "n"(Columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(base)),
                 "n"(Columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}

template <bool Pair, int Columns> __device__ __forceinline__ void tmem_free(uint32_t base) {
  if constexpr (Pair)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(Columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(Columns));
}

// 32 lanes x W columns of tensor memory; the values are there after
// tmem_wait on them.
#define AUT_R8(v, o)                                                                        \
  "=f"(v[o]), "=f"(v[o + 1]), "=f"(v[o + 2]), "=f"(v[o + 3]), "=f"(v[o + 4]), "=f"(v[o + 5]), \
      "=f"(v[o + 6]), "=f"(v[o + 7])
#define AUT_W8(v, o)                                                                        \
  "+f"(v[o]), "+f"(v[o + 1]), "+f"(v[o + 2]), "+f"(v[o + 3]), "+f"(v[o + 4]), "+f"(v[o + 5]), \
      "+f"(v[o + 6]), "+f"(v[o + 7])

__device__ __forceinline__ void tmem_load(float (&v)[16], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : AUT_R8(v, 0), AUT_R8(v, 8)
               : "r"(addr));
}
// Naming the values keeps their uses behind the wait.
__device__ __forceinline__ void tmem_wait(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : AUT_W8(v, 0), AUT_W8(v, 8)::"memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack_fp16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// Eight neighbouring results of row i from column j on.
__device__ __forceinline__ void store_eight(const tile_params &p, uint64_t i, uint64_t j,
                                            const float2 *v) {
  const gemm_params &g = p.g;
  if (p.wide_out && j + 8 <= g.n) {
    const uint64_t at = i * g.out_stride + j;
    if (g.type == AUT_TYPE_FP32) {
      float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(g.out) + at);
      o[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
      o[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    } else if (g.type == AUT_TYPE_BF16) {
      *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(g.out) + at) =
          make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y),
                     pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
    } else {
      *reinterpret_cast<uint4 *>(static_cast<__half *>(g.out) + at) =
          make_uint4(pack_fp16(v[0].x, v[0].y), pack_fp16(v[1].x, v[1].y),
                     pack_fp16(v[2].x, v[2].y), pack_fp16(v[3].x, v[3].y));
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (j + 2 * c < g.n) store_out(g, i, j + 2 * c, v[c].x);
    if (j + 2 * c + 1 < g.n) store_out(g, i, j + 2 * c + 1, v[c].y);
  }
}

// W words (of one or two results of Size bytes) of each of a warp's 32 rows from
// row i0 on, lane by lane a row, written by lines of rows.
template <int Size, int W>
__device__ __forceinline__ void store_turned(const tile_params &p, uint32_t *turn, int lane,
                                             uint64_t i0, uint64_t j0, const uint32_t (&words)[W]) {
  constexpr int kEach = 4 / Size; // results to a word
  const gemm_params &g = p.g;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    __syncwarp();
    if (lane / 16 == half) {
#pragma unroll
      for (int w = 0; w < W; ++w) turn[lane % 16 * kTurnPitch + w] = words[w];
    }
    __syncwarp();
#pragma unroll
    for (int at = 0; at < 16 * W; at += 32) {
      const int r = (at + lane) / W, w = (at + lane) % W;
      const uint64_t i = i0 + 16 * half + r, j = j0 + kEach * w;
      const uint32_t word = turn[r * kTurnPitch + w];
      if (i >= g.m || j >= g.n) continue;
      unsigned char *to = static_cast<unsigned char *>(g.out) + (i * g.out_stride + j) * Size;
      if (Size == 4 || (j + 1 < g.n && reinterpret_cast<uintptr_t>(to) % 4 == 0)) {
        *reinterpret_cast<uint32_t *>(to) = word;
      } else {
        reinterpret_cast<uint16_t *>(to)[0] = static_cast<uint16_t>(word);
        if (j + 1 < g.n) reinterpret_cast<uint16_t *>(to)[1] = static_cast<uint16_t>(word >> 16);
      }
    }
  }
}

// Four neighbouring results.
__device__ __forceinline__ void store_four(const tile_params &p, uint64_t i, uint64_t j,
                                           const float2 *v) {
  const gemm_params &g = p.g;
  if (p.wide_out && j + 4 <= g.n) {
    const uint64_t at = i * g.out_stride + j;
    if (g.type == AUT_TYPE_FP32)
      *reinterpret_cast<float4 *>(static_cast<float *>(g.out) + at) =
          make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    else if (g.type == AUT_TYPE_BF16)
      *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(g.out) + at) =
          make_uint2(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y));
    else
      *reinterpret_cast<uint2 *>(static_cast<__half *>(g.out) + at) =
          make_uint2(pack_fp16(v[0].x, v[0].y), pack_fp16(v[1].x, v[1].y));
    return;
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (j + 2 * c < g.n) store_out(g, i, j + 2 * c, v[c].x);
    if (j + 2 * c + 1 < g.n) store_out(g, i, j + 2 * c + 1, v[c].y);
  }
}

// Blocks of k to each of `parts` parts: whole steps, so that a step goes beyond
// its part only where k ends (and zeros follow), never into the next part's blocks.
__device__ __forceinline__ uint32_t blocks_to_a_part(uint32_t blocks, uint32_t parts,
                                                     uint32_t step) {
  return ((blocks + parts - 1) / parts + step - 1) / step * step;
}

// BN columns of out by 128 rows for each block; the two blocks of a pair share
// the columns, and each holds half of the rows of b that they stand for.
// Tensor memory holds the products of kDepth steps.
template <int BN, bool Pair> struct tile_shape {
  static constexpr int kABytes = kTileM * kBlock;
  static constexpr int kBRows = Pair ? BN / 2 : BN;
  static constexpr int kBBytes = kBRows * kBlock;
  static constexpr int kMostStages = 10;
  static constexpr int kRingBytes = (BN == 256 ? 192 : BN == 128 ? 200 : 204) * 1024;
  // Epilogue warps: four to a scheduler for the wide tiles, so that some read
  // tensor memory while others add (4096 x 8192 x 8192: 865 cycles a block of
  // k and tile where two to a scheduler took 962; the products alone, 513).  The
  // pair's 96 registers a thread leave 16 bytes to local memory, 52 where results
  // are turned.
  static constexpr int kEpilogueWarps = BN >= 128 ? 16 : 8;
  static constexpr int kParts = kEpilogueWarps / 4; // of the columns
  static constexpr int kLoadWarp = kEpilogueWarps, kScaleWarp = kEpilogueWarps + 1,
                       kProductWarp = kEpilogueWarps + 2; // and the next
  static constexpr int kThreads = 32 * (kEpilogueWarps + 4);
  // Blocks of k to a step.  A step costs every role 300 to 500 cycles of waits
  // and arrivals, more than a narrow tile's products of one block.
  static constexpr int kBatch = BN == 32 ? 4 : BN == 64 ? 2 : 1;
  static constexpr int kDepth = 512 / (kBatch * BN) < 4 ? 512 / (kBatch * BN) : 4;
  static constexpr int kSides = BN == 256 ? 2 : 1; // column blocks of b's scales
  static constexpr int kStepColumns = kBatch * BN;
  static constexpr int kTmemColumns = kDepth * kStepColumns;
  static constexpr int kTileRows = Pair ? 2 * kTileM : kTileM; // of out, by both blocks
};

// Tiles in bands of rows of tiles (2048 rows of a), column by column within a
// band: the tiles that run at one time share few rows and few columns.
template <int Rows>
__device__ __forceinline__ void tile_at(uint32_t tile, const tile_params &p, uint32_t &tm,
                                        uint32_t &tn) {
  constexpr uint32_t kBand = 2048 / Rows;
  const uint32_t per_band = kBand * p.tiles_n;
  const uint32_t band = tile / per_band, rest = tile % per_band;
  const uint32_t left = p.tiles_m - band * kBand;
  const uint32_t height = left < kBand ? left : kBand;
  tm = band * kBand + rest % height;
  tn = rest / height;
}

// Split: the blocks of a cluster share a tile's blocks of k, where there are
// fewer tiles than SMs; each has one tile, and their sums are joined over
// distributed shared memory in the order of the parts.  Turn: rows of out do not
// start on 16 bytes; a kernel of its own, whose registers the others do without
// (4096 x 8192 x 8192: 256 against 279 us).
template <int BN, bool Pair, bool Split, bool Turn>
__global__ void __launch_bounds__(tile_shape<BN, Pair>::kThreads, 1)
    tiles_kernel(const __grid_constant__ CUtensorMap map_a,
                 const __grid_constant__ CUtensorMap map_b, const tile_params p) {
  using shape = tile_shape<BN, Pair>;
  [[maybe_unused]] constexpr int kJoinPitch = BN + 4; // floats of a row of sums to be joined
  const int stages = static_cast<int>(p.stages);
  const uint32_t block_bytes = p.block_bytes, a_bytes = block_bytes - shape::kBBytes;
  const uint32_t stage_bytes = shape::kBatch * block_bytes;
  extern __shared__ unsigned char dynamic[];
  unsigned char *ring = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(dynamic) + 1023) & ~uintptr_t{1023});
  __shared__ __align__(8) uint64_t full[shape::kMostStages], empty[shape::kMostStages];
  __shared__ __align__(8) uint64_t made[shape::kDepth], taken[shape::kDepth];
  __shared__ __align__(8) uint64_t scales_in[kScaleSlots], scales_used[kScaleSlots];
  __shared__ __align__(8) uint64_t drained;
  // of both operands multiplied, for either side of the columns
  __shared__ float scales[shape::kSides][kScaleSlots][kScaleBatch][kTileM];
  __shared__ uint32_t turn[Turn ? shape::kEpilogueWarps : 1][16 * kTurnPitch];
  __shared__ uint32_t tmem_base;
  __shared__ int gave_up_word;
  volatile int *gave_up = &gave_up_word;

  // the same for all lanes, and known to be
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x / 32), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = Pair ? blockIdx.x % 2 : 0;
  const uint32_t shared_by = Pair ? 2 : Split ? p.parts : 1; // blocks to a worker
  const uint32_t worker = blockIdx.x / shared_by, workers = gridDim.x / shared_by;
  const uint32_t part = Split ? blockIdx.x % shared_by : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      bar_init(&full[s], 1);
      bar_init(&empty[s], 1);
    }
    for (int u = 0; u < shape::kDepth; ++u) {
      bar_init(&made[u], 1);
      bar_init(&taken[u], (Pair ? 2 : 1) * shape::kEpilogueWarps);
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      bar_init(&scales_in[s], 1);
      bar_init(&scales_used[s], shape::kEpilogueWarps);
    }
    bar_init(&drained, 2);
    gave_up_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == shape::kLoadWarp) {
    tmem_alloc<Pair, shape::kTmemColumns>(&tmem_base);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  if (Pair) cluster_sync(); // the barriers of both blocks are there
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
  }
  aut::dev::pdl_wait();
  aut::dev::pdl_release();

  const uint32_t tiles = p.tiles_m * p.tiles_n;
  // blocks of k: all, or this part's
  const uint32_t all_blocks = static_cast<uint32_t>((p.g.k + kBlock - 1) / kBlock);
  const uint32_t each =
      Split ? blocks_to_a_part(all_blocks, shared_by, shape::kBatch) : all_blocks;
  const uint32_t first_block = part * each;
  const uint32_t blocks = !Split ? all_blocks
                          : first_block >= all_blocks ? 0 : min(each, all_blocks - first_block);
  uint64_t loads = 0; // by the loading thread
  const uint64_t withheld = p.stall_tile / shape::kBatch; // of the loads, by the test hook
  if (warp >= shape::kEpilogueWarps) {
    if constexpr (shape::kEpilogueWarps == 16)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 64;"); // 5 x 96 = 4 x 104 + 64
    constexpr int kLoaders = shape::kBatch == 1 ? 1 : 2 * shape::kBatch;
    if (warp == shape::kLoadWarp && lane < kLoaders) {
      // One lane loads both operands of a step of one block; of several blocks,
      // lane l loads block l / 2, the even lanes of a, the odd of b.
      constexpr uint32_t kLanes = (1u << kLoaders) - 1;
      const bool of_a = lane % 2 == 0;
      const CUtensorMap *map = of_a ? &map_a : &map_b;
      const uint32_t offset = lane / 2 * block_bytes + (of_a ? 0 : a_bytes);
      const uint32_t expected =
          (Pair ? 2 : 1) * shape::kBatch * (p.a_rows * kBlock + shape::kBBytes);
      int s = 0;
      uint32_t parity = 1; // of the wait for a free stage; at first all are
      bool ok = true;
      for (uint32_t tile = worker; tile < tiles && ok; tile += workers) {
        uint32_t tm, tn;
        tile_at<shape::kTileRows>(tile, p, tm, tn);
        const int a_row = static_cast<int>(tm * shape::kTileRows + rank * kTileM);
        const int b_row = static_cast<int>(tn * BN + rank * shape::kBRows);
        for (uint32_t block = 0; block < blocks; block += shape::kBatch) {
          ok = bar_wait(&empty[s], parity, p.wait_cycles, gave_up);
          if constexpr (kLoaders > 1) ok = __all_sync(kLanes, ok);
          if (!ok) {
            *gave_up = 1;
            break;
          }
          if (rank == 0 && lane == 0) bar_expect(&full[s], expected);
          if constexpr (kLoaders > 1) __syncwarp(kLanes);
          const uint32_t bar = Pair ? leader_addr(&full[s]) : smem_addr(&full[s]);
          unsigned char *stage = ring + s * stage_bytes;
          const int column = static_cast<int>((first_block + block) * kBlock);
          if (loads != withheld) {
            if constexpr (kLoaders > 1) {
              load_tile<Pair>(stage + offset, map, column + lane / 2 * kBlock,
                              of_a ? a_row : b_row, bar);
            } else {
              load_tile<Pair>(stage, &map_a, column, a_row, bar);
              load_tile<Pair>(stage + a_bytes, &map_b, column, b_row, bar);
            }
          }
          ++loads;
          if (++s == stages) s = 0, parity ^= 1;
        }
      }
    }
    if (warp >= shape::kProductWarp && rank == 0) {
      // Two warps issue the products of every other step: what a warp spends
      // from step to step (two waits, four products a block and two arrivals,
      // about 500 cycles one after the other) is longer than the products of a narrow
      // tile, and no product adds to another's.  The stages of the ring and of
      // tensor memory are even in number, so that each belongs to one of the
      // warps: a wait tells a barrier's phase from the one before, not from the
      // one after, and only the warp that waited for a stage's last use knows
      // that it is over.  The whole warp goes through
      // the loop and one lane issues: in a branch of one lane the compiler
      // would move every operand of every product into the uniform registers
      // that the instruction takes.
      static_assert(shape::kDepth % 2 == 0 && shape::kMostStages % 2 == 0);
      const uint32_t a0 = descriptor_low(smem_addr(ring));
      int s = 0, depth = 0;
      uint32_t parity = 0, free_parity = 1; // tensor memory is all free at first
      int turn = warp - shape::kProductWarp; // 0: this warp's
      bool ok = true;
      for (uint32_t tile = worker; tile < tiles && ok; tile += workers) {
        for (uint32_t block = 0; block < blocks; block += shape::kBatch, turn ^= 1) {
          if (turn == 0) {
            ok = bar_wait(&full[s], parity, p.wait_cycles, gave_up) &&
                 bar_wait(&taken[depth], free_parity, p.wait_cycles, gave_up);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elected()) {
              uint32_t a = a0 + s * (stage_bytes >> 4), d = tmem + depth * shape::kStepColumns;
#pragma unroll
              for (int b = 0; b < shape::kBatch; ++b) {
                mma_block<Pair>(d, a, a + (a_bytes >> 4), p.idesc);
                a += block_bytes >> 4;
                d += BN;
              }
              mma_commit<Pair>(&made[depth]);
              mma_commit<Pair>(&empty[s]);
            }
            __syncwarp();
          }
          if (++s == stages) s = 0, parity ^= 1;
          if (++depth == shape::kDepth) depth = 0, free_parity ^= 1;
        }
      }
      if (!ok) *gave_up = 1;
    }
    if (warp == shape::kScaleWarp) {
      // a_scale * b_scale of 128 rows and either side of the columns, four rows
      // a lane, a batch of blocks at a time
      uint32_t batch = 0;
      bool ok = true;
      for (uint32_t tile = worker; tile < tiles && ok; tile += workers) {
        uint32_t tm, tn;
        tile_at<shape::kTileRows>(tile, p, tm, tn);
        const uint64_t i = uint64_t{tm} * shape::kTileRows + rank * kTileM + lane;
        const uint64_t j = uint64_t{tn} * BN;
        const float *sa = p.g.a_scales + first_block * p.g.a_scale_stride + i;
        const float *sb[shape::kSides];
#pragma unroll
        for (int side = 0; side < shape::kSides; ++side) {
          const uint64_t at = j + side * kBlock;
          sb[side] =
              p.g.b_scales + first_block * p.g.b_scale_stride + (at < p.g.n ? at / kBlock : 0);
        }
        for (uint32_t block = 0; block < blocks; block += kScaleBatch, ++batch) {
          float row[kScaleBatch][4], column[kScaleBatch][shape::kSides];
#pragma unroll
          for (int b = 0; b < kScaleBatch; ++b) {
            const bool has = block + b < blocks;
#pragma unroll
            for (int side = 0; side < shape::kSides; ++side) {
              column[b][side] = has ? __ldg(sb[side]) : 0.0f;
              sb[side] += p.g.b_scale_stride;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
              row[b][r] = has && i + 32 * r < p.g.m ? __ldg(sa + 32 * r) : 0.0f;
            sa += p.g.a_scale_stride;
          }
          const uint32_t slot = batch % kScaleSlots;
          ok = batch < kScaleSlots ||
               bar_wait(&scales_used[slot], (batch / kScaleSlots - 1) & 1u, p.wait_cycles, gave_up);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) {
            *gave_up = 1;
            break;
          }
#pragma unroll
          for (int b = 0; b < kScaleBatch; ++b)
#pragma unroll
            for (int side = 0; side < shape::kSides; ++side)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                scales[side][slot][b][32 * r + lane] = row[b][r] * column[b][side];
          __syncwarp();
          if (lane == 0) bar_arrive(&scales_in[slot]);
        }
      }
    }
  } else {
    if constexpr (shape::kEpilogueWarps == 16)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // Warps w, w + 4, ... take the tensor-memory lanes (rows of the tile)
    // 32 (w % 4) ..., each a stripe of the columns.
    constexpr int kColumns = BN / shape::kParts;
    constexpr int kChunk = kColumns < 16 ? kColumns : 16;
    constexpr int kChunks = kColumns / kChunk;
    const int row = warp % 4 * 32 + lane, stripe = warp / 4,
              side = stripe * shape::kSides / shape::kParts;
    const uint32_t tmem_own = tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16) + stripe * kColumns;
    uint32_t depth = 0, made_parity = 0, batch = 0;
    bool lost = false;
    for (uint32_t tile = worker; tile < tiles; tile += workers) {
      uint32_t tm, tn;
      tile_at<shape::kTileRows>(tile, p, tm, tn);
      float2 acc[kColumns / 2];
#pragma unroll
      for (int c = 0; c < kColumns / 2; ++c) acc[c] = make_float2(0.0f, 0.0f);
      for (uint32_t block = 0; block < blocks; block += shape::kBatch) {
        const uint32_t at = block % kScaleBatch, slot = batch % kScaleSlots;
        bool ok = at != 0 || bar_wait(&scales_in[slot], batch / kScaleSlots & 1u, p.wait_cycles,
                                      gave_up);
        float s[shape::kBatch];
#pragma unroll
        for (int b = 0; b < shape::kBatch; ++b) s[b] = scales[side][slot][at + b][row];
        ok = ok && bar_wait(&made[depth], made_parity, p.wait_cycles, gave_up);
        if (!__all_sync(0xffffffffu, ok)) {
          lost = true;
          break;
        }
        if (at + shape::kBatch == kScaleBatch || block + shape::kBatch >= blocks) {
          __syncwarp(); // of all lanes' reads: a vote orders no memory
          if (lane == 0) bar_arrive(&scales_used[slot]);
          ++batch;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t from = tmem_own + depth * shape::kStepColumns;
#pragma unroll
        for (int c0 = 0; c0 < kChunks; ++c0) {
          float now[shape::kBatch][kChunk];
#pragma unroll
          for (int b = 0; b < shape::kBatch; ++b) tmem_load(now[b], from + b * BN + c0 * kChunk);
#pragma unroll
          for (int b = 0; b < shape::kBatch; ++b) tmem_wait(now[b]);
          if (c0 + 1 == kChunks) {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              if (Pair) bar_arrive_leader(&taken[depth]);
              else bar_arrive(&taken[depth]);
            }
          }
#pragma unroll
          for (int b = 0; b < shape::kBatch; ++b)
#pragma unroll
            for (int c = 0; c < kChunk / 2; ++c)
              acc[c0 * kChunk / 2 + c] = fma2(make_float2(now[b][2 * c], now[b][2 * c + 1]),
                                              make_float2(s[b], s[b]), acc[c0 * kChunk / 2 + c]);
        }
        if (++depth == shape::kDepth) depth = 0, made_parity ^= 1;
      }
      if (lost) {
        *gave_up = 1;
#pragma unroll
        for (int c = 0; c < kColumns / 2; ++c)
          acc[c] = make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
      }
      if constexpr (Split) {
        // all of this block's products are done: the ring is free for its sums (if
        // a wait has run out, they are written again once its loads have landed)
        float *sums = reinterpret_cast<float *>(ring) + row * kJoinPitch + stripe * kColumns;
#pragma unroll
        for (int c = 0; c < kColumns / 2; c += 2)
          *reinterpret_cast<float4 *>(sums + 2 * c) =
              make_float4(acc[c].x, acc[c].y, acc[c + 1].x, acc[c + 1].y);
        break;
      }
      const uint64_t i0 = uint64_t{tm} * shape::kTileRows + rank * kTileM + warp % 4 * 32;
      const uint64_t j0 = uint64_t{tn} * BN + stripe * kColumns;
      if constexpr (!Turn) {
        if (i0 + lane < p.g.m) {
#pragma unroll
          for (int c = 0; c < kColumns; c += 8) store_eight(p, i0 + lane, j0 + c, acc + c / 2);
        }
      } else if (p.g.type == AUT_TYPE_FP32) {
#pragma unroll
        for (int c = 0; c < kColumns; c += 16) {
          uint32_t words[16];
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            words[2 * w] = __float_as_uint(acc[c / 2 + w].x);
            words[2 * w + 1] = __float_as_uint(acc[c / 2 + w].y);
          }
          store_turned<4>(p, turn[warp], lane, i0, j0 + c, words);
        }
      } else {
        constexpr int kWords = kColumns < 32 ? 8 : 16;
#pragma unroll
        for (int c = 0; c < kColumns; c += 2 * kWords) {
          uint32_t words[kWords];
#pragma unroll
          for (int w = 0; w < kWords; ++w)
            words[w] = p.g.type == AUT_TYPE_BF16 ? pack_bf16(acc[c / 2 + w].x, acc[c / 2 + w].y)
                                                 : pack_fp16(acc[c / 2 + w].x, acc[c / 2 + w].y);
          store_turned<2>(p, turn[warp], lane, i0, j0 + c, words);
        }
      }
    }
  }
  __syncthreads();
  if (*gave_up != 0) {
    // Let what is under way end before its memory is given back: this block's
    // loads, which in a pair only the first block's barriers show, and the
    // products.
    int none = 0;
    if (warp == shape::kLoadWarp && lane == 0) {
      atomicOr(p.status, static_cast<unsigned int>(AUT_STATUS_WAIT_TIMEOUT));
      if (Pair) {
        const long long start = clock64();
        while (clock64() - start < kPairDrainCycles) {
        }
      } else {
        for (uint64_t l = loads > p.stages ? loads - p.stages : 0; l < loads; ++l)
          if (l != withheld)
            bar_wait(&full[l % p.stages], static_cast<uint32_t>(l / p.stages) & 1u, p.wait_cycles,
                     &none);
      }
    }
    // by the lane that issued them: a commit counts its own thread's products
    if (warp >= shape::kProductWarp && rank == 0 && elected()) {
      mma_commit<Pair>(&drained);
      bar_wait(&drained, 0, p.wait_cycles, &none);
    }
    __syncthreads();
    if constexpr (Split) {
      float *sums = reinterpret_cast<float *>(ring);
      for (int at = threadIdx.x; at < kTileM * kJoinPitch; at += shape::kThreads)
        sums[at] = __int_as_float(0x7fffffff);
    }
  }
  if constexpr (Split) {
    __syncwarp();
    cluster_sync();
    // Every block joins a share of the sums, a thread four columns of a row at a
    // time, so that a warp reads whole lines of the others' shared memory.
    uint32_t tm, tn;
    tile_at<shape::kTileRows>(worker, p, tm, tn);
    const uint64_t i0 = uint64_t{tm} * kTileM, j0 = uint64_t{tn} * BN;
    const uint32_t fours = static_cast<uint32_t>(min(uint64_t{kTileM}, p.g.m - i0)) * (BN / 4);
    const uint32_t share = (fours + shared_by - 1) / shared_by;
    const float *sums = reinterpret_cast<const float *>(ring);
    for (uint32_t at = part * share + threadIdx.x; at < min(fours, (part + 1) * share);
         at += shape::kThreads) {
      const uint32_t row = at / (BN / 4), column = at % (BN / 4) * 4;
      float2 v[2] = {};
      float4 u[8];
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q)
        if (q < shared_by) u[q] = cluster_load_four(sums + row * kJoinPitch + column, q);
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q)
        if (q < shared_by) {
          v[0] = add2(v[0], make_float2(u[q].x, u[q].y));
          v[1] = add2(v[1], make_float2(u[q].z, u[q].w));
        }
      store_four(p, i0 + row, j0 + column, v);
    }
  }
  // no block of a cluster leaves before the others are done with its barriers
  // and its sums
  if (Pair || Split) cluster_sync();
  if (warp == shape::kLoadWarp) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_free<Pair, shape::kTmemColumns>(tmem);
  }
}

// ---- host -----------------------------------------------------------------------

using encode_map_fn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                   const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                   const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

encode_map_fn encode_map() {
  static const encode_map_fn fn = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult found{};
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<encode_map_fn>(f);
  }();
  return fn;
}

// A row-major matrix of codes, read in boxes of box_rows x 128.
aut_status make_map(CUtensorMap *map, const uint8_t *codes, uint64_t rows, uint64_t columns,
                    uint64_t stride, int box_rows) {
  const encode_map_fn fn = encode_map();
  if (fn == nullptr) return aut::lib::fail(AUT_ERR_CUDA, "cuTensorMapEncodeTiled is missing");
  const cuuint64_t dims[2] = {columns, rows};
  const cuuint64_t strides[1] = {rows > 1 ? stride : (columns + 15) / 16 * 16};
  const cuuint32_t box[2] = {kBlock, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t steps[2] = {1, 1};
  const CUresult r =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dims, strides, box,
         steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return aut::lib::fail(AUT_ERR_CUDA, "cuTensorMapEncodeTiled: error " + std::to_string(r));
  return AUT_OK;
}

template <int BN, bool Pair, bool Split, bool Turn>
aut_status launch_kind(aut_workspace *ws, tile_params p, int a_code, int b_code,
                        cudaStream_t stream) {
  using shape = tile_shape<BN, Pair>;
  auto kernel = tiles_kernel<BN, Pair, Split, Turn>;
  CUtensorMap map_a, map_b;
  // rows of a tile beyond a's are not even filled with zeros: what the products
  // make of them is not stored
  p.a_rows = static_cast<uint32_t>(std::min<uint64_t>(kTileM, (p.g.m + 7) / 8 * 8));
  aut_status st = make_map(&map_a, p.g.a, p.g.m, p.g.k, p.g.a_stride, static_cast<int>(p.a_rows));
  if (st == AUT_OK) st = make_map(&map_b, p.g.b, p.g.n, p.g.k, p.g.b_stride, shape::kBRows);
  if (st != AUT_OK) return st;
  const uint64_t tiles_m = (p.g.m + shape::kTileRows - 1) / shape::kTileRows;
  const uint64_t tiles_n = (p.g.n + BN - 1) / BN;
  if (tiles_m * tiles_n > 0x7fffffffull)
    return aut::lib::fail(AUT_ERR_TOO_LARGE, "more than 2^31 - 1 tiles of the product");
  p.tiles_m = static_cast<uint32_t>(tiles_m);
  p.tiles_n = static_cast<uint32_t>(tiles_n);
  // FP32 sums, both operands with k contiguous, tiles of kTileRows x BN
  p.idesc = (1u << 4) | (static_cast<uint32_t>(a_code) << 7) |
            (static_cast<uint32_t>(b_code) << 10) | (static_cast<uint32_t>(BN / 8) << 17) |
            (static_cast<uint32_t>(shape::kTileRows / 16) << 24);
  // The products read 128 rows of a whatever the ring holds of them: the room
  // behind the last stage is there for that.
  p.block_bytes = (p.a_rows * kBlock + 1023) / 1024 * 1024 + shape::kBBytes;
  const uint32_t stage_bytes = shape::kBatch * p.block_bytes;
  const uint32_t behind =
      p.block_bytes < static_cast<uint32_t>(shape::kABytes) ? shape::kABytes - p.block_bytes : 0;
  // even: see where the products are issued
  p.stages =
      std::min<uint32_t>(shape::kMostStages, (shape::kRingBytes - behind) / stage_bytes) / 2 * 2;
  const uint32_t smem = p.stages * stage_bytes + behind + 1024;
  const unsigned cluster = Pair ? 2 : Split ? p.parts : 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(shape::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  // once per device and kernel: shared memory, and how many pairs run at a time
  static std::atomic<int> resident[kMaxDevices];
  int at_once = ws->device < kMaxDevices ? resident[ws->device].load() : 0;
  if (at_once == 0) {
    AUT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      shape::kRingBytes + 1024));
    at_once = ws->sm_count;
    if (Pair) {
      cfg.gridDim = dim3(static_cast<unsigned>(ws->sm_count / 2 * 2));
      cfg.attrs = attr + 1;
      cfg.numAttrs = 1;
      AUT_CUDA_TRY(cudaOccupancyMaxActiveClusters(&at_once, kernel, &cfg));
      cfg.attrs = attr;
      cfg.numAttrs = 2;
      if (at_once < 1) at_once = 1;
    }
    if (ws->device < kMaxDevices) resident[ws->device].store(at_once);
  }
  // a split tile has workers of its own
  const uint64_t workers =
      Split ? tiles_m * tiles_n : std::min<uint64_t>(tiles_m * tiles_n, static_cast<uint64_t>(at_once));
  cfg.gridDim = dim3(static_cast<unsigned>(workers * cluster));
  AUT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, p));
  return AUT_OK;
}

template <int BN, bool Pair>
aut_status launch_tiles(aut_workspace *ws, const tile_params &p, int a_code, int b_code,
                        cudaStream_t stream) {
  if constexpr (!Pair)
    if (p.parts > 1) return launch_kind<BN, Pair, true, false>(ws, p, a_code, b_code, stream);
  return p.wide_out ? launch_kind<BN, Pair, false, false>(ws, p, a_code, b_code, stream)
                    : launch_kind<BN, Pair, false, true>(ws, p, a_code, b_code, stream);
}

} // namespace

aut_status gemm_tiles(aut_workspace *ws, const gemm_params &g, int a_code, int b_code,
                      cudaStream_t stream) {
  tile_params p{};
  p.g = g;
  const uint64_t size = g.type == AUT_TYPE_FP32 ? 4 : 2;
  p.wide_out = reinterpret_cast<uintptr_t>(g.out) % 16 == 0 && g.out_stride * size % 16 == 0;
  p.status = ws->tickets + aut::lib::kMaxBatchPerLaunch;
  p.wait_cycles = ws->wait_cycles;
  p.stall_tile = ws->stall_tile;
  // The way is the one that takes the shortest time by what was measured: beside
  // a start of about 3 us, for every block of k that an SM goes through 0.14 to
  // 0.18 us with 32 columns (32 and 128 x 4096 x 4096: 7.1 and 8.9 us), 0.2 with
  // 64 (16 x 8192 x 8192: 16.4), 0.3 with 128 (256 x 8192 x 8192: 24.6), 0.54
  // for a pair on 256 x 256 (4096 x 8192 x 8192: 256, at 1.6 GHz), and to join S parts of k
  // 0.5 + 0.4 S us (64 x 1024 x 8192 with 64 columns, S = 1, 2, 4: 14.9, 10.3,
  // 7.5 us).  What a last step goes through beyond its blocks is not counted: it
  // loads nothing where k has ended, and with whole steps in the price 40 sizes of
  // 17 to 400 rows took 240 us in all for 235.
  const uint64_t blocks = (g.k + kBlock - 1) / kBlock;
  const uint64_t rows = (g.m + kTileM - 1) / kTileM;
  const uint64_t sms = static_cast<uint64_t>(ws->sm_count);
  const auto rounds = [](uint64_t work, uint64_t at_once) { return (work + at_once - 1) / at_once; };
  int columns = 256;
  double best = 0.54 * blocks * rounds((rows + 1) / 2 * ((g.n + 255) / 256), sms / 2);
  if (rows == 1) best *= 2; // half of the pair has nothing to do
  p.parts = 1;
  const struct {
    int columns;
    double block;
  } kinds[] = {{32, 0.12 + 0.0005 * std::min<uint64_t>(g.m, kTileM)}, {64, 0.2}, {128, 0.3}};
  for (const auto &kind : kinds) {
    const uint64_t tiles = rows * ((g.n + kind.columns - 1) / kind.columns);
    for (uint32_t parts = 1; parts <= 8; parts *= 2) {
      if (parts > 1 && (tiles * parts > sms || blocks < 2 * parts)) break;
      const double t = kind.block * rounds(blocks, parts) * rounds(tiles * parts, sms) +
                       (parts > 1 ? 0.5 + 0.4 * parts : 0);
      if (t < best) best = t, columns = kind.columns, p.parts = parts;
    }
  }
  switch (columns) {
  case 32: return launch_tiles<32, false>(ws, p, a_code, b_code, stream);
  case 64: return launch_tiles<64, false>(ws, p, a_code, b_code, stream);
  case 128: return launch_tiles<128, false>(ws, p, a_code, b_code, stream);
  default: return launch_tiles<256, true>(ws, p, a_code, b_code, stream);
  }
}

} // namespace aut::scaled

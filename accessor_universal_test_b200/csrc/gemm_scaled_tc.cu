// gemm_scaled_tc.cu -- the product of block-scaled 8-bit codes on the
// fifth-generation tensor cores.
//
// out = sum over the blocks b of 128 of k: (a_b . b_b^T) * a_scale[b, row] *
// b_scale[b, column / 128].  The scales are FP32, so they cannot go into the
// instruction: each block's product is made in tensor memory by itself (four
// instructions of 32 codes, the first without an addend) and added, times its
// scales, to the sums in the epilogue warps' registers, while the next block's
// product is made in the other half of tensor memory.
#include "gemm_scaled.cuh"

#include <cuda.h>

namespace aut::scaled {
namespace {

constexpr int kTileM = 128;
constexpr int kEpilogueWarps = 8;
constexpr int kTileThreads = 32 * (kEpilogueWarps + 2);

struct tile_params {
  gemm_params g;
  uint32_t idesc;
  uint32_t tiles_m, tiles_n;
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

__device__ __forceinline__ void load_tile(void *dst, const CUtensorMap *map, int column, int row,
                                          uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
               "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst)),
               "l"(map), "r"(column), "r"(row), "r"(smem_addr(bar))
               : "memory");
}

// Shared-memory descriptor of a tile of rows of 128 bytes with the 128-byte
// swizzle: eight rows make an atom of 1024 bytes, the stride between atoms.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (uint64_t{1} << 16) |
         (uint64_t{1024 >> 4} << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}

__device__ __forceinline__ void mma_f8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool add) {
  asm volatile("{\n\t.reg .pred p;\n\t"
               "setp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
               "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
               : "memory");
}

__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_addr(bar))
               : "memory");
}

// 32 lanes x W columns of tensor memory; the values are there after
// tmem_wait on them.
#define AUT_R8(v, o)                                                                        \
  "=f"(v[o]), "=f"(v[o + 1]), "=f"(v[o + 2]), "=f"(v[o + 3]), "=f"(v[o + 4]), "=f"(v[o + 5]), \
      "=f"(v[o + 6]), "=f"(v[o + 7])
#define AUT_W8(v, o)                                                                        \
  "+f"(v[o]), "+f"(v[o + 1]), "+f"(v[o + 2]), "+f"(v[o + 3]), "+f"(v[o + 4]), "+f"(v[o + 5]), \
      "+f"(v[o + 6]), "+f"(v[o + 7])

__device__ __forceinline__ void tmem_load(float (&v)[32], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
               "[%32];"
               : AUT_R8(v, 0), AUT_R8(v, 8), AUT_R8(v, 16), AUT_R8(v, 24)
               : "r"(addr));
}
__device__ __forceinline__ void tmem_load(float (&v)[16], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : AUT_R8(v, 0), AUT_R8(v, 8)
               : "r"(addr));
}
// Naming the values keeps their uses behind the wait.
__device__ __forceinline__ void tmem_wait(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : AUT_W8(v, 0), AUT_W8(v, 8), AUT_W8(v, 16), AUT_W8(v, 24)::"memory");
}
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
                                            const float *v) {
  const gemm_params &g = p.g;
  if (p.wide_out && j + 8 <= g.n) {
    const uint64_t at = i * g.out_stride + j;
    if (g.type == AUT_TYPE_FP32) {
      float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(g.out) + at);
      o[0] = make_float4(v[0], v[1], v[2], v[3]);
      o[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if (g.type == AUT_TYPE_BF16) {
      *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(g.out) + at) =
          make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                     pack_bf16(v[6], v[7]));
    } else {
      *reinterpret_cast<uint4 *>(static_cast<__half *>(g.out) + at) =
          make_uint4(pack_fp16(v[0], v[1]), pack_fp16(v[2], v[3]), pack_fp16(v[4], v[5]),
                     pack_fp16(v[6], v[7]));
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (j + c < g.n) store_out(g, i, j + c, v[c]);
}

template <int BN> struct tile_shape {
  static constexpr int kABytes = kTileM * kBlock;
  static constexpr int kBBytes = BN * kBlock;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 200 * 1024 / kStageBytes < 8 ? 200 * 1024 / kStageBytes : 8;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static constexpr int kTmemColumns = 2 * BN;
};

// Tiles in bands of 16 rows of tiles, column by column within a band: the
// tiles that run at one time share few rows and few columns.
__device__ __forceinline__ void tile_at(uint32_t tile, const tile_params &p, uint32_t &tm,
                                        uint32_t &tn) {
  constexpr uint32_t kBand = 16;
  const uint32_t per_band = kBand * p.tiles_n;
  const uint32_t band = tile / per_band, rest = tile % per_band;
  const uint32_t left = p.tiles_m - band * kBand;
  const uint32_t height = left < kBand ? left : kBand;
  tm = band * kBand + rest % height;
  tn = rest / height;
}

template <int BN>
__global__ void __launch_bounds__(kTileThreads, 1)
    tiles_kernel(const __grid_constant__ CUtensorMap map_a,
                 const __grid_constant__ CUtensorMap map_b, const tile_params p) {
  using shape = tile_shape<BN>;
  constexpr int kStages = shape::kStages;
  extern __shared__ unsigned char dynamic[];
  unsigned char *ring = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(dynamic) + 1023) & ~uintptr_t{1023});
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], made[2], taken[2], drained;
  __shared__ uint32_t tmem_base;
  __shared__ int gave_up_word;
  volatile int *gave_up = &gave_up_word;

  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      bar_init(&full[s], 1);
      bar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      bar_init(&made[s], 1);
      bar_init(&taken[s], kEpilogueWarps);
    }
    bar_init(&drained, 1);
    gave_up_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kEpilogueWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&tmem_base)),
                 "n"(shape::kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base;

  aut::dev::pdl_wait();
  aut::dev::pdl_release();

  const uint32_t tiles = p.tiles_m * p.tiles_n;
  const uint32_t blocks = static_cast<uint32_t>((p.g.k + kBlock - 1) / kBlock);
  uint64_t loads = 0; // by the loading thread
  if (warp == kEpilogueWarps) {
    if (lane == 0) {
      for (uint32_t tile = blockIdx.x; tile < tiles && *gave_up == 0; tile += gridDim.x) {
        uint32_t tm, tn;
        tile_at(tile, p, tm, tn);
        for (uint32_t block = 0; block < blocks; ++block) {
          const int s = static_cast<int>(loads % kStages);
          if (loads >= kStages &&
              !bar_wait(&empty[s], static_cast<uint32_t>(loads / kStages - 1) & 1u, p.wait_cycles,
                        gave_up)) {
            *gave_up = 1;
            break;
          }
          unsigned char *stage = ring + s * shape::kStageBytes;
          bar_expect(&full[s], shape::kStageBytes);
          if (loads != p.stall_tile) {
            load_tile(stage, &map_a, static_cast<int>(block * kBlock),
                      static_cast<int>(tm * kTileM), &full[s]);
            load_tile(stage + shape::kABytes, &map_b, static_cast<int>(block * kBlock),
                      static_cast<int>(tn * BN), &full[s]);
          }
          ++loads;
        }
      }
    }
  } else if (warp == kEpilogueWarps + 1) {
    if (lane == 0) {
      uint64_t step = 0;
      for (uint32_t tile = blockIdx.x; tile < tiles && *gave_up == 0; tile += gridDim.x) {
        for (uint32_t block = 0; block < blocks; ++block, ++step) {
          const int s = static_cast<int>(step % kStages), half = static_cast<int>(step & 1);
          if ((step >= 2 && !bar_wait(&taken[half], static_cast<uint32_t>(step / 2 - 1) & 1u,
                                      p.wait_cycles, gave_up)) ||
              !bar_wait(&full[s], static_cast<uint32_t>(step / kStages) & 1u, p.wait_cycles,
                        gave_up)) {
            *gave_up = 1;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t stage = smem_addr(ring + s * shape::kStageBytes);
#pragma unroll
          for (int i = 0; i < kBlock / 32; ++i)
            mma_f8(tmem + half * BN, tile_descriptor(stage + 32 * i),
                   tile_descriptor(stage + shape::kABytes + 32 * i), p.idesc, i > 0);
          mma_commit(&empty[s]);
          mma_commit(&made[half]);
        }
      }
    }
  } else {
    // Warps w and w + 4 take the tensor-memory lanes (rows of the tile)
    // 32 (w % 4) ..., each one half of the columns.
    constexpr int kColumns = BN / 2;
    constexpr int kChunk = BN == 256 || BN == 32 ? 16 : 32; // 256: registers
    const int row = warp % 4 * 32 + lane, side = warp / 4;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    uint64_t step = 0;
    bool lost = false;
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      uint32_t tm, tn;
      tile_at(tile, p, tm, tn);
      const uint64_t i = uint64_t{tm} * kTileM + row;
      const uint64_t j0 = uint64_t{tn} * BN + side * kColumns;
      const bool has_row = i < p.g.m;
      const float *sa = p.g.a_scales + i;
      const float *sb = p.g.b_scales + (j0 < p.g.n ? j0 : 0) / kBlock;
      float acc[kColumns];
#pragma unroll
      for (int c = 0; c < kColumns; ++c) acc[c] = 0.0f;
      for (uint32_t block = 0; block < blocks && !lost; ++block, ++step) {
        const float s = (has_row ? __ldg(sa + block * p.g.a_scale_stride) : 0.0f) *
                        __ldg(sb + block * p.g.b_scale_stride);
        const int half = static_cast<int>(step & 1);
        const bool ok =
            bar_wait(&made[half], static_cast<uint32_t>(step / 2) & 1u, p.wait_cycles, gave_up);
        if (!__all_sync(0xffffffffu, ok)) {
          lost = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int c0 = 0; c0 < kColumns; c0 += kChunk) {
          float v[kChunk];
          __syncwarp();
          tmem_load(v, tmem + lanes + half * BN + side * kColumns + c0);
          tmem_wait(v);
          if (c0 + kChunk == kColumns) {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&taken[half]);
          }
#pragma unroll
          for (int c = 0; c < kChunk; ++c) acc[c0 + c] = fmaf(v[c], s, acc[c0 + c]);
        }
      }
      if (lost) {
        *gave_up = 1;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) acc[c] = __int_as_float(0x7fffffff);
      }
      if (has_row) {
#pragma unroll
        for (int c = 0; c < kColumns; c += 8) store_eight(p, i, j0 + c, acc + c);
      }
    }
  }
  __syncthreads();
  if (*gave_up != 0) {
    // Let what is under way end before its memory is given back.
    if (warp == kEpilogueWarps && lane == 0) {
      atomicOr(p.status, static_cast<unsigned int>(AUT_STATUS_WAIT_TIMEOUT));
      const uint64_t first = loads > kStages ? loads - kStages : 0;
      int none = 0;
      for (uint64_t l = first; l < loads; ++l)
        if (l != p.stall_tile)
          bar_wait(&full[l % kStages], static_cast<uint32_t>(l / kStages) & 1u, p.wait_cycles,
                   &none);
    }
    if (warp == kEpilogueWarps + 1 && lane == 0) {
      int none = 0;
      mma_commit(&drained);
      bar_wait(&drained, 0, p.wait_cycles, &none);
    }
    __syncthreads();
  }
  if (warp == kEpilogueWarps + 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "n"(shape::kTmemColumns));
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

template <int BN>
aut_status launch_tiles(aut_workspace *ws, tile_params p, int a_code, int b_code,
                        cudaStream_t stream) {
  using shape = tile_shape<BN>;
  CUtensorMap map_a, map_b;
  aut_status st = make_map(&map_a, p.g.a, p.g.m, p.g.k, p.g.a_stride, kTileM);
  if (st == AUT_OK) st = make_map(&map_b, p.g.b, p.g.n, p.g.k, p.g.b_stride, BN);
  if (st != AUT_OK) return st;
  p.tiles_m = static_cast<uint32_t>((p.g.m + kTileM - 1) / kTileM);
  p.tiles_n = static_cast<uint32_t>((p.g.n + BN - 1) / BN);
  // FP32 sums, both operands with k contiguous, tiles of 128 x BN
  p.idesc = (1u << 4) | (static_cast<uint32_t>(a_code) << 7) |
            (static_cast<uint32_t>(b_code) << 10) | (static_cast<uint32_t>(BN / 8) << 17) |
            (static_cast<uint32_t>(kTileM / 16) << 24);
  const uint64_t tiles = uint64_t{p.tiles_m} * p.tiles_n;
  if (tiles > 0x7fffffffull)
    return aut::lib::fail(AUT_ERR_TOO_LARGE, "more than 2^31 - 1 tiles of the product");
  AUT_CUDA_TRY(cudaFuncSetAttribute(tiles_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    shape::kSmem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(
      tiles < static_cast<uint64_t>(ws->sm_count) ? tiles : ws->sm_count));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = shape::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  AUT_CUDA_TRY(cudaLaunchKernelEx(&cfg, tiles_kernel<BN>, map_a, map_b, p));
  return AUT_OK;
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
  const uint64_t rows = (g.m + kTileM - 1) / kTileM;
  if (rows * ((g.n + 255) / 256) >= static_cast<uint64_t>(ws->sm_count))
    return launch_tiles<256>(ws, p, a_code, b_code, stream);
  if (rows * ((g.n + 127) / 128) >= static_cast<uint64_t>(ws->sm_count))
    return launch_tiles<128>(ws, p, a_code, b_code, stream);
  if (rows * ((g.n + 63) / 64) >= static_cast<uint64_t>(ws->sm_count))
    return launch_tiles<64>(ws, p, a_code, b_code, stream);
  return launch_tiles<32>(ws, p, a_code, b_code, stream);
}

} // namespace aut::scaled

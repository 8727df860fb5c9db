// gemm_scaled.cu -- aut_gemm_scaled: the product of two matrices of
// block-scaled 8-bit codes.
#include "gemm_scaled.cuh"

namespace aut::scaled {
namespace {

// Sixteen codes of a row from column c on; codes at or beyond column k read
// as zero (what a caller's row padding holds never enters the product).
__device__ __forceinline__ uint4 load_codes(const uint8_t *row, uint64_t c, uint64_t k) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t at = c + 4 * i + j;
      if (at < k) w[i] |= uint32_t{row[at]} << (8 * j);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// d += a (16 x 32) * b (32 x 8), FP32 sums.  LeftCode and RightCode name the
// formats of the instruction's two operands.
template <int LeftCode, int RightCode>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
#define AUT_MMA(L, R)                                                                        \
  asm("mma.sync.aligned.m16n8k32.row.col.f32." L "." R ".f32 "                               \
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                      \
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                       \
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
  if (LeftCode == AUT_FP8_E4M3 && RightCode == AUT_FP8_E4M3) AUT_MMA("e4m3", "e4m3");
  else if (LeftCode == AUT_FP8_E4M3) AUT_MMA("e4m3", "e5m2");
  else if (RightCode == AUT_FP8_E4M3) AUT_MMA("e5m2", "e4m3");
  else AUT_MMA("e5m2", "e5m2");
#undef AUT_MMA
}

// Both kernels below take both operands from memory straight into the matrix
// instruction's registers.  The sum over k does not depend on its order, so lane
// (g, t) of a warp takes contiguous codes of rows g and g + 8 of b and of row g
// of a as its part of two instructions for every 16, the same of both operands.

// Joins the sums of a thread block's eight warps, in warp order, and stores them.
template <int Rows, int Columns>
__device__ __forceinline__ void join_warps(const gemm_params &p, const float (&sums)[8][Rows][Columns],
                                           uint64_t m0, uint64_t n0) {
  for (int at = threadIdx.x; at < Rows * Columns; at += 256) {
    const int r = at % Rows, c = at / Rows;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][r][c];
    if (n0 + r < p.n && m0 + c < p.m) store_out(p, m0 + c, n0 + r, s);
  }
}

// ---- any alignment -------------------------------------------------------------------
// A thread block computes 16 rows of b against 8 rows of a; its warps share the
// blocks of k.  Codes are read byte by byte.
template <int ACode, int BCode>
__global__ void __launch_bounds__(256) rows_kernel(const gemm_params p) {
  __shared__ float sums[8][16][8];
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int g = lane >> 2, t = lane & 3;
  const uint64_t blocks = (p.k + kBlock - 1) / kBlock;
  const uint64_t groups = (p.n + 15) / 16;
  const uint64_t tasks = groups * ((p.m + 7) / 8);
  for (uint64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const uint64_t n0 = task % groups * 16, m0 = task / groups * 8;
    const uint8_t *b0 = p.b + (n0 + g) * p.b_stride, *b1 = b0 + 8 * p.b_stride;
    const uint8_t *a = p.a + (m0 + g) * p.a_stride;
    const bool has_b0 = n0 + g < p.n, has_b1 = n0 + g + 8 < p.n, has_a = m0 + g < p.m;
    const bool has_s0 = m0 + 2 * t < p.m, has_s1 = m0 + 2 * t + 1 < p.m;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint64_t block = warp; block < blocks; block += 8) {
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint64_t c = block * kBlock + 64 * half + 16 * t;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const uint4 u = has_b0 ? load_codes(b0, c, p.k) : zero;
        const uint4 v = has_b1 ? load_codes(b1, c, p.k) : zero;
        const uint4 w = has_a ? load_codes(a, c, p.k) : zero;
        mma<BCode, ACode>(d, u.x, v.x, u.y, v.y, w.x, w.y);
        mma<BCode, ACode>(d, u.z, v.z, u.w, v.w, w.z, w.w);
      }
      const float sb = p.b_scales[block * p.b_scale_stride + n0 / kBlock];
      const float *sa = p.a_scales + block * p.a_scale_stride + m0 + 2 * t;
      const float s0 = has_s0 ? sb * sa[0] : 0.0f, s1 = has_s1 ? sb * sa[1] : 0.0f;
      acc[0] = fmaf(d[0], s0, acc[0]);
      acc[1] = fmaf(d[1], s1, acc[1]);
      acc[2] = fmaf(d[2], s0, acc[2]);
      acc[3] = fmaf(d[3], s1, acc[3]);
    }
    sums[warp][g][2 * t] = acc[0];
    sums[warp][g][2 * t + 1] = acc[1];
    sums[warp][g + 8][2 * t] = acc[2];
    sums[warp][g + 8][2 * t + 1] = acc[3];
    __syncthreads();
    join_warps<16, 8>(p, sums, m0, n0);
    __syncthreads();
  }
}

// ---- few rows of a -----------------------------------------------------------------
// The product reads b once and computes little: what counts is how many bytes
// are under way.  A thread block computes 16 R rows of b against all rows of a
// (8 T); its eight warps share the blocks of k, kAhead at a time, all of whose
// loads are issued before the first product.  Measured (m x n x k, GB/s of
// codes): 1 x 4096 x 4096 with kAhead 1, 2, 3, 4: 3387, 3640, 2963, 2729;
// 8 x 8192 x 8192: 3763, 4364, 4063, 4004 (registers: fewer blocks to an SM);
// keeping the next kAhead blocks' loads under way behind each product: 4181.

// 32 codes of a row, in one load or two.  Measured: one load is faster where b is
// small (1 x 4096 x 4096: 4.1 against 4.7 us), two where it is large (8 x 8192 x
// 8192: 15.0 against 16.1 us).
template <bool Wide>
__device__ __forceinline__ void stream_load(const uint8_t *p, uint4 &v, uint4 &w) {
  if constexpr (Wide) {
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v8.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w), "=r"(w.x), "=r"(w.y), "=r"(w.z),
                   "=r"(w.w)
                 : "l"(p));
  } else {
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "l"(p + 16));
  }
}

template <int ACode, int BCode, int R, int T, bool Wide>
__global__ void __launch_bounds__(256, 2) stream_kernel(const gemm_params p) {
  constexpr int kAhead = T == 1 ? 2 : 1;
  __shared__ float sums[8][16 * R][8 * T];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int g = lane >> 2, t = lane & 3;
  const uint64_t n0 = uint64_t{blockIdx.x} * (16 * R);
  // A hint for the second-level cache, which is coherent, so it may come before
  // the kernels before this one have ended (1 x 4096 x 4096: 6.1 -> 4.6 us with
  // launches one behind the other): each lane's line of its row pairs' blocks
  // warp, warp + 8, + 16 and + 24.
  const uint64_t ahead = (uint64_t{static_cast<uint32_t>(warp)} + 8 * t) * kBlock;
  if (ahead < p.k)
#pragma unroll
    for (int r = 0; r < 2 * R; ++r)
      if (n0 + 8 * r + g < p.n)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.b + (n0 + 8 * r + g) * p.b_stride + ahead));
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const uint32_t blocks = static_cast<uint32_t>((p.k + kBlock - 1) / kBlock);
  const uint32_t whole = static_cast<uint32_t>(p.k / kBlock);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint8_t *b[R][2], *a[T]; // lane (g, t): the codes from 32 t of a block
  bool has_b[R][2], has_a[T];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint64_t row = n0 + 16 * r + 8 * h + g;
      has_b[r][h] = row < p.n;
      b[r][h] = p.b + (has_b[r][h] ? row : 0) * p.b_stride + 32 * t;
    }
#pragma unroll
  for (int i = 0; i < T; ++i) {
    const uint64_t row = 8 * i + g;
    has_a[i] = row < p.m;
    a[i] = p.a + (has_a[i] ? row : 0) * p.a_stride + 32 * t;
  }
  float acc[R][T][4] = {};
  for (uint32_t first = warp; first < blocks; first += 8 * kAhead) {
    uint4 u[kAhead][R][2][2], w[kAhead][T][2];
    float s[kAhead][T][2], column[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint32_t block = first + 8 * i;
      const uint64_t c = uint64_t{block} * kBlock;
      const bool in = block < whole;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (half == 0) { // both halves at once
              u[i][r][h][0] = u[i][r][h][1] = zero;
              if (in && has_b[r][h]) stream_load<Wide>(b[r][h] + c, u[i][r][h][0], u[i][r][h][1]);
            }
#pragma unroll
        for (int x = 0; x < T; ++x)
          w[i][x][half] = in && has_a[x]
                              ? __ldg(reinterpret_cast<const uint4 *>(a[x] + c + 16 * half))
                              : zero;
      }
      column[i] =
          block < blocks ? __ldg(p.b_scales + n0 / kBlock + block * p.b_scale_stride) : 0.0f;
#pragma unroll
      for (int x = 0; x < T; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          s[i][x][e] = block < blocks && 8 * x + 2 * t + e < p.m
                           ? __ldg(p.a_scales + block * p.a_scale_stride + 8 * x + 2 * t + e)
                           : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint32_t block = first + 8 * i;
      if (block == whole && whole < blocks) { // the last block, cut short by k
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint64_t c = uint64_t{block} * kBlock + 32 * t + 16 * half;
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (has_b[r][h]) u[i][r][h][half] = load_codes(b[r][h] - 32 * t, c, p.k);
#pragma unroll
          for (int x = 0; x < T; ++x)
            if (has_a[x]) w[i][x][half] = load_codes(a[x] - 32 * t, c, p.k);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int x = 0; x < T; ++x) {
          float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4 lo = u[i][r][0][half], hi = u[i][r][1][half], v = w[i][x][half];
            mma<BCode, ACode>(d, lo.x, hi.x, lo.y, hi.y, v.x, v.y);
            mma<BCode, ACode>(d, lo.z, hi.z, lo.w, hi.w, v.z, v.w);
          }
          const float s0 = s[i][x][0] * column[i], s1 = s[i][x][1] * column[i];
          acc[r][x][0] = fmaf(d[0], s0, acc[r][x][0]);
          acc[r][x][1] = fmaf(d[1], s1, acc[r][x][1]);
          acc[r][x][2] = fmaf(d[2], s0, acc[r][x][2]);
          acc[r][x][3] = fmaf(d[3], s1, acc[r][x][3]);
        }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int x = 0; x < T; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sums[warp][16 * r + 8 * (e / 2) + g][8 * x + 2 * t + e % 2] = acc[r][x][e];
  __syncthreads();
  join_warps<16 * R, 8 * T>(p, sums, 0, n0);
}

template <class Params>
aut_status launch(void (*kernel)(Params), uint64_t grid, int max_grid, int threads,
                  const Params &p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid < static_cast<uint64_t>(max_grid) ? grid : max_grid));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  AUT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return AUT_OK;
}

template <int ACode, int BCode, bool Wide>
aut_status gemm_few(aut_workspace *ws, const gemm_params &p, cudaStream_t stream) {
  if (p.m <= 8)
    return launch(stream_kernel<ACode, BCode, 1, 1, Wide>, (p.n + 15) / 16, 0x7fffffff, 256, p,
                  stream);
  // 32 rows of b to a block where that still gives every SM one
  if ((p.n + 31) / 32 >= static_cast<uint64_t>(ws->sm_count))
    return launch(stream_kernel<ACode, BCode, 2, 2, Wide>, (p.n + 31) / 32, 0x7fffffff, 256, p,
                  stream);
  return launch(stream_kernel<ACode, BCode, 1, 2, Wide>, (p.n + 15) / 16, 0x7fffffff, 256, p,
                stream);
}

template <int ACode, int BCode>
aut_status gemm_typed(aut_workspace *ws, const gemm_params &p, cudaStream_t stream) {
  if (!aligned_operands(p, 16) || p.k == 0)
    return launch(rows_kernel<ACode, BCode>, (p.n + 15) / 16 * ((p.m + 7) / 8),
                  64 * ws->max_blocks, 256, p, stream);
  if (p.m > 16) return gemm_tiles(ws, p, ACode, BCode, stream);
  // Measured: up to 8 rows streaming is faster than tiles (8 x 8192 x 8192: 15.0
  // against 16.4 us, 1 x 4096 x 4096: 4.1 against 6.8); up to 16 it is
  // where b is small (16 x 4096 x 4096: 6.1 against 7.1 us; 8192 x 8192: 19.5
  // against 16.4).
  if (p.m > 8 && p.n * p.k >= uint64_t{1} << 25) return gemm_tiles(ws, p, ACode, BCode, stream);
  return aligned_operands(p, 32) && p.n * p.k < uint64_t{1} << 25
             ? gemm_few<ACode, BCode, true>(ws, p, stream)
             : gemm_few<ACode, BCode, false>(ws, p, stream);
}

} // namespace
} // namespace aut::scaled

namespace aut::lib {
using namespace aut::scaled;

aut_status gemm_scaled_launch(aut_workspace *ws, int32_t a_code, int32_t b_code, int32_t type,
                              const void *a, uint64_t a_stride, const float *a_scales,
                              uint64_t a_scale_stride, const void *b, uint64_t b_stride,
                              const float *b_scales, uint64_t b_scale_stride, uint64_t m,
                              uint64_t n, uint64_t k, void *out, uint64_t out_stride,
                              cudaStream_t stream) {
  gemm_params p{};
  p.a = static_cast<const uint8_t *>(a);
  p.b = static_cast<const uint8_t *>(b);
  p.a_scales = a_scales;
  p.b_scales = b_scales;
  p.out = out;
  p.a_stride = a_stride;
  p.b_stride = b_stride;
  p.a_scale_stride = a_scale_stride;
  p.b_scale_stride = b_scale_stride;
  p.out_stride = out_stride;
  p.m = m;
  p.n = n;
  p.k = k;
  p.type = type;
  if (a_code == AUT_FP8_E4M3)
    return b_code == AUT_FP8_E4M3 ? gemm_typed<AUT_FP8_E4M3, AUT_FP8_E4M3>(ws, p, stream)
                                  : gemm_typed<AUT_FP8_E4M3, AUT_FP8_E5M2>(ws, p, stream);
  return b_code == AUT_FP8_E4M3 ? gemm_typed<AUT_FP8_E5M2, AUT_FP8_E4M3>(ws, p, stream)
                                : gemm_typed<AUT_FP8_E5M2, AUT_FP8_E5M2>(ws, p, stream);
}

} // namespace aut::lib

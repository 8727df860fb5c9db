// gemm_scaled.cu -- aut_gemm_scaled: the product of two matrices of
// block-scaled 8-bit codes.
#include "gemm_scaled.cuh"

namespace aut::scaled {
namespace {

// Sixteen codes of a row from column c on; codes at or beyond column k read
// as zero (what a caller's row padding holds never enters the product).
template <bool Aligned>
__device__ __forceinline__ uint4 load_codes(const uint8_t *row, uint64_t c, uint64_t k) {
  if (Aligned && c + 16 <= k) return __ldg(reinterpret_cast<const uint4 *>(row + c));
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

// ---- few rows of a: b streams through registers ---------------------------------
// A thread block computes 16 rows of b against 8 rows of a; its eight warps
// share the blocks of k and their sums are joined in warp order.  Both
// operands go from memory straight into the matrix instruction's registers:
// the sum over k does not depend on its order, so lane (g, t) takes the 16
// contiguous codes from 16 t (+ 64) of rows g and g + 8 as its part of two
// instructions, for both operands alike.
template <int ACode, int BCode, bool Aligned>
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
        const uint4 u = has_b0 ? load_codes<Aligned>(b0, c, p.k) : zero;
        const uint4 v = has_b1 ? load_codes<Aligned>(b1, c, p.k) : zero;
        const uint4 w = has_a ? load_codes<Aligned>(a, c, p.k) : zero;
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
    if (threadIdx.x < 128) {
      const int r = threadIdx.x & 15, c = threadIdx.x >> 4;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += sums[w][r][c];
      if (n0 + r < p.n && m0 + c < p.m) store_out(p, m0 + c, n0 + r, s);
    }
    __syncthreads();
  }
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

template <int ACode, int BCode>
aut_status gemm_typed(aut_workspace *ws, const gemm_params &p, cudaStream_t stream) {
  const bool aligned = aligned_operands(p);
  if (aligned && p.m > 16 && p.k > 0) return gemm_tiles(ws, p, ACode, BCode, stream);
  const uint64_t tasks = (p.n + 15) / 16 * ((p.m + 7) / 8);
  return launch(aligned ? rows_kernel<ACode, BCode, true> : rows_kernel<ACode, BCode, false>,
                tasks, 64 * ws->max_blocks, 256, p, stream);
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

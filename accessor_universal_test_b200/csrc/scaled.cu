// scaled.cu -- encoding into block-scaled 8-bit codes: aut_encode_scaled and
// aut_rms_norm_scaled.
#include "internal.hpp"
#include "dot_device.cuh"
#include "scaled_device.cuh"

namespace aut::scaled {
namespace {

struct encode_params {
  const void *x;
  uint64_t x_stride;
  uint64_t rows, columns;
  uint8_t *codes;
  uint64_t code_stride;
  float *scales;
  uint64_t scale_stride;
};

struct norm_params {
  encode_params e;
  const void *residual;
  void *residual_out;
  uint64_t residual_stride;
  const void *weight;
  float eps;
};

// ---- one row of 128 columns per warp -----------------------------------------
template <int Type, int Code>
__global__ void __launch_bounds__(256) encode_rows_kernel(const encode_params p) {
  using T = element_t<Type>;
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31;
  const uint64_t blocks = (p.columns + kBlock - 1) / kBlock;
  const uint64_t tasks = p.rows * blocks;
  for (uint64_t task = uint64_t{blockIdx.x} * 8 + threadIdx.x / 32; task < tasks;
       task += uint64_t{gridDim.x} * 8) {
    const uint64_t row = task / blocks, block = task % blocks;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    float v[4], largest = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t c = block * kBlock + j * 32 + lane;
      v[j] = c < p.columns ? widen(x[c]) : 0.0f;
      largest = fmaxf(largest, finite_magnitude(v[j]));
    }
    const float scale = scale_of<Code>(warp_max(largest));
    const float reciprocal = __frcp_rn(scale);
    if (lane == 0) p.scales[block * p.scale_stride + row] = scale;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t c = block * kBlock + j * 32 + lane;
      if (c < p.columns)
        p.codes[row * p.code_stride + c] =
            static_cast<uint8_t>(codes_of<Code>(quotient(v[j], scale, reciprocal), 0.0f));
    }
  }
}

// ---- 128 rows of 128 columns per thread block ----------------------------------
template <int Type, int Code>
__global__ void __launch_bounds__(256) encode_tiles_kernel(const encode_params p) {
  using T = element_t<Type>;
  __shared__ float part[8];
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint64_t blocks = (p.columns + kBlock - 1) / kBlock;
  const uint64_t tasks = (p.rows + kBlock - 1) / kBlock * blocks;
  for (uint64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const uint64_t group = task / blocks, block = task % blocks;
    float largest = 0.0f;
    for (int r = warp; r < kBlock; r += 8) {
      const uint64_t row = group * kBlock + r;
      if (row >= p.rows) break;
      const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
      for (int j = 0; j < 4; ++j) {
        const uint64_t c = block * kBlock + j * 32 + lane;
        if (c < p.columns) largest = fmaxf(largest, finite_magnitude(widen(x[c])));
      }
    }
    largest = warp_max(largest);
    if (lane == 0) part[warp] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) largest = fmaxf(largest, part[w]);
    __syncthreads();
    const float scale = scale_of<Code>(largest);
    const float reciprocal = __frcp_rn(scale);
    if (threadIdx.x == 0) p.scales[block * p.scale_stride + group] = scale;
    for (int r = warp; r < kBlock; r += 8) {
      const uint64_t row = group * kBlock + r;
      if (row >= p.rows) break;
      const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
      for (int j = 0; j < 4; ++j) {
        const uint64_t c = block * kBlock + j * 32 + lane;
        if (c < p.columns)
          p.codes[row * p.code_stride + c] = static_cast<uint8_t>(
              codes_of<Code>(quotient(widen(x[c]), scale, reciprocal), 0.0f));
      }
    }
  }
}

// ---- norm: one row per thread block ----------------------------------------------
template <int Type, int Code>
__global__ void __launch_bounds__(256) norm_kernel(const norm_params p) {
  using T = element_t<Type>;
  __shared__ float part[8];
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint64_t columns = p.e.columns;
  const uint64_t blocks = (columns + kBlock - 1) / kBlock;
  const T *weight = static_cast<const T *>(p.weight);
  for (uint64_t row = blockIdx.x; row < p.e.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(p.e.x) + row * p.e.x_stride;
    const T *res = p.residual == nullptr
                       ? nullptr
                       : static_cast<const T *>(p.residual) + row * p.residual_stride;
    T *after = p.residual_out == nullptr
                   ? nullptr
                   : static_cast<T *>(p.residual_out) + row * p.residual_stride;
    float sum = 0.0f;
    for (uint64_t c = threadIdx.x; c < columns; c += 256) {
      const float h = widen(x[c]) + (res == nullptr ? 0.0f : widen(res[c]));
      sum = fmaf(h, h, sum);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += part[w];
    __syncthreads();
    const float r = rsqrtf(sum / static_cast<float>(columns) + p.eps);
    for (uint64_t block = warp; block < blocks; block += 8) {
      float v[4], largest = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t c = block * kBlock + j * 32 + lane;
        v[j] = 0.0f;
        if (c < columns) {
          const float h = widen(x[c]) + (res == nullptr ? 0.0f : widen(res[c]));
          if (after != nullptr) after[c] = narrow<T>(h);
          v[j] = h * r * (weight == nullptr ? 1.0f : widen(weight[c]));
        }
        largest = fmaxf(largest, finite_magnitude(v[j]));
      }
      const float scale = scale_of<Code>(warp_max(largest));
      const float reciprocal = __frcp_rn(scale);
      if (lane == 0) p.e.scales[block * p.e.scale_stride + row] = scale;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t c = block * kBlock + j * 32 + lane;
        if (c < columns)
          p.e.codes[row * p.e.code_stride + c] =
              static_cast<uint8_t>(codes_of<Code>(quotient(v[j], scale, reciprocal), 0.0f));
      }
    }
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

template <int Type, int Code>
aut_status encode_typed(aut_workspace *ws, int32_t block_rows, const encode_params &p,
                        cudaStream_t stream) {
  const uint64_t blocks = (p.columns + kBlock - 1) / kBlock;
  if (block_rows == 1)
    return launch(encode_rows_kernel<Type, Code>, (p.rows * blocks + 7) / 8, 8 * ws->max_blocks,
                  256, p, stream);
  return launch(encode_tiles_kernel<Type, Code>, (p.rows + kBlock - 1) / kBlock * blocks,
                8 * ws->max_blocks, 256, p, stream);
}

template <int Type, int Code>
aut_status norm_typed(aut_workspace *ws, const norm_params &p, cudaStream_t stream) {
  return launch(norm_kernel<Type, Code>, p.e.rows, 8 * ws->max_blocks, 256, p, stream);
}

} // namespace
} // namespace aut::scaled

namespace aut::lib {
using namespace aut::scaled;

aut_status encode_scaled_launch(aut_workspace *ws, int32_t code, int32_t type, int32_t block_rows,
                                const void *values, uint64_t rows, uint64_t columns,
                                uint64_t value_stride, void *codes, uint64_t code_stride,
                                float *scales, uint64_t scale_stride, cudaStream_t stream) {
  const encode_params p{values, value_stride, rows, columns, static_cast<uint8_t *>(codes),
                        code_stride, scales, scale_stride};
  const bool e4m3 = code == AUT_FP8_E4M3;
  switch (type) {
  case AUT_TYPE_FP32:
    return e4m3 ? encode_typed<AUT_TYPE_FP32, AUT_FP8_E4M3>(ws, block_rows, p, stream)
                : encode_typed<AUT_TYPE_FP32, AUT_FP8_E5M2>(ws, block_rows, p, stream);
  case AUT_TYPE_BF16:
    return e4m3 ? encode_typed<AUT_TYPE_BF16, AUT_FP8_E4M3>(ws, block_rows, p, stream)
                : encode_typed<AUT_TYPE_BF16, AUT_FP8_E5M2>(ws, block_rows, p, stream);
  default:
    return e4m3 ? encode_typed<AUT_TYPE_FP16, AUT_FP8_E4M3>(ws, block_rows, p, stream)
                : encode_typed<AUT_TYPE_FP16, AUT_FP8_E5M2>(ws, block_rows, p, stream);
  }
}

aut_status rms_norm_scaled_launch(aut_workspace *ws, int32_t code, int32_t type, const void *x,
                                  uint64_t x_stride, const void *residual, void *residual_out,
                                  uint64_t residual_stride, const void *weight, float eps,
                                  uint64_t rows, uint64_t columns, void *codes,
                                  uint64_t code_stride, float *scales, uint64_t scale_stride,
                                  cudaStream_t stream) {
  norm_params p{};
  p.e = encode_params{x, x_stride, rows, columns, static_cast<uint8_t *>(codes), code_stride,
                      scales, scale_stride};
  p.residual = residual;
  p.residual_out = residual_out;
  p.residual_stride = residual_stride;
  p.weight = weight;
  p.eps = eps;
  const bool e4m3 = code == AUT_FP8_E4M3;
  switch (type) {
  case AUT_TYPE_FP32:
    return e4m3 ? norm_typed<AUT_TYPE_FP32, AUT_FP8_E4M3>(ws, p, stream)
                : norm_typed<AUT_TYPE_FP32, AUT_FP8_E5M2>(ws, p, stream);
  case AUT_TYPE_BF16:
    return e4m3 ? norm_typed<AUT_TYPE_BF16, AUT_FP8_E4M3>(ws, p, stream)
                : norm_typed<AUT_TYPE_BF16, AUT_FP8_E5M2>(ws, p, stream);
  default:
    return e4m3 ? norm_typed<AUT_TYPE_FP16, AUT_FP8_E4M3>(ws, p, stream)
                : norm_typed<AUT_TYPE_FP16, AUT_FP8_E5M2>(ws, p, stream);
  }
}

} // namespace aut::lib

// scaled.cu -- encoding into block-scaled 8-bit codes: aut_encode_scaled and
// aut_rms_norm_scaled.
#include "internal.hpp"
#include "dot_device.cuh"
#include "scaled_device.cuh"

#include <cstring>

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

// ---- a warp's chunk: 256 columns, eight values a lane ---------------------------
// Vec: lane l holds the columns 8 l .. 8 l + 7, one or two 16-byte loads and one
// 8-byte store of codes; 16 lanes share a scale.  Needs rows of values on
// 16-byte and rows of codes on 8-byte boundaries.
// Not Vec: lane l holds the columns l + 32 j, so that any alignment is read and
// written in whole lines; all 32 lanes share the scale of four values.
template <bool Vec>
__device__ __forceinline__ uint32_t column_of(uint32_t chunk, int lane, int j) {
  return Vec ? (chunk * 32 + lane) * 8 + j : chunk * 256 + j * 32 + lane;
}

__device__ __forceinline__ void widen_pair(__nv_bfloat162 p, float &a, float &b) {
  const float2 f = __bfloat1622float2(p);
  a = f.x;
  b = f.y;
}
__device__ __forceinline__ void widen_pair(__half2 p, float &a, float &b) {
  const float2 f = __half22float2(p);
  a = f.x;
  b = f.y;
}

template <class T> struct pair_of;
template <> struct pair_of<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct pair_of<__half> { using type = __half2; };

__device__ __forceinline__ void load_eight(const float *x, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(x)[0];
  const float4 b = reinterpret_cast<const float4 *>(x)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <class T> __device__ __forceinline__ void load_eight(const T *x, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4 *>(x);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    widen_pair(*reinterpret_cast<const typename pair_of<T>::type *>(&w[i]), v[2 * i],
               v[2 * i + 1]);
}

__device__ __forceinline__ void store_eight(float *x, const float (&v)[8]) {
  reinterpret_cast<float4 *>(x)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4 *>(x)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <class T> __device__ __forceinline__ void store_eight(T *x, const float (&v)[8]) {
  T n[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) n[j] = narrow<T>(v[j]);
  uint4 u;
  memcpy(&u, n, 16);
  *reinterpret_cast<uint4 *>(x) = u;
}

// The chunk's values of a row; columns beyond the row read as zero.
template <bool Vec, class T>
__device__ __forceinline__ void load_chunk(const T *row, uint32_t chunk, int lane,
                                           uint32_t columns, float (&v)[8]) {
  if (Vec && column_of<Vec>(chunk, lane, 8) <= columns) {
    load_eight(row + column_of<Vec>(chunk, lane, 0), v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t c = column_of<Vec>(chunk, lane, j);
    v[j] = c < columns ? widen(row[c]) : 0.0f;
  }
}

template <bool Vec, class T>
__device__ __forceinline__ void store_chunk(T *row, uint32_t chunk, int lane, uint32_t columns,
                                            const float (&v)[8]) {
  if (Vec && column_of<Vec>(chunk, lane, 8) <= columns) {
    store_eight(row + column_of<Vec>(chunk, lane, 0), v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t c = column_of<Vec>(chunk, lane, j);
    if (c < columns) row[c] = narrow<T>(v[j]);
  }
}

template <int Code> __device__ __forceinline__ uint32_t four_codes(const float *q) {
  return __byte_perm(codes_of<Code>(q[0], q[1]), codes_of<Code>(q[2], q[3]), 0x5410);
}

// Largest magnitude of the eight values' block or blocks (Vec: m[0]; else
// m[h] for the values 4 h ..).
template <bool Vec, bool Finite>
__device__ __forceinline__ void largest_of(const float (&v)[8], float (&m)[2]) {
  m[0] = m[1] = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float &to = m[Vec ? 0 : j / 4];
    to = fmaxf(to, Finite ? finite_magnitude(v[j]) : fabsf(v[j]));
  }
#pragma unroll
  for (int d = Vec ? 8 : 16; d > 0; d >>= 1) {
    m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], d));
    if (!Vec) m[1] = fmaxf(m[1], __shfl_xor_sync(0xffffffffu, m[1], d));
  }
}

// Encodes the chunk: codes into the row, scales into scales[block * stride].
// All lanes of the warp take part.
template <int Code, bool Vec>
__device__ __forceinline__ void encode_chunk(const float (&v)[8], uint32_t chunk, int lane,
                                             uint32_t columns, uint8_t *row, float *scales,
                                             uint64_t scale_stride) {
  // fmaxf passes over NaN; an infinity shows in the maximum, and only then
  // are the values looked at again without it.
  float m[2];
  largest_of<Vec, false>(v, m);
  if (__any_sync(0xffffffffu, fmaxf(m[0], m[1]) > 3.40282347e38f)) largest_of<Vec, true>(v, m);
  float q[8];
#pragma unroll
  for (int h = 0; h < (Vec ? 1 : 2); ++h) {
    const float scale = scale_of<Code>(m[h]);
    const float reciprocal = __frcp_rn(scale);
    const uint32_t block = chunk * 2 + (Vec ? lane / 16 : h);
    if ((Vec ? lane % 16 : lane) == 0 && block * kBlock < columns)
      scales[block * scale_stride] = scale;
#pragma unroll
    for (int j = h * 4; j < (Vec ? 8 : h * 4 + 4); ++j) q[j] = quotient(v[j], scale, reciprocal);
  }
  const uint32_t lo = four_codes<Code>(q), hi = four_codes<Code>(q + 4);
  if (Vec && column_of<Vec>(chunk, lane, 8) <= columns) {
    *reinterpret_cast<uint2 *>(row + column_of<Vec>(chunk, lane, 0)) = make_uint2(lo, hi);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t c = column_of<Vec>(chunk, lane, j);
    if (c < columns) row[c] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j % 4)));
  }
}

// ---- encode by rows ---------------------------------------------------------------
// A block takes 256 columns of 16 rows, a warp two of the rows, both loaded
// before either is encoded.  The rows of a block are neighbours, so the scales
// of one column block fill whole lines.
constexpr int kEncodeRows = 16;

template <int Type, int Code, bool Vec>
__global__ void __launch_bounds__(256) encode_rows_kernel(const encode_params p) {
  using T = element_t<Type>;
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint32_t columns = static_cast<uint32_t>(p.columns);
  const uint32_t chunks = (columns + 255) / 256;
  const uint32_t chunk = blockIdx.x % chunks;
  const uint64_t first = uint64_t{blockIdx.x / chunks} * kEncodeRows + warp;
  float v[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (first + 8 * i < p.rows)
      load_chunk<Vec>(static_cast<const T *>(p.x) + (first + 8 * i) * p.x_stride, chunk, lane,
                      columns, v[i]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint64_t row = first + 8 * i;
    if (row < p.rows)
      encode_chunk<Code, Vec>(v[i], chunk, lane, columns, p.codes + row * p.code_stride,
                              p.scales + row, p.scale_stride);
  }
}

// ---- encode by tiles of 128 x 128 ----------------------------------------------------
// A block holds its tile in registers, 32 values a thread, so the tile is read
// once.  Vec: lane l holds the columns 4 l ..; else l + 32 j (see above).
template <class T> __device__ __forceinline__ void load_four(const T *x, float *v) {
  const uint2 u = *reinterpret_cast<const uint2 *>(x);
  widen_pair(*reinterpret_cast<const typename pair_of<T>::type *>(&u.x), v[0], v[1]);
  widen_pair(*reinterpret_cast<const typename pair_of<T>::type *>(&u.y), v[2], v[3]);
}
__device__ __forceinline__ void load_four(const float *x, float *v) {
  const float4 f = *reinterpret_cast<const float4 *>(x);
  v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
}

template <int Type, int Code, bool Vec>
__global__ void __launch_bounds__(512) encode_tiles_kernel(const encode_params p) {
  using T = element_t<Type>;
  __shared__ float part[16];
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint32_t columns = static_cast<uint32_t>(p.columns);
  const uint32_t blocks = (columns + kBlock - 1) / kBlock;
  const uint32_t block = blockIdx.x % blocks;
  const uint64_t group = blockIdx.x / blocks;
  uint32_t column[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) column[j] = block * kBlock + (Vec ? lane * 4 + j : lane + 32 * j);
  float v[8][4], largest = 0.0f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const uint64_t row = group * kBlock + r * 16 + warp;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    if (Vec && row < p.rows && column[3] < columns) {
      load_four(x + column[0], v[r]);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[r][j] = row < p.rows && column[j] < columns ? widen(x[column[j]]) : 0.0f;
  }
#pragma unroll
  for (int r = 0; r < 8; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) largest = fmaxf(largest, finite_magnitude(v[r][j]));
  largest = warp_max(largest);
  if (lane == 0) part[warp] = largest;
  __syncthreads();
  largest = part[0];
#pragma unroll
  for (int w = 1; w < 16; ++w) largest = fmaxf(largest, part[w]);
  const float scale = scale_of<Code>(largest);
  const float reciprocal = __frcp_rn(scale);
  if (threadIdx.x == 0) p.scales[block * p.scale_stride + group] = scale;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const uint64_t row = group * kBlock + r * 16 + warp;
    if (row >= p.rows) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[r][j] = quotient(v[r][j], scale, reciprocal);
    const uint32_t codes = four_codes<Code>(v[r]);
    uint8_t *to = p.codes + row * p.code_stride;
    if (Vec && column[3] < columns) {
      *reinterpret_cast<uint32_t *>(to + column[0]) = codes;
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (column[j] < columns) to[column[j]] = static_cast<uint8_t>(codes >> (8 * j));
  }
}

// ---- norm ---------------------------------------------------------------------------
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// A row by Threads threads, which hold it in registers (FP32 h, Chunks times
// eight values a thread), so x and the residual are read once.  Threads = 32:
// four rows to a block of 128.
template <int Type, int Code, bool Vec, int Threads, int Chunks>
__global__ void __launch_bounds__(Threads < 128 ? 128 : Threads)
    norm_kernel(const norm_params p) {
  using T = element_t<Type>;
  constexpr int kWarps = Threads / 32;
  __shared__ float part[kWarps];
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31;
  const int warp = Threads == 32 ? 0 : threadIdx.x / 32;
  const uint64_t row = Threads == 32 ? uint64_t{blockIdx.x} * 4 + threadIdx.x / 32 : blockIdx.x;
  if (row >= p.e.rows) return; // whole warps; whole blocks where a block has one row
  const uint32_t columns = static_cast<uint32_t>(p.e.columns);
  const T *x = static_cast<const T *>(p.e.x) + row * p.e.x_stride;
  float h[Chunks][8], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < Chunks; ++i) load_chunk<Vec>(x, i * kWarps + warp, lane, columns, h[i]);
  if (p.residual != nullptr) {
    const T *residual = static_cast<const T *>(p.residual) + row * p.residual_stride;
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      float r[8];
      load_chunk<Vec>(residual, i * kWarps + warp, lane, columns, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] += r[j];
    }
  }
#pragma unroll
  for (int i = 0; i < Chunks; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
  sum = warp_sum(sum);
  if (Threads > 32) {
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = warp_sum(lane < kWarps ? part[lane] : 0.0f);
  }
  const float r = rsqrtf(sum / static_cast<float>(columns) + p.eps);
#pragma unroll
  for (int i = 0; i < Chunks; ++i) {
    const uint32_t chunk = i * kWarps + warp;
    if (chunk * 256 >= columns) break;
    if (p.residual_out != nullptr)
      store_chunk<Vec>(static_cast<T *>(p.residual_out) + row * p.residual_stride, chunk, lane,
                       columns, h[i]);
    float w[8];
    if (p.weight != nullptr) load_chunk<Vec>(static_cast<const T *>(p.weight), chunk, lane, columns, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[i][j] *= r;
      if (p.weight != nullptr) h[i][j] *= w[j];
    }
    encode_chunk<Code, Vec>(h[i], chunk, lane, columns, p.e.codes + row * p.e.code_stride,
                            p.e.scales + row, p.e.scale_stride);
  }
}

// Rows too long for the registers: read twice, the second time mostly from
// the second-level cache.  A value is read and, in place, written by one and
// the same thread.
template <int Type, int Code>
__global__ void __launch_bounds__(1024) norm_long_kernel(const norm_params p) {
  using T = element_t<Type>;
  __shared__ float part[32];
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint64_t row = blockIdx.x;
  const uint32_t columns = static_cast<uint32_t>(p.e.columns);
  const uint32_t chunks = (columns + 255) / 256;
  const T *x = static_cast<const T *>(p.e.x) + row * p.e.x_stride;
  const T *residual = p.residual == nullptr
                          ? nullptr
                          : static_cast<const T *>(p.residual) + row * p.residual_stride;
  float sum = 0.0f;
  for (uint32_t chunk = warp; chunk < chunks; chunk += 32) {
    float h[8], s[8];
    load_chunk<false>(x, chunk, lane, columns, h);
    if (residual != nullptr) {
      load_chunk<false>(residual, chunk, lane, columns, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] += s[j];
    }
    float own = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) own = fmaf(h[j], h[j], own);
    sum += own;
  }
  sum = warp_sum(sum);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  const float r = rsqrtf(warp_sum(part[lane]) / static_cast<float>(columns) + p.eps);
  for (uint32_t chunk = warp; chunk < chunks; chunk += 32) {
    float h[8], s[8];
    load_chunk<false>(x, chunk, lane, columns, h);
    if (residual != nullptr) {
      load_chunk<false>(residual, chunk, lane, columns, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] += s[j];
    }
    if (p.residual_out != nullptr)
      store_chunk<false>(static_cast<T *>(p.residual_out) + row * p.residual_stride, chunk, lane,
                         columns, h);
    if (p.weight != nullptr)
      load_chunk<false>(static_cast<const T *>(p.weight), chunk, lane, columns, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[j] *= r;
      if (p.weight != nullptr) h[j] *= s[j];
    }
    encode_chunk<Code, false>(h, chunk, lane, columns, p.e.codes + row * p.e.code_stride,
                              p.e.scales + row, p.e.scale_stride);
  }
}

template <class Params>
aut_status launch(void (*kernel)(Params), uint64_t grid, int threads, const Params &p,
                  cudaStream_t stream) {
  if (grid > 0x7fffffffull)
    return aut::lib::fail(AUT_ERR_TOO_LARGE, "more than 2^31 - 1 blocks of rows and columns");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
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

// Whether every row of a matrix starts on a boundary of `bytes`.
bool on_boundaries(const void *p, uint64_t rows, uint64_t stride, uint64_t size, uint64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (rows == 1 || stride * size % bytes == 0);
}

template <int Type, int Code>
aut_status encode_typed(int32_t block_rows, const encode_params &p, cudaStream_t stream) {
  constexpr uint64_t size = sizeof(element_t<Type>);
  if (block_rows == 1) {
    const uint64_t grid = (p.rows + kEncodeRows - 1) / kEncodeRows * ((p.columns + 255) / 256);
    const bool vec = on_boundaries(p.x, p.rows, p.x_stride, size, 16) &&
                     on_boundaries(p.codes, p.rows, p.code_stride, 1, 8);
    return launch(vec ? encode_rows_kernel<Type, Code, true> : encode_rows_kernel<Type, Code, false>,
                  grid, 256, p, stream);
  }
  const uint64_t grid = (p.rows + kBlock - 1) / kBlock * ((p.columns + kBlock - 1) / kBlock);
  const bool vec = on_boundaries(p.x, p.rows, p.x_stride, size, 4 * size) &&
                   on_boundaries(p.codes, p.rows, p.code_stride, 1, 4);
  return launch(vec ? encode_tiles_kernel<Type, Code, true> : encode_tiles_kernel<Type, Code, false>,
                grid, 512, p, stream);
}

// The fewest threads that hold a row with 16 values each (32 beyond 16384
// columns, where a block has no more threads).
template <int Type, int Code, bool Vec>
aut_status norm_rows(const norm_params &p, cudaStream_t stream) {
  const uint64_t rows = p.e.rows, columns = p.e.columns;
  if (columns <= 512)
    return launch(norm_kernel<Type, Code, Vec, 32, 2>, (rows + 3) / 4, 128, p, stream);
  if (columns <= 2048) return launch(norm_kernel<Type, Code, Vec, 128, 2>, rows, 128, p, stream);
  if (columns <= 8192) return launch(norm_kernel<Type, Code, Vec, 512, 2>, rows, 512, p, stream);
  return launch(norm_kernel<Type, Code, Vec, 1024, 4>, rows, 1024, p, stream);
}

template <int Type, int Code>
aut_status norm_typed(const norm_params &p, cudaStream_t stream) {
  constexpr uint64_t size = sizeof(element_t<Type>);
  if (p.e.columns > 32768)
    return launch(norm_long_kernel<Type, Code>, p.e.rows, 1024, p, stream);
  const bool vec = on_boundaries(p.e.x, p.e.rows, p.e.x_stride, size, 16) &&
                   (p.residual == nullptr ||
                    on_boundaries(p.residual, p.e.rows, p.residual_stride, size, 16)) &&
                   (p.residual_out == nullptr ||
                    on_boundaries(p.residual_out, p.e.rows, p.residual_stride, size, 16)) &&
                   (p.weight == nullptr || on_boundaries(p.weight, 1, 0, size, 16)) &&
                   on_boundaries(p.e.codes, p.e.rows, p.e.code_stride, 1, 8);
  return vec ? norm_rows<Type, Code, true>(p, stream) : norm_rows<Type, Code, false>(p, stream);
}

} // namespace
} // namespace aut::scaled

namespace aut::lib {
using namespace aut::scaled;

aut_status encode_scaled_launch(aut_workspace *, int32_t code, int32_t type, int32_t block_rows,
                                const void *values, uint64_t rows, uint64_t columns,
                                uint64_t value_stride, void *codes, uint64_t code_stride,
                                float *scales, uint64_t scale_stride, cudaStream_t stream) {
  const encode_params p{values, value_stride, rows, columns, static_cast<uint8_t *>(codes),
                        code_stride, scales, scale_stride};
  const bool e4m3 = code == AUT_FP8_E4M3;
  switch (type) {
  case AUT_TYPE_FP32:
    return e4m3 ? encode_typed<AUT_TYPE_FP32, AUT_FP8_E4M3>(block_rows, p, stream)
                : encode_typed<AUT_TYPE_FP32, AUT_FP8_E5M2>(block_rows, p, stream);
  case AUT_TYPE_BF16:
    return e4m3 ? encode_typed<AUT_TYPE_BF16, AUT_FP8_E4M3>(block_rows, p, stream)
                : encode_typed<AUT_TYPE_BF16, AUT_FP8_E5M2>(block_rows, p, stream);
  default:
    return e4m3 ? encode_typed<AUT_TYPE_FP16, AUT_FP8_E4M3>(block_rows, p, stream)
                : encode_typed<AUT_TYPE_FP16, AUT_FP8_E5M2>(block_rows, p, stream);
  }
}

aut_status rms_norm_scaled_launch(aut_workspace *, int32_t code, int32_t type, const void *x,
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
    return e4m3 ? norm_typed<AUT_TYPE_FP32, AUT_FP8_E4M3>(p, stream)
                : norm_typed<AUT_TYPE_FP32, AUT_FP8_E5M2>(p, stream);
  case AUT_TYPE_BF16:
    return e4m3 ? norm_typed<AUT_TYPE_BF16, AUT_FP8_E4M3>(p, stream)
                : norm_typed<AUT_TYPE_BF16, AUT_FP8_E5M2>(p, stream);
  default:
    return e4m3 ? norm_typed<AUT_TYPE_FP16, AUT_FP8_E4M3>(p, stream)
                : norm_typed<AUT_TYPE_FP16, AUT_FP8_E5M2>(p, stream);
  }
}

} // namespace aut::lib

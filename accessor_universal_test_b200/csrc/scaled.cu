// scaled.cu -- encoding into block-scaled 8-bit codes: aut_encode_scaled and
// aut_rms_norm_scaled.
#include "internal.hpp"
#include "dot_device.cuh"
#include "scaled_device.cuh"

#include <algorithm>
#include <atomic>

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
// 16-byte and rows of codes on 8-byte boundaries, and a multiple of 8 columns.
// Not Vec: lane l holds the columns l + 32 j, so that any alignment is read and
// written in whole lines; all 32 lanes share the scale of four values.
template <bool Vec>
__device__ __forceinline__ uint32_t column_of(uint32_t chunk, int lane, int j) {
  return Vec ? (chunk * 32 + lane) * 8 + j : chunk * 256 + j * 32 + lane;
}

__device__ __forceinline__ float2 widen_pair(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 widen_pair(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ uint32_t narrow_pair(float2 v, __nv_bfloat16) {
  const __nv_bfloat162 n = __float22bfloat162_rn(v);
  return *reinterpret_cast<const uint32_t *>(&n);
}
__device__ __forceinline__ uint32_t narrow_pair(float2 v, __half) {
  const __half2 n = __float22half2_rn(v);
  return *reinterpret_cast<const uint32_t *>(&n);
}

// Eight values as they stand in memory.
template <class T> struct raw_chunk { uint32_t w[2 * sizeof(T)]; };
template <size_t Size> struct raw_word { using type = uint32_t; };
template <> struct raw_word<2> { using type = uint16_t; };

__device__ __forceinline__ void widen_chunk(const raw_chunk<float> &r, float2 (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = make_float2(__uint_as_float(r.w[2 * j]), __uint_as_float(r.w[2 * j + 1]));
}
template <class T>
__device__ __forceinline__ void widen_chunk(const raw_chunk<T> &r, float2 (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = widen_pair(r.w[j], T{});
}

__device__ __forceinline__ void store_eight(float *x, const float2 (&v)[4]) {
  reinterpret_cast<float4 *>(x)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
  reinterpret_cast<float4 *>(x)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
}
template <class T> __device__ __forceinline__ void store_eight(T *x, const float2 (&v)[4]) {
  *reinterpret_cast<uint4 *>(x) = make_uint4(narrow_pair(v[0], T{}), narrow_pair(v[1], T{}),
                                             narrow_pair(v[2], T{}), narrow_pair(v[3], T{}));
}

// The chunk's values of a row; columns beyond the row read as zero.
template <bool Vec, class T>
__device__ __forceinline__ raw_chunk<T> load_raw(const T *row, uint32_t chunk, int lane,
                                                 uint32_t columns) {
  raw_chunk<T> r;
  const uint32_t c0 = column_of<Vec>(chunk, lane, 0);
  if constexpr (Vec) {
    const uint4 *x = reinterpret_cast<const uint4 *>(row + c0);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      const uint4 u = c0 < columns ? x[i] : make_uint4(0u, 0u, 0u, 0u);
      r.w[4 * i] = u.x, r.w[4 * i + 1] = u.y, r.w[4 * i + 2] = u.z, r.w[4 * i + 3] = u.w;
    }
  } else {
    using word = typename raw_word<sizeof(T)>::type;
    const word *x = reinterpret_cast<const word *>(row + c0);
    uint32_t bits[8];
    if (chunk * 256 + 256 <= columns) {
#pragma unroll
      for (int j = 0; j < 8; ++j) bits[j] = x[32 * j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) bits[j] = c0 + 32 * j < columns ? x[32 * j] : word{0};
    }
#pragma unroll
    for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i)
      r.w[i] = sizeof(T) == 4 ? bits[i] : bits[2 * i % 8] | bits[(2 * i + 1) % 8] << 16;
  }
  return r;
}

template <bool Vec, class T>
__device__ __forceinline__ void load_chunk(const T *row, uint32_t chunk, int lane,
                                           uint32_t columns, float2 (&v)[4]) {
  widen_chunk(load_raw<Vec>(row, chunk, lane, columns), v);
}

template <bool Vec, class T>
__device__ __forceinline__ void store_chunk(T *row, uint32_t chunk, int lane, uint32_t columns,
                                            const float2 (&v)[4]) {
  const uint32_t c0 = column_of<Vec>(chunk, lane, 0);
  if constexpr (Vec) {
    if (c0 < columns) store_eight(row + c0, v);
  } else {
    T *to = row + c0;
    if (chunk * 256 + 256 <= columns) {
#pragma unroll
      for (int j = 0; j < 8; ++j) to[32 * j] = narrow<T>(j % 2 == 0 ? v[j / 2].x : v[j / 2].y);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + 32 * j < columns) to[32 * j] = narrow<T>(j % 2 == 0 ? v[j / 2].x : v[j / 2].y);
    }
  }
}

template <int Code> __device__ __forceinline__ uint32_t four_codes(float2 a, float2 b) {
  return __byte_perm(codes_of<Code>(a.x, a.y), codes_of<Code>(b.x, b.y), 0x5410);
}

// Largest magnitude of four values (not NaN, which is passed over; infinite
// if one of them is).
__device__ __forceinline__ float largest_of(float2 a, float2 b) {
  return fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y)));
}

// Takes infinities out of a value's block: they encode as NaN and do not
// count for the scale.
__device__ __forceinline__ float without_infinity(float v) {
  return fabsf(v) <= 3.40282347e38f ? v : __int_as_float(0x7fffffff);
}

// Encodes a chunk of numbers with the largest magnitudes m of the lane's values
// (of either half of them, or of all in both): codes into the row, scales into
// scales[block * stride], times back.  All lanes of the warp take part.
template <int Code, bool Vec>
__device__ __forceinline__ void encode_numbers(const float2 (&v)[4], const float (&m)[2],
                                               uint32_t chunk, int lane, uint32_t columns,
                                               uint8_t *row, float *scales,
                                               uint64_t scale_stride, const float (&back)[2]) {
  uint32_t codes[4]; // two each
  block_scale s;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h < (Vec ? 1 : 2)) {
      s = scale_of<Code>(Vec ? half_warp_max(m[h], lane) : warp_max(m[h]));
      const uint32_t block = chunk * 2 + (Vec ? lane / 16 : h);
      if ((Vec ? lane % 16 : lane) == 0 && block * kBlock < columns)
        scales[block * scale_stride] = s.scale * back[h];
    }
#pragma unroll
    for (int j = 2 * h; j < 2 * h + 2; ++j) {
      const float2 q = quotient(v[j], s);
      codes[j] = codes_of<Code>(q.x, q.y);
    }
  }
  const uint32_t c0 = column_of<Vec>(chunk, lane, 0);
  if constexpr (Vec) {
    if (c0 < columns)
      *reinterpret_cast<uint2 *>(row + c0) = make_uint2(__byte_perm(codes[0], codes[1], 0x5410),
                                                        __byte_perm(codes[2], codes[3], 0x5410));
  } else {
    uint8_t *to = row + c0;
    if (chunk * 256 + 256 <= columns) {
#pragma unroll
      for (int j = 0; j < 8; ++j) to[32 * j] = static_cast<uint8_t>(codes[j / 2] >> (8 * (j % 2)));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + 32 * j < columns)
          to[32 * j] = static_cast<uint8_t>(codes[j / 2] >> (8 * (j % 2)));
    }
  }
}

// The same of any values.  Exact: with scales above kLargeScale too (of a norm's
// values, which are within some ulp of theirs, no quotient's rounding is that exact).
template <int Code, bool Vec, bool Exact>
__device__ __forceinline__ void encode_chunk(float2 (&v)[4], uint32_t chunk, int lane,
                                             uint32_t columns, uint8_t *row, float *scales,
                                             uint64_t scale_stride) {
  float m[2] = {largest_of(v[0], v[1]), largest_of(v[2], v[3])}, back[2] = {1.0f, 1.0f};
  if (Vec) m[0] = m[1] = fmaxf(m[0], m[1]);
  // Rare, and not worth a test for every value: an infinity or a large scale.
  if (__any_sync(0xffffffffu, fmaxf(m[0], m[1]) > (Exact ? kLargeScale : 3.40282347e38f))) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = make_float2(without_infinity(v[j].x), without_infinity(v[j].y));
    m[0] = largest_of(v[0], v[1]), m[1] = largest_of(v[2], v[3]);
    if (Vec) m[0] = m[1] = fmaxf(m[0], m[1]);
    if constexpr (Exact) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool large = (Vec ? half_warp_max(m[h], lane) : warp_max(m[h])) > kLargeScale;
        const float down = large ? kDown : 1.0f;
        back[h] = large ? kUp : 1.0f;
        m[h] *= down;
#pragma unroll
        for (int j = 2 * h; j < 2 * h + 2; ++j) v[j] = mul2(v[j], make_float2(down, down));
      }
      // code of its own: a factor of every scale made all others 6 % slower
      encode_numbers<Code, Vec>(v, m, chunk, lane, columns, row, scales, scale_stride, back);
      return;
    }
  }
  encode_numbers<Code, Vec>(v, m, chunk, lane, columns, row, scales, scale_stride, back);
}

// ---- encode by rows ---------------------------------------------------------------
// Block (c, y) takes chunk c of the row groups y, y + gridDim.y, ... of 16
// rows, a warp two rows of a group; the next group's values are loaded before
// this one's are encoded, so loads are under way all the time.  The rows of a
// group are neighbours: the scales of one column block fill whole lines.
// Bound by memory, with the schedulers busy two thirds of the time (the search
// for the maximum, the scale and the conversions).  Measured, copy bandwidth
// 6.55 TB/s: 4096 x 8192 BF16 17.9 us (5.6 TB/s), FP32 26.2 (6.4); 4096 x 5001 FP32
// 18.3 (5.6), FP16 20.1 (3.1: eight loads and eight stores of a lane for
// one of each where rows start on 16 bytes).
constexpr int kEncodeRows = 16;

template <int Type, int Code, bool Vec>
__global__ void __launch_bounds__(256) encode_rows_kernel(const encode_params p) {
  using T = element_t<Type>;
  constexpr bool kExact = Type != AUT_TYPE_FP16; // FP16 has no values that large
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint32_t columns = static_cast<uint32_t>(p.columns);
  const uint32_t chunk = blockIdx.x;
  const uint64_t step = uint64_t{gridDim.y} * kEncodeRows;
  const uint64_t first = uint64_t{blockIdx.y} * kEncodeRows + warp;
  const T *x = static_cast<const T *>(p.x) + first * p.x_stride;
  uint8_t *codes = p.codes + first * p.code_stride;
  const uint64_t x_step = step * p.x_stride, code_step = step * p.code_stride;
  raw_chunk<T> next[2];
  if (first < p.rows) next[0] = load_raw<Vec>(x, chunk, lane, columns);
  if (first + 8 < p.rows) next[1] = load_raw<Vec>(x + 8 * p.x_stride, chunk, lane, columns);
  for (uint64_t row = first; row < p.rows; row += step, codes += code_step) {
    const bool two = row + 8 < p.rows;
    float2 v[2][4];
    widen_chunk(next[0], v[0]);
    widen_chunk(next[1], v[1]);
    x += x_step;
    if (row + step < p.rows) next[0] = load_raw<Vec>(x, chunk, lane, columns);
    if (row + step + 8 < p.rows) next[1] = load_raw<Vec>(x + 8 * p.x_stride, chunk, lane, columns);
    encode_chunk<Code, Vec, kExact>(v[0], chunk, lane, columns, codes, p.scales + row, p.scale_stride);
    if (two)
      encode_chunk<Code, Vec, kExact>(v[1], chunk, lane, columns, codes + 8 * p.code_stride,
                              p.scales + row + 8, p.scale_stride);
  }
}

// ---- encode by tiles of 128 x 128 ----------------------------------------------------
// A block holds a tile in registers (16 a thread: 32 values of 16 bits, 16 of
// 32), so the tile is read once, and loads its next one before it encodes this
// one.  Vec: lane l holds the columns 4 l .., a multiple of 4 in all; else
// l + 32 j (see above).  Measured: 8192 x 8192 FP32 51.1 us (6.6 TB/s), BF16 36.7
// (5.5), 8192 x 5120 BF16 24.3 (5.2), 8191 x 5001 FP32 35.1 (5.8), FP16 40.1 (3.1;
// with a test of row and column at each value of every tile 51.7).
template <class T> struct tile_of {
  static constexpr int kThreads = sizeof(T) == 4 ? 1024 : 512;
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kRows = kBlock / kWarps; // of each warp
};
// Four values of a row.
template <class T> struct raw_four { uint32_t w[sizeof(T)]; };

__device__ __forceinline__ void widen_four(const raw_four<float> &r, float2 (&v)[2]) {
  v[0] = make_float2(__uint_as_float(r.w[0]), __uint_as_float(r.w[1]));
  v[1] = make_float2(__uint_as_float(r.w[2]), __uint_as_float(r.w[3]));
}
template <class T> __device__ __forceinline__ void widen_four(const raw_four<T> &r, float2 (&v)[2]) {
  v[0] = widen_pair(r.w[0], T{}), v[1] = widen_pair(r.w[1], T{});
}

// column: the lane's first; what is beyond the matrix reads as zero.  whole: the
// tile lies in the matrix.
template <bool Vec, class T>
__device__ __forceinline__ raw_four<T> load_four(const T *row, bool whole, bool has_row,
                                                 uint32_t column, uint32_t columns) {
  raw_four<T> r;
  if constexpr (Vec) {
    const bool has = has_row && column < columns;
    if constexpr (sizeof(T) == 4) {
      const uint4 u = has ? *reinterpret_cast<const uint4 *>(row + column) : make_uint4(0, 0, 0, 0);
      r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
    } else {
      const uint2 u = has ? *reinterpret_cast<const uint2 *>(row + column) : make_uint2(0, 0);
      r.w[0] = u.x, r.w[1] = u.y;
    }
  } else {
    using word = typename raw_word<sizeof(T)>::type;
    const word *x = reinterpret_cast<const word *>(row + column);
    uint32_t bits[4];
    if (whole) {
#pragma unroll
      for (int j = 0; j < 4; ++j) bits[j] = x[32 * j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        bits[j] = has_row && column + 32 * j < columns ? x[32 * j] : word{0};
    }
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i)
      r.w[i] = sizeof(T) == 4 ? bits[i] : bits[2 * i % 4] | bits[(2 * i + 1) % 4] << 16;
  }
  return r;
}

template <int Type, int Code, bool Vec>
__global__ void __launch_bounds__(tile_of<element_t<Type>>::kThreads,
                                  1024 / tile_of<element_t<Type>>::kThreads)
    encode_tiles_kernel(const encode_params p) {
  using T = element_t<Type>;
  using tile = tile_of<T>;
  __shared__ float part[2][tile::kWarps];
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint32_t columns = static_cast<uint32_t>(p.columns);
  const uint32_t blocks = (columns + kBlock - 1) / kBlock;
  const uint64_t groups = (p.rows + kBlock - 1) / kBlock;
  // tile = (row group, column block); blocks take every gridDim.x-th
  const uint32_t step_groups = gridDim.x / blocks, step_blocks = gridDim.x % blocks;
  uint64_t group = blockIdx.x / blocks;
  uint32_t block = blockIdx.x % blocks;
  const uint32_t lane_column = Vec ? lane * 4 : lane;
  raw_four<T> next[tile::kRows];
  auto is_whole = [&](uint64_t group, uint32_t block) {
    return (group + 1) * kBlock <= p.rows && (block + 1) * kBlock <= columns;
  };
  auto load = [&] {
    const uint64_t first = group * kBlock + warp;
    const T *x = static_cast<const T *>(p.x) + first * p.x_stride;
    const bool whole = is_whole(group, block);
#pragma unroll
    for (int r = 0; r < tile::kRows; ++r)
      next[r] = load_four<Vec>(x + r * tile::kWarps * p.x_stride, whole,
                               first + r * tile::kWarps < p.rows, block * kBlock + lane_column,
                               columns);
  };
  load();
  for (int turn = 0; group < groups; turn ^= 1) {
    raw_four<T> now[tile::kRows];
#pragma unroll
    for (int r = 0; r < tile::kRows; ++r) now[r] = next[r];
    const uint64_t group_now = group;
    const uint32_t block_now = block;
    group += step_groups;
    block += step_blocks;
    if (block >= blocks) {
      block -= blocks;
      ++group;
    }
    if (group < groups) load();
    float largest = 0.0f;
#pragma unroll
    for (int r = 0; r < tile::kRows; ++r) {
      float2 v[2];
      widen_four(now[r], v);
      largest = fmaxf(largest, largest_of(v[0], v[1]));
    }
    largest = warp_max(largest);
    // two sets of maxima: no warp is more than one tile ahead of another
    if (lane == 0) part[turn][warp] = largest;
    __syncthreads();
    largest = warp_max(part[turn][lane % tile::kWarps]);
    // rare, and the same for all: an infinity or a large scale
    const bool large = largest > kLargeScale;
    float down = 1.0f, back = 1.0f;
    if (large) {
      __syncthreads();
      largest = 0.0f;
#pragma unroll
      for (int r = 0; r < tile::kRows; ++r) {
        float2 v[2];
        widen_four(now[r], v);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          largest = fmaxf(largest, fmaxf(finite_magnitude(v[j].x), finite_magnitude(v[j].y)));
      }
      largest = warp_max(largest);
      if (lane == 0) part[turn][warp] = largest;
      __syncthreads();
      largest = warp_max(part[turn][lane % tile::kWarps]);
      if (largest > kLargeScale) largest *= kDown, down = kDown, back = kUp;
    }
    const block_scale s = scale_of<Code>(largest);
    if (threadIdx.x == 0) p.scales[block_now * p.scale_stride + group_now] = s.scale * back;
    const uint64_t first = group_now * kBlock + warp;
    const uint32_t column = block_now * kBlock + lane_column;
    uint8_t *to = p.codes + first * p.code_stride + column;
    const bool whole = is_whole(group_now, block_now);
#pragma unroll
    for (int r = 0; r < tile::kRows; ++r, to += tile::kWarps * p.code_stride) {
      float2 v[2];
      widen_four(now[r], v);
      if (large) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          v[j] = mul2(make_float2(without_infinity(v[j].x), without_infinity(v[j].y)),
                      make_float2(down, down));
      }
      const uint32_t codes = four_codes<Code>(quotient(v[0], s), quotient(v[1], s));
      const bool has_row = first + r * tile::kWarps < p.rows;
      if constexpr (Vec) {
        if (has_row && column < columns) *reinterpret_cast<uint32_t *>(to) = codes;
      } else if (whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) to[32 * j] = static_cast<uint8_t>(codes >> (8 * j));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (has_row && column + 32 * j < columns)
            to[32 * j] = static_cast<uint8_t>(codes >> (8 * j));
      }
    }
  }
}

// ---- norm ---------------------------------------------------------------------------
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Rows by up to Threads threads each, which hold a row in registers (FP32 h,
// Chunks times eight values a thread), so x and the residual are read once; the
// weight stays in registers over the rows of a block.  The next row's values
// are loaded before this one's are summed and encoded.  Threads = 32: four
// rows to a block of 128.  Bound by memory; one barrier a row, which the other
// blocks of the SM fill.  Measured with a residual in place: 4096 x 8192 BF16 40.0 us
// (5.9 TB/s), 4096 x 4096 FP32 35.9 (6.1), 4096 x 5001 FP32 48.2 (5.5), BF16 55.5 (2.6:
// the same count of instructions as FP32 for half the bytes, and stores of 64
// bytes that begin and end within a sector), 1 x 4096 BF16 1.6.  FP32 rows of 8193 to
// 16384 columns do not fit: 120 bytes a thread go to local memory (240 off 16-byte
// boundaries) and 4096 x 12288 takes 132 us (5.0 TB/s); 16-bit rows there, 24 to 32.
template <int Type, int Code, bool Vec, int Threads, int Chunks>
__global__ void __launch_bounds__(Threads < 128 ? 128 : Threads,
                                  65536 / (Threads < 256 ? 48 : Threads < 512 ? 80 : 64) /
                                      (Threads < 128 ? 128 : Threads))
    norm_kernel(const norm_params p) {
  using T = element_t<Type>;
  __shared__ float part[2][Threads / 32];
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31;
  const int warp = Threads == 32 ? 0 : threadIdx.x / 32;
  const int warps = Threads == 32 ? 1 : blockDim.x / 32;
  const uint64_t rows_a_block = Threads == 32 ? 4 : 1;
  const uint64_t step = gridDim.x * rows_a_block;
  uint64_t row = blockIdx.x * rows_a_block + (Threads == 32 ? threadIdx.x / 32 : 0);
  if (row >= p.e.rows) return; // whole warps; whole blocks where a block has one row
  const uint32_t columns = static_cast<uint32_t>(p.e.columns);
  const float mean_of = static_cast<float>(columns);
  const T *x = static_cast<const T *>(p.e.x) + row * p.e.x_stride;
  const T *residual = static_cast<const T *>(p.residual) + row * p.residual_stride;
  raw_chunk<T> next[Chunks], more[Chunks], weight[Chunks];
#pragma unroll
  for (int i = 0; i < Chunks; ++i) {
    next[i] = load_raw<Vec>(x, i * warps + warp, lane, columns);
    if (p.residual != nullptr)
      more[i] = load_raw<Vec>(residual, i * warps + warp, lane, columns);
  }
#pragma unroll
  for (int i = 0; i < Chunks; ++i)
    if (p.weight != nullptr)
      weight[i] = load_raw<Vec>(static_cast<const T *>(p.weight), i * warps + warp, lane, columns);
  for (int turn = 0; row < p.e.rows; row += step, turn ^= 1) {
    float2 h[Chunks][4], squares = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      widen_chunk(next[i], h[i]);
      if (p.residual != nullptr) {
        float2 r[4];
        widen_chunk(more[i], r);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[i][j] = add2(h[i][j], r[j]);
      }
    }
    if (row + step < p.e.rows) {
      x += step * p.e.x_stride;
      residual += step * p.residual_stride;
#pragma unroll
      for (int i = 0; i < Chunks; ++i) {
        next[i] = load_raw<Vec>(x, i * warps + warp, lane, columns);
        if (p.residual != nullptr)
          more[i] = load_raw<Vec>(residual, i * warps + warp, lane, columns);
      }
    }
#pragma unroll
    for (int i = 0; i < Chunks; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) squares = fma2(h[i][j], h[i][j], squares);
    float sum = warp_sum(squares.x + squares.y);
    if constexpr (Threads > 32) {
      // two sets of sums: no warp is more than one row ahead of another
      if (lane == 0) part[turn][warp] = sum;
      __syncthreads();
      sum = warp_sum(lane < warps ? part[turn][lane] : 0.0f);
    }
    const float r = rsqrtf(sum / mean_of + p.eps);
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      const uint32_t chunk = i * warps + warp;
      if (chunk * 256 >= columns) break;
      if (p.residual_out != nullptr)
        store_chunk<Vec>(static_cast<T *>(p.residual_out) + row * p.residual_stride, chunk, lane,
                         columns, h[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[i][j] = mul2(h[i][j], make_float2(r, r));
      if (p.weight != nullptr) {
        float2 w[4];
        widen_chunk(weight[i], w);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[i][j] = mul2(h[i][j], w[j]);
      }
      encode_chunk<Code, Vec, false>(h[i], chunk, lane, columns, p.e.codes + row * p.e.code_stride,
                              p.e.scales + row, p.e.scale_stride);
    }
  }
}

// Rows too long for the registers: read twice, the second time mostly from
// the second-level cache.  A value is read and, in place, written by one and
// the same thread.  Element by element on any boundary: 4096 x 18432 BF16 155 us
// (3.4 TB/s of what has to move).
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
    float2 h[4], s[4];
    load_chunk<false>(x, chunk, lane, columns, h);
    if (residual != nullptr) {
      load_chunk<false>(residual, chunk, lane, columns, s);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = add2(h[j], s[j]);
    }
    float2 own = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < 4; ++j) own = fma2(h[j], h[j], own);
    sum += own.x + own.y;
  }
  sum = warp_sum(sum);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  const float r = rsqrtf(warp_sum(part[lane]) / static_cast<float>(columns) + p.eps);
  for (uint32_t chunk = warp; chunk < chunks; chunk += 32) {
    float2 h[4], s[4];
    load_chunk<false>(x, chunk, lane, columns, h);
    if (residual != nullptr) {
      load_chunk<false>(residual, chunk, lane, columns, s);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = add2(h[j], s[j]);
    }
    if (p.residual_out != nullptr)
      store_chunk<false>(static_cast<T *>(p.residual_out) + row * p.residual_stride, chunk, lane,
                         columns, h);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = mul2(h[j], make_float2(r, r));
    if (p.weight != nullptr) {
      load_chunk<false>(static_cast<const T *>(p.weight), chunk, lane, columns, s);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = mul2(h[j], s[j]);
    }
    encode_chunk<Code, false, false>(h, chunk, lane, columns, p.e.codes + row * p.e.code_stride,
                              p.e.scales + row, p.e.scale_stride);
  }
}

template <class Params>
aut_status launch(void (*kernel)(Params), uint64_t grid, int threads, const Params &p,
                  cudaStream_t stream, unsigned grid_y = 1) {
  if (grid > 0x7fffffffull)
    return aut::lib::fail(AUT_ERR_TOO_LARGE, "more than 2^31 - 1 blocks of rows and columns");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), grid_y);
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

// How many blocks of a kernel run on one SM at a time.
template <class Params> int resident_blocks(void (*kernel)(Params), int threads) {
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess) n = 1;
  return std::max(n, 1);
}

// All the kernels run as many blocks as fit at one time, each block over many
// rows or tiles.
template <int Type, int Code, bool Vec>
aut_status encode_by_rows(aut_workspace *ws, const encode_params &p, cudaStream_t stream) {
  auto kernel = encode_rows_kernel<Type, Code, Vec>;
  static const int resident = resident_blocks(kernel, 256);
  const uint64_t chunks = (p.columns + 255) / 256;
  const uint64_t groups = (p.rows + kEncodeRows - 1) / kEncodeRows;
  const uint64_t most = std::max<uint64_t>(1, static_cast<uint64_t>(resident * ws->sm_count) / chunks);
  return launch(kernel, chunks, 256, p, stream, static_cast<unsigned>(std::min(groups, most)));
}

template <int Type, int Code, bool Vec>
aut_status encode_by_tiles(aut_workspace *ws, const encode_params &p, cudaStream_t stream) {
  constexpr int kThreads = tile_of<element_t<Type>>::kThreads;
  auto kernel = encode_tiles_kernel<Type, Code, Vec>;
  static const int resident = resident_blocks(kernel, kThreads);
  const uint64_t tiles =
      (p.rows + kBlock - 1) / kBlock * ((p.columns + kBlock - 1) / kBlock);
  return launch(kernel, std::min(tiles, static_cast<uint64_t>(resident * ws->sm_count)), kThreads,
                p, stream);
}

template <int Type, int Code>
aut_status encode_typed(aut_workspace *ws, int32_t block_rows, const encode_params &p,
                        cudaStream_t stream) {
  constexpr uint64_t size = sizeof(element_t<Type>);
  if (block_rows == 1) {
    const bool vec = p.columns % 8 == 0 && on_boundaries(p.x, p.rows, p.x_stride, size, 16) &&
                     on_boundaries(p.codes, p.rows, p.code_stride, 1, 8);
    return vec ? encode_by_rows<Type, Code, true>(ws, p, stream)
               : encode_by_rows<Type, Code, false>(ws, p, stream);
  }
  const bool vec = p.columns % 4 == 0 && on_boundaries(p.x, p.rows, p.x_stride, size, 4 * size) &&
                   on_boundaries(p.codes, p.rows, p.code_stride, 1, 4);
  return vec ? encode_by_tiles<Type, Code, true>(ws, p, stream)
             : encode_by_tiles<Type, Code, false>(ws, p, stream);
}

template <int Type, int Code, bool Vec, int Threads, int Chunks>
aut_status norm_launch(aut_workspace *ws, const norm_params &p, cudaStream_t stream) {
  auto kernel = norm_kernel<Type, Code, Vec, Threads, Chunks>;
  // as many warps as hold the row
  const uint64_t columns = 256 * Chunks;
  const int warps = Threads == 32 ? 4 : static_cast<int>((p.e.columns + columns - 1) / columns);
  static std::atomic<int> resident[33];
  int n = resident[warps].load(std::memory_order_relaxed);
  if (n == 0)
    resident[warps].store(n = resident_blocks(kernel, 32 * warps), std::memory_order_relaxed);
  const uint64_t blocks = Threads == 32 ? (p.e.rows + 3) / 4 : p.e.rows;
  return launch(kernel, std::min(blocks, static_cast<uint64_t>(n * ws->sm_count)), 32 * warps, p,
                stream);
}

// Sixteen values a thread, or eight: where that is one warp or few (4096 x 640
// BF16: 5.0 against 5.8 us), for values of 32 bits, which sixteen leave no
// registers for the next row (4096 x 5001: 47 against 59 us), and where there
// is less than a row for every SM, so that the time of one row counts (1 x 4096:
// 1.8 against 2.0 us).  Elsewhere sixteen keep more rows under way (4096 x 5000
// BF16: 27 against 31 us).
template <int Type, int Code, bool Vec>
aut_status norm_rows(aut_workspace *ws, const norm_params &p, cudaStream_t stream) {
  const uint64_t columns = p.e.columns;
  if (columns <= 256) return norm_launch<Type, Code, Vec, 32, 1>(ws, p, stream);
  if (columns <= 1024) return norm_launch<Type, Code, Vec, 128, 1>(ws, p, stream);
  if (columns <= 8192) {
    if constexpr (Type != AUT_TYPE_FP32) {
      if (p.e.rows > static_cast<uint64_t>(ws->sm_count))
        return columns <= 4096 ? norm_launch<Type, Code, Vec, 256, 2>(ws, p, stream)
                               : norm_launch<Type, Code, Vec, 512, 2>(ws, p, stream);
    }
    return norm_launch<Type, Code, Vec, 1024, 1>(ws, p, stream);
  }
  return norm_launch<Type, Code, Vec, 1024, 2>(ws, p, stream);
}

template <int Type, int Code>
aut_status norm_typed(aut_workspace *ws, const norm_params &p, cudaStream_t stream) {
  constexpr uint64_t size = sizeof(element_t<Type>);
  if (p.e.columns > 16384)
    return launch(norm_long_kernel<Type, Code>, p.e.rows, 1024, p, stream);
  const bool vec = p.e.columns % 8 == 0 && on_boundaries(p.e.x, p.e.rows, p.e.x_stride, size, 16) &&
                   (p.residual == nullptr ||
                    on_boundaries(p.residual, p.e.rows, p.residual_stride, size, 16)) &&
                   (p.residual_out == nullptr ||
                    on_boundaries(p.residual_out, p.e.rows, p.residual_stride, size, 16)) &&
                   (p.weight == nullptr || on_boundaries(p.weight, 1, 0, size, 16)) &&
                   on_boundaries(p.e.codes, p.e.rows, p.e.code_stride, 1, 8);
  return vec ? norm_rows<Type, Code, true>(ws, p, stream)
             : norm_rows<Type, Code, false>(ws, p, stream);
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

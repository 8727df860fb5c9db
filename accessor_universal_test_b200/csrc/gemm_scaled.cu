// gemm_scaled.cu -- aut_gemm_scaled: the product of two matrices of
// block-scaled 8-bit codes.
#include "gemm_scaled.cuh"

namespace aut::scaled {
namespace {

// Four codes of a row from column c on, which may be negative; row + c is on a
// 4-byte boundary.  What lies outside the row's k codes is not read and counts
// as zero (what a caller's row padding holds never enters the product).
__device__ __forceinline__ uint32_t load_word(const uint8_t *row, int64_t c, int64_t k) {
  if (c >= 0 && c + 4 <= k) return __ldg(reinterpret_cast<const uint32_t *>(row + c));
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j >= 0 && c + j < k) w |= uint32_t{row[c + j]} << (8 * j);
  return w;
}

// Bytes of `row` beyond a 4-byte boundary.
__device__ __forceinline__ int offset_in_word(const uint8_t *row) {
  return static_cast<int>(reinterpret_cast<uintptr_t>(row) & 3);
}

// Sixteen codes of a row of any alignment from column c, a multiple of 16, on.
__device__ __forceinline__ uint4 load_codes(const uint8_t *row, uint64_t c, uint64_t k) {
  const int s = offset_in_word(row);
  const int64_t first = static_cast<int64_t>(c) - s, end = static_cast<int64_t>(k);
  uint32_t w[5];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = load_word(row, first + 4 * i, end);
  w[4] = s == 0 ? 0u : load_word(row, first + 16, end);
  return make_uint4(__funnelshift_r(w[0], w[1], 8 * s), __funnelshift_r(w[1], w[2], 8 * s),
                    __funnelshift_r(w[2], w[3], 8 * s), __funnelshift_r(w[3], w[4], 8 * s));
}

// The same of a row on a 16-byte boundary; what its end cuts is read byte by byte
// in a loop, which takes few registers (1 x 4096 x 4000: 5.1 us; 8.4 with all bytes
// at once, which spills).
__device__ __forceinline__ uint4 load_end(const uint8_t *row, uint64_t c, uint64_t k) {
  if (c + 16 <= k) return __ldg(reinterpret_cast<const uint4 *>(row + c));
  uint64_t lo = 0, hi = 0;
#pragma unroll 1
  for (uint64_t at = k; at-- > c;) {
    hi = hi << 8 | lo >> 56;
    lo = lo << 8 | row[at];
  }
  return make_uint4(static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32),
                    static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32));
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

// The same over the thread blocks of a cluster, in rank order: each stores a
// share of the sums.
template <int Rows, int Columns, int Parts>
__device__ __forceinline__ void join_cluster(const gemm_params &p,
                                             const float (&sums)[8][Rows][Columns], uint64_t n0,
                                             uint32_t rank) {
  __shared__ float joined[Rows * Columns];
  for (int at = threadIdx.x; at < Rows * Columns; at += 256) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][at % Rows][at / Rows];
    joined[at] = s;
  }
  cluster_sync();
  constexpr uint32_t share = Rows * Columns / Parts;
  for (uint32_t i = threadIdx.x; i < share; i += 256) {
    const uint32_t at = rank * share + i;
    float s = 0.0f;
#pragma unroll
    for (uint32_t q = 0; q < Parts; ++q) s += cluster_load(&joined[at], q);
    if (n0 + at % Rows < p.n && at / Rows < p.m) store_out(p, at / Rows, n0 + at % Rows, s);
  }
  cluster_sync(); // no block leaves before the others have read its sums
}

// ---- any alignment, few rows of a ----------------------------------------------------
// A thread block computes 16 rows of b against 8 rows of a; its warps share the
// blocks of k.
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

// ---- any alignment, many rows of a ---------------------------------------------------
// A thread block computes 128 rows of b against 64 rows of a, a warp 32 against
// 32.  The blocks of k go through shared memory: rows are read as the aligned
// words that hold them, a line of a row to a warp, moved into place and widened
// to FP16, which holds every code's value (4096 x 4096 x 1999: 462 us; with the codes
// as they are, 509, more of whose registers spill: here 92 bytes a thread).  The next block's words are
// under way behind this block's products.  Eight values stand
// at chunk ^ 4 in odd rows, so that eight lanes' reads of two rows meet no bank
// twice.  The few rows' kernel took 4170 us there; operands on 16-byte
// boundaries take about 30.
constexpr int kAnyN = 128, kAnyM = 64, kAnyThreads = 256;

struct any_tile {
  union {
    uint4 values[kAnyN + kAnyM][kBlock / 8];
    float out[kAnyM][kAnyN + 1];
  };
  float scales[kAnyM];
  const uint8_t *rows[kAnyN + kAnyM];
};

// Four codes as FP16.
template <int Code> __device__ __forceinline__ uint2 widen_codes(uint32_t w) {
  uint2 v;
  if (Code == AUT_FP8_E4M3)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(v.x), "=r"(v.y)
        : "r"(w));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e5m2x2 %0, l;\n\tcvt.rn.f16x2.e5m2x2 %1, h;\n\t}"
        : "=r"(v.x), "=r"(v.y)
        : "r"(w));
  return v;
}

// d += a (16 x 16) * b (16 x 8) of FP16, FP32 sums.
__device__ __forceinline__ void mma_half(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int ACode, int BCode>
__global__ void __launch_bounds__(kAnyThreads, 2) any_tiles_kernel(const gemm_params p) {
  constexpr int kWarps = kAnyThreads / 32, kRows = (kAnyN + kAnyM) / kWarps; // of a warp
  extern __shared__ __align__(16) unsigned char shared[];
  any_tile &tile = *reinterpret_cast<any_tile *>(shared);
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int g = lane >> 2, t = lane & 3;
  const int rows_n = warp % 4 * 32, rows_m = kAnyN + warp / 4 * 32; // of the tile
  const uint32_t blocks = static_cast<uint32_t>((p.k + kBlock - 1) / kBlock);
  const uint64_t groups = (p.n + kAnyN - 1) / kAnyN;
  const uint64_t tasks = groups * ((p.m + kAnyM - 1) / kAnyM);
  for (uint64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const uint64_t n0 = task % groups * kAnyN, m0 = task / groups * kAnyM;
    const uint32_t n_left = static_cast<uint32_t>(min(p.n - n0, uint64_t{kAnyN}));
    const uint32_t m_left = static_cast<uint32_t>(min(p.m - m0, uint64_t{kAnyM}));
    const uint8_t *b0 = p.b + n0 * p.b_stride, *a0 = p.a + m0 * p.a_stride;
    // the tile's rows; beyond the matrices the last one, whose products are not stored
    if (threadIdx.x < kAnyN)
      tile.rows[threadIdx.x] = b0 + min(threadIdx.x, n_left - 1) * p.b_stride;
    else if (threadIdx.x < kAnyN + kAnyM)
      tile.rows[threadIdx.x] = a0 + min(threadIdx.x - kAnyN, m_left - 1) * p.a_stride;
    __syncthreads();
    uint32_t word[kRows], last = 0; // lane r < kRows: the 33rd word of row r
    float scale = 0.0f;
    auto fetch = [&](uint32_t block) {
      const uint64_t c = uint64_t{block} * kBlock;
      if (c != 0 && c + kBlock + 4 <= p.k) { // all the words lie in the row
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const uintptr_t at = reinterpret_cast<uintptr_t>(tile.rows[r * kWarps + warp] + c);
          word[r] = __ldg(reinterpret_cast<const uint32_t *>(at & ~uintptr_t{3}) + lane);
        }
        if (lane < kRows) {
          const uintptr_t at = reinterpret_cast<uintptr_t>(tile.rows[lane * kWarps + warp] + c);
          last = __ldg(reinterpret_cast<const uint32_t *>(at & ~uintptr_t{3}) + 32);
        }
      } else {
        // the words that lie in the row, then the ones that its ends cut: lane r
        // puts those of row r together
        const int64_t k = static_cast<int64_t>(p.k), first = static_cast<int64_t>(c);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const uint8_t *row = tile.rows[r * kWarps + warp];
          const int64_t at = first - offset_in_word(row) + 4 * lane;
          word[r] = at >= 0 && at + 4 <= k ? __ldg(reinterpret_cast<const uint32_t *>(row + at)) : 0u;
        }
        uint32_t head = 0, tail = 0;
        int head_lane = -1, tail_lane = -1;
        if (lane < kRows) {
          const uint8_t *row = tile.rows[lane * kWarps + warp];
          const int s = offset_in_word(row);
          if (first == 0 && s != 0) head = load_word(row, -s, k), head_lane = 0;
          const int64_t cut = (k + s) / 4 * 4 - s; // the word with the row's end
          if (cut < k && cut >= 0) tail = load_word(row, cut, k);
          if (cut < k && cut >= 0 && cut < first + kBlock - s)
            tail_lane = static_cast<int>((cut - first + s) / 4);
          last = load_word(row, first - s + kBlock, k);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const uint32_t h = __shfl_sync(0xffffffffu, head, r), e = __shfl_sync(0xffffffffu, tail, r);
          const int h_lane = __shfl_sync(0xffffffffu, head_lane, r);
          const int e_lane = __shfl_sync(0xffffffffu, tail_lane, r);
          word[r] = lane == e_lane ? e : lane == h_lane ? h : word[r];
        }
      }
      if (threadIdx.x < m_left) scale = p.a_scales[block * p.a_scale_stride + m0 + threadIdx.x];
    };
    float acc[2][4][4] = {};
    if (blocks != 0) fetch(0);
    for (uint32_t block = 0; block < blocks; ++block) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int at = r * kWarps + warp;
        const uint32_t after = __shfl_down_sync(0xffffffffu, word[r], 1);
        const uint32_t end = __shfl_sync(0xffffffffu, last, r);
        const uint32_t w = __funnelshift_r(word[r], lane == 31 ? end : after,
                                           8 * offset_in_word(tile.rows[at]));
        reinterpret_cast<uint2 *>(&tile.values[at][lane / 2 ^ (at & 1) << 2])[lane % 2] =
            r < kAnyN / kWarps ? widen_codes<BCode>(w) : widen_codes<ACode>(w);
      }
      if (threadIdx.x < kAnyM) tile.scales[threadIdx.x] = scale;
      __syncthreads();
      if (block + 1 < blocks) fetch(block + 1);
      const float column = p.b_scales[block * p.b_scale_stride + n0 / kBlock];
      float d[2][4][4] = {};
#pragma unroll
      for (int part = 0; part < 4; ++part) {
        const int chunk = (4 * part + t) ^ (g & 1) << 2; // all row offsets are even
        uint4 u[2][2], w[4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) u[r][h] = tile.values[rows_n + 16 * r + 8 * h + g][chunk];
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = tile.values[rows_m + 8 * x + g][chunk];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint4 lo = u[r][0], hi = u[r][1];
            mma_half(d[r][x], lo.x, hi.x, lo.y, hi.y, w[x].x, w[x].y);
            mma_half(d[r][x], lo.z, hi.z, lo.w, hi.w, w[x].z, w[x].w);
          }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float *s = tile.scales + rows_m - kAnyN + 8 * x + 2 * t;
        const float s0 = s[0] * column, s1 = s[1] * column;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          acc[r][x][0] = fmaf(d[r][x][0], s0, acc[r][x][0]);
          acc[r][x][1] = fmaf(d[r][x][1], s1, acc[r][x][1]);
          acc[r][x][2] = fmaf(d[r][x][2], s0, acc[r][x][2]);
          acc[r][x][3] = fmaf(d[r][x][3], s1, acc[r][x][3]);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          tile.out[rows_m - kAnyN + 8 * x + 2 * t + e % 2][rows_n + 16 * r + 8 * (e / 2) + g] =
              acc[r][x][e];
    __syncthreads();
    for (int at = threadIdx.x; at < kAnyM * kAnyN; at += kAnyThreads) {
      const int i = at / kAnyN, j = at % kAnyN;
      if (m0 + i < p.m && n0 + j < p.n) store_out(p, m0 + i, n0 + j, tile.out[i][j]);
    }
    __syncthreads();
  }
}

// ---- few rows of a -----------------------------------------------------------------
// The product reads b once and computes little: what counts is how many bytes
// are under way.  A thread block computes 16 rows of b against all rows of a
// (8 T); its eight warps, or those of a cluster of Parts blocks, share the blocks
// of k, kAhead at a time, all of whose loads are issued before the first product.  Measured (m x n x k, GB/s of
// codes): 1 x 4096 x 4096 with kAhead 1, 2, 3, 4: 3387, 3640, 2963, 2729;
// 8 x 8192 x 8192: 3763, 4364, 4063, 4004 (registers: fewer blocks to an SM);
// keeping the next kAhead blocks' loads under way behind each product: 4181.  (b
// partly in the second-level cache; from memory 1 x 4096 x 4096 takes 4.6 us, 3.7
// TB/s, and 8 x 8192 x 8192 15.9.)  For 9 to 16 rows 12 to 40 bytes a thread spill.

// 32 codes of a row, in one load or two.  Measured with three b in turn, one load
// against two: faster for b below 2^25 codes, which stays in the second-level cache
// (8 x 2048 x 2048 1.96 and 2.14 us, 8 x 4096 x 4096 4.02 and 4.60, 8 x 1024 x 16384
// 5.03 and 5.60), slower where part of a larger one does (8 x 8192 x 8192 15.7 and
// 14.9, 1 x 16384 x 8192 26.8 and 25.9).  With b read from memory every time, one
// load is as fast or faster at all sizes up to 8 rows (1 x 4096 x 4096 4.56 and 4.72,
// 8 x 8192 x 8192 15.4 and 15.9, 1 x 28672 x 4096 22.5 and 25.1; 16 x 4096 x 8192
// 12.4 and 12.1).
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

template <int ACode, int BCode, int T, bool Wide, int Parts>
__global__ void __launch_bounds__(256, 2) stream_kernel(const gemm_params p) {
  constexpr int kAhead = T == 1 ? 2 : 1;
  __shared__ float sums[8][16][8 * T];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t rank = blockIdx.x % Parts;
  const uint64_t n0 = uint64_t{blockIdx.x / Parts} * 16;
  // this one of the warps that share the blocks of k
  constexpr uint32_t sharers = 8 * Parts;
  const uint32_t own = rank * 8 + warp;
  // A hint for the second-level cache, which is coherent, so it may come before
  // the kernels before this one have ended (1 x 4096 x 4096: 6.1 -> 4.6 us with
  // launches one behind the other): each lane's line of its two rows' blocks
  // own, own + sharers and so on.
  const uint64_t ahead = (uint64_t{own} + sharers * t) * kBlock;
  if (ahead < p.k)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (n0 + 8 * h + g < p.n)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.b + (n0 + 8 * h + g) * p.b_stride + ahead));
  aut::dev::pdl_wait();
  aut::dev::pdl_release();
  const uint32_t blocks = static_cast<uint32_t>((p.k + kBlock - 1) / kBlock);
  const uint32_t whole = static_cast<uint32_t>(p.k / kBlock);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint8_t *b[2], *a[T]; // lane (g, t): the codes from 32 t of a block
  bool has_b[2], has_a[T];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint64_t row = n0 + 8 * h + g;
    has_b[h] = row < p.n;
    b[h] = p.b + (has_b[h] ? row : 0) * p.b_stride + 32 * t;
  }
#pragma unroll
  for (int i = 0; i < T; ++i) {
    const uint64_t row = 8 * i + g;
    has_a[i] = row < p.m;
    a[i] = p.a + (has_a[i] ? row : 0) * p.a_stride + 32 * t;
  }
  float acc[T][4] = {};
  for (uint32_t first = own; first < whole; first += sharers * kAhead) {
    uint4 u[kAhead][2][2], w[kAhead][T][2];
    float s[kAhead][T][2], column[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint32_t block = first + sharers * i;
      const uint64_t c = uint64_t{block} * kBlock;
      const bool in = block < whole;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u[i][h][0] = u[i][h][1] = zero;
        if (in && has_b[h]) stream_load<Wide>(b[h] + c, u[i][h][0], u[i][h][1]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int x = 0; x < T; ++x)
          w[i][x][half] = in && has_a[x]
                              ? __ldg(reinterpret_cast<const uint4 *>(a[x] + c + 16 * half))
                              : zero;
      column[i] = in ? __ldg(p.b_scales + n0 / kBlock + block * p.b_scale_stride) : 0.0f;
#pragma unroll
      for (int x = 0; x < T; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          s[i][x][e] = in && 8 * x + 2 * t + e < p.m
                           ? __ldg(p.a_scales + block * p.a_scale_stride + 8 * x + 2 * t + e)
                           : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int x = 0; x < T; ++x) {
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint4 lo = u[i][0][half], hi = u[i][1][half], v = w[i][x][half];
          mma<BCode, ACode>(d, lo.x, hi.x, lo.y, hi.y, v.x, v.y);
          mma<BCode, ACode>(d, lo.z, hi.z, lo.w, hi.w, v.z, v.w);
        }
        const float s0 = s[i][x][0] * column[i], s1 = s[i][x][1] * column[i];
        acc[x][0] = fmaf(d[0], s0, acc[x][0]);
        acc[x][1] = fmaf(d[1], s1, acc[x][1]);
        acc[x][2] = fmaf(d[2], s0, acc[x][2]);
        acc[x][3] = fmaf(d[3], s1, acc[x][3]);
      }
  }
  // the last block, cut short by k
  if (whole < blocks && own == whole % sharers) {
    const float column = p.b_scales[whole * p.b_scale_stride + n0 / kBlock];
#pragma unroll
    for (int x = 0; x < T; ++x) {
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const uint64_t c = uint64_t{whole} * kBlock + 32 * t + 16 * half;
        const uint4 lo = has_b[0] ? load_end(b[0] - 32 * t, c, p.k) : zero;
        const uint4 hi = has_b[1] ? load_end(b[1] - 32 * t, c, p.k) : zero;
        const uint4 v = has_a[x] ? load_end(a[x] - 32 * t, c, p.k) : zero;
        mma<BCode, ACode>(d, lo.x, hi.x, lo.y, hi.y, v.x, v.y);
        mma<BCode, ACode>(d, lo.z, hi.z, lo.w, hi.w, v.z, v.w);
      }
      const float *s = p.a_scales + whole * p.a_scale_stride + 8 * x + 2 * t;
      const float s0 = 8 * x + 2 * t < p.m ? s[0] * column : 0.0f;
      const float s1 = 8 * x + 2 * t + 1 < p.m ? s[1] * column : 0.0f;
      acc[x][0] = fmaf(d[0], s0, acc[x][0]);
      acc[x][1] = fmaf(d[1], s1, acc[x][1]);
      acc[x][2] = fmaf(d[2], s0, acc[x][2]);
      acc[x][3] = fmaf(d[3], s1, acc[x][3]);
    }
  }
#pragma unroll
  for (int x = 0; x < T; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[warp][8 * (e / 2) + g][8 * x + 2 * t + e % 2] = acc[x][e];
  __syncthreads();
  if constexpr (Parts == 1) join_warps<16, 8 * T>(p, sums, 0, n0);
  else join_cluster<16, 8 * T, Parts>(p, sums, n0, rank);
}

template <class Params>
aut_status launch(void (*kernel)(Params), uint64_t grid, int max_grid, int threads,
                  const Params &p, cudaStream_t stream, size_t shared = 0, unsigned cluster = 1) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid < static_cast<uint64_t>(max_grid) ? grid : max_grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  AUT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return AUT_OK;
}

template <int ACode, int BCode, int T, bool Wide>
aut_status gemm_stream(const gemm_params &p, bool shared, cudaStream_t stream) {
  const uint64_t groups = (p.n + 15) / 16;
  return shared ? launch(stream_kernel<ACode, BCode, T, Wide, 4>, 4 * groups, 0x7fffffff, 256, p,
                         stream, 0, 4)
                : launch(stream_kernel<ACode, BCode, T, Wide, 1>, groups, 0x7fffffff, 256, p, stream);
}

template <int ACode, int BCode>
aut_status gemm_typed(aut_workspace *ws, const gemm_params &p, cudaStream_t stream) {
  // Measured (n = 4096, k = 4099): 32 rows take 73 us by the few rows' kernel,
  // 86 by tiles; 512 rows 1050 and 133.
  if (!aligned_operands(p, 16) && p.m > 32) {
    auto kernel = any_tiles_kernel<ACode, BCode>;
    AUT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      sizeof(any_tile)));
    return launch(kernel, (p.n + kAnyN - 1) / kAnyN * ((p.m + kAnyM - 1) / kAnyM),
                  64 * ws->max_blocks, kAnyThreads, p, stream, sizeof(any_tile));
  }
  if (!aligned_operands(p, 16) || p.k == 0)
    return launch(rows_kernel<ACode, BCode>, (p.n + 15) / 16 * ((p.m + 7) / 8),
                  64 * ws->max_blocks, 256, p, stream);
  const uint64_t groups = (p.n + 15) / 16, at_once = 2 * static_cast<uint64_t>(ws->sm_count);
  // Few rows of b and a long k: a cluster of four blocks shares k.  Measured: 1 x
  // 1024 x 16384 4.9 against 7.0 us, 16 x 1024 x 8192 4.9 against 6.5; 8 x 1024 x
  // 4096 3.4 against 2.8.
  const bool shared = 4 * groups <= at_once && p.k >= 64 * kBlock;
  // Measured: up to 8 rows streaming is faster than tiles (8 x 8192 x 8192: 15.0
  // against 16.4 us, 1 x 4096 x 4096: 4.1 against 6.8); up to 16 it is where all
  // of b goes through at once and k is not long (16 x 4096 x 4096: 5.7 against 7.1
  // us, 10 x 2048 x 8192 6.4 against 8.6; 16 x 16384 x 1024 8.3 against 5.5, 10 x
  // 2048 x 16000 16.6 against 11.0).
  if (p.m > 16 || (p.m > 8 && !shared && (groups > at_once || p.k > 64 * kBlock)))
    return gemm_tiles(ws, p, ACode, BCode, stream);
  const bool wide = aligned_operands(p, 32) && p.n * p.k < uint64_t{1} << 25;
  if (p.m <= 8)
    return wide ? gemm_stream<ACode, BCode, 1, true>(p, shared, stream)
                : gemm_stream<ACode, BCode, 1, false>(p, shared, stream);
  return wide ? gemm_stream<ACode, BCode, 2, true>(p, shared, stream)
              : gemm_stream<ACode, BCode, 2, false>(p, shared, stream);
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

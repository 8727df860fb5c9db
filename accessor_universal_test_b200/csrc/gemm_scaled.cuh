// gemm_scaled.cuh -- what the kernels of aut_gemm_scaled share.
#ifndef AUT_GEMM_SCALED_CUH_
#define AUT_GEMM_SCALED_CUH_

#include "internal.hpp"
#include "dot_device.cuh"
#include "scaled_device.cuh"

namespace aut::scaled {

struct gemm_params {
  const uint8_t *a; // m rows of k codes, one scale per row and 128 columns
  const uint8_t *b; // n rows of k codes, one scale per 128 rows and 128 columns
  const float *a_scales, *b_scales;
  void *out;
  uint64_t a_stride, b_stride, a_scale_stride, b_scale_stride, out_stride;
  uint64_t m, n, k;
  int type;
};

__device__ __forceinline__ void store_out(const gemm_params &p, uint64_t i, uint64_t j, float v) {
  const uint64_t at = i * p.out_stride + j;
  if (p.type == AUT_TYPE_FP32) static_cast<float *>(p.out)[at] = v;
  else if (p.type == AUT_TYPE_BF16)
    static_cast<__nv_bfloat16 *>(p.out)[at] = narrow<__nv_bfloat16>(v);
  else static_cast<__half *>(p.out)[at] = narrow<__half>(v);
}

// Of all threads of the cluster's blocks.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
               "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// What stands at p in the shared memory of the cluster's block `rank`.
__device__ __forceinline__ float cluster_load(const float *p, uint32_t rank) {
  uint32_t a;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(a)
      : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// Whether every row of both operands starts on a boundary of `bytes`.
inline bool aligned_operands(const gemm_params &p, uint64_t bytes) {
  return reinterpret_cast<uintptr_t>(p.a) % bytes == 0 && (p.m == 1 || p.a_stride % bytes == 0) &&
         reinterpret_cast<uintptr_t>(p.b) % bytes == 0 && (p.n == 1 || p.b_stride % bytes == 0);
}

// The tensor-core path over tensor memory (gemm_scaled_tc.cu).
aut_status gemm_tiles(aut_workspace *ws, const gemm_params &p, int a_code, int b_code,
                      cudaStream_t stream);

} // namespace aut::scaled

#endif

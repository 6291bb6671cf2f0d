// Shared helpers of the layer-stack kernels (sm_100a): element types, warp and
// block sums, the sticky device error word (one per source file that uses it).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace nnue_ls {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kNumSMs = 148;

// Sticky flags raised by kernels instead of hanging or faulting.
static __device__ unsigned int g_device_errors = 0;
enum : unsigned {
  kErrWaitTimeout = 1u,  // a matrix kernel's wait on its own copies or products ran out
  kErrBadIndex = 2u,     // route backward: a chosen index outside [-1, experts) was skipped
};
__device__ __forceinline__ void flag_error(unsigned e) { atomicOr(&g_device_errors, e); }

// Adds this file's word to *flags; clears it on demand.  Synchronises.
static inline cudaError_t read_device_errors(unsigned* flags, bool clear) {
  unsigned v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_device_errors, sizeof(v));
  *flags |= v;
  const unsigned zero = 0;
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(g_device_errors, &zero, sizeof(zero));
  return e;
}

using bf16 = __nv_bfloat16;
using f16 = __half;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<f16>(f16 v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ f16 from_f<f16>(float v) { return __float2half_rn(v); }

// A value stored either as fp32 or as T (parameters and row gates may be kept
// in 32 bits beside 16-bit activations).
template <typename T>
__device__ __forceinline__ float load_mixed(const void* p, int64_t i, bool is_f32) {
  return is_f32 ? __ldg(static_cast<const float*>(p) + i) : to_f(static_cast<const T*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void store_mixed(void* p, int64_t i, bool is_f32, float v) {
  if (is_f32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = from_f<T>(v);
}

// 1 / (1 + exp(-v)) to about three units at any v: with e = exp(-|v|) the sum lies in [1, 2], where the short reciprocal
// (one unit) needs neither a division's slow path nor care for subnormal results.  fp32 65536 x 1040, elementwise gate,
// layer norm forward: 260 us; with a division 305, with the short exponential, whose error grows with |v|, 246.
__device__ __forceinline__ float logistic(float v) {
  float r;
  const float e = expf(-fabsf(v));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return v < 0.f ? e * r : r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// Sums N values over the block; every thread gets the totals.  `scratch` holds
// 32 * N floats.  The order of the adds is fixed by the thread numbering.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  __syncthreads();  // the previous use of scratch is over
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) scratch[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? scratch[i * 32 + lane] : 0.f);
}

}  // namespace nnue_ls

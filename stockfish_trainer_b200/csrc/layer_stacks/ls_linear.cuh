// Fused linear layer: out = act(x W^T + b) + residual, and its gradients.
#pragma once

#include "ls_common.cuh"

namespace nnue_ls {

enum Activation : int { kNone = 0, kRelu = 1, kCrelu = 2, kSqrCrelu = 3, kSilu = 4, kGelu = 5, kActivations = 6 };

// act(z) and act'(z).  At the kinks of the clipped forms the derivative is 0,
// as in clamp's backward outside the open interval.
__device__ __forceinline__ float activate(float z, int act, float& d) {
  switch (act) {
    case kRelu: d = z > 0.f ? 1.f : 0.f; return z > 0.f || z != z ? z : 0.f;
    case kCrelu: d = z > 0.f && z < 1.f ? 1.f : 0.f; return z != z ? z : fminf(fmaxf(z, 0.f), 1.f);
    case kSqrCrelu: {
      const float c = z != z ? z : fminf(fmaxf(z, 0.f), 1.f);
      d = z > 0.f && z < 1.f ? 2.f * z : 0.f;
      return c * c;
    }
    case kSilu: {
      const float s = 1.f / (1.f + expf(-z));
      d = s * (1.f + z * (1.f - s));
      return z * s;
    }
    case kGelu: {
      const float phi = 0.5f * erfcf(-0.70710678118654752f * z);
      d = phi + z * (0.39894228040143268f * expf(-0.5f * z * z));
      return z * phi;
    }
    default: d = 1.f; return z;
  }
}

struct LinearEpilogue {
  const void* bias;
  const void* residual;
  void* out;
  void* act_grad;  // act'(z) in the tensors' type, [rows, outputs]; null when no gradient is wanted
  int64_t ldr, ldo;
  int act;
  bool bias_f32;
};

// C[m, n] = sum_k A[m, k] B[n, k] with any strides, fp32 accumulation: 64 x 64
// tiles through shared memory, 4 x 4 outputs per thread.
constexpr int kTile = 64, kTileK = 16;
template <typename T>
__global__ void __launch_bounds__(256) simple_gemm_kernel(const T* __restrict__ a, int64_t sam, int64_t sak,
                                                          const T* __restrict__ b, int64_t sbn, int64_t sbk, int64_t M,
                                                          int64_t N, int64_t K, LinearEpilogue e) {
  __shared__ float sa[kTileK][kTile + 1], sb[kTileK][kTile + 1];
  const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += kTileK) {
    for (int i = threadIdx.x; i < kTile * kTileK; i += 256) {
      const int kk = i & (kTileK - 1), r = i / kTileK;
      const int64_t k = k0 + kk;
      sa[kk][r] = m0 + r < M && k < K ? to_f(a[(m0 + r) * sam + k * sak]) : 0.f;
      sb[kk][r] = n0 + r < N && k < K ? to_f(b[(n0 + r) * sbn + k * sbk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kTileK; ++kk) {
      float va[4], vb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        va[i] = sa[kk][ty + 16 * i];
        vb[i] = sb[kk][tx + 16 * i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(va[i], vb[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (n >= N) continue;
      float z = acc[i][j], d;
      if (e.bias) z += load_mixed<T>(e.bias, n, e.bias_f32);
      float o = activate(z, e.act, d);
      if (e.residual) o += to_f(static_cast<const T*>(e.residual)[m * e.ldr + n]);
      static_cast<T*>(e.out)[m * e.ldo + n] = from_f<T>(o);
      if (e.act_grad) static_cast<T*>(e.act_grad)[m * N + n] = from_f<T>(d);
    }
  }
}

// dz = g * act'(z) (written when act_grad is given) and, per block, the column
// sums of dz over a range of rows.  blockDim = (32 columns, 8 rows).
template <typename T>
__global__ void __launch_bounds__(256) dz_bias_kernel(const T* __restrict__ g, int64_t ldg,
                                                      const T* __restrict__ act_grad, T* __restrict__ dz,
                                                      float* __restrict__ partial, int64_t M, int64_t N,
                                                      int64_t rows_per_block) {
  __shared__ float red[8][33];
  const int64_t n = (int64_t)blockIdx.x * 32 + threadIdx.x;
  const int64_t m0 = (int64_t)blockIdx.y * rows_per_block, m1 = min(M, m0 + rows_per_block);
  float sum = 0.f;
  if (n < N) {
    for (int64_t m = m0 + threadIdx.y; m < m1; m += 8) {
      float v = to_f(g[m * ldg + n]);
      if (act_grad) {
        v *= to_f(act_grad[m * N + n]);
        dz[m * N + n] = from_f<T>(v);
      }
      sum += v;
    }
  }
  if (!partial) return;
  red[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && n < N) {
    for (int i = 1; i < 8; ++i) sum += red[i][threadIdx.x];
    partial[(int64_t)blockIdx.y * N + n] = sum;
  }
}

// out[n] = sum over parts of partial[part, n], in part order within each of
// the block's 8 rows of threads.
template <typename T>
__global__ void __launch_bounds__(256) column_total_kernel(const float* __restrict__ partial, int64_t parts, int64_t N,
                                                           void* out, bool out_f32) {
  __shared__ float red[8][33];
  const int64_t n = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  if (n < N)
    for (int64_t p = threadIdx.y; p < parts; p += 8) sum += partial[p * N + n];
  red[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && n < N) {
    for (int i = 1; i < 8; ++i) sum += red[i][threadIdx.x];
    store_mixed<T>(out, n, out_f32, sum);
  }
}

}  // namespace nnue_ls

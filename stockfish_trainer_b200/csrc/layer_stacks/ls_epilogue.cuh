// What happens to a finished sum z before it leaves the chip:
//   out = act(z + bias) + residual,  and act'(z) for the backward.
#pragma once

#include "ls_common.cuh"

namespace nnue_ls {

enum Activation : int { kNone = 0, kRelu = 1, kCrelu = 2, kSqrCrelu = 3, kSilu = 4, kGelu = 5, kActivations = 6 };

// act(z) and act'(z).  At the kinks of the clipped forms the derivative is 0,
// as in clamp's backward outside the open interval.
// For 16-bit results the short exponential (2^-21 relative) does.
template <typename T>
__device__ __forceinline__ float exponential(float v) { return sizeof(T) == 4 ? expf(v) : __expf(v); }

template <typename T>
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
      const float s = 1.f / (1.f + exponential<T>(-z));
      d = s * (1.f + z * (1.f - s));
      return z * s;
    }
    case kGelu: {
      const float phi = 0.5f * erfcf(-0.70710678118654752f * z);
      d = phi + z * (0.39894228040143268f * exponential<T>(-0.5f * z * z));
      return z * phi;
    }
    default: d = 1.f; return z;
  }
}

// act'(z) as it waits for the backward.  fp32 tensors keep it in fp32; 16-bit
// tensors as a 16-bit fixed-point number on [-1/7, 2.14] (every derivative here
// lies in [-0.13, 2]) with exact 0, 1 and 2 and steps of 3.5e-5: a bf16 or fp16
// value there would be a second rounding as large as the product's own.
template <typename T>
struct Derivative;
template <>
struct Derivative<float> {
  using Code = float;
  static __device__ __forceinline__ float encode(float d) { return d; }
  static __device__ __forceinline__ float decode(float c) { return c; }
};
template <>
struct Derivative<bf16> {
  using Code = uint16_t;
  static constexpr float kScale = 28672.f;
  static constexpr int kZero = 4096, kNan = 65535;
  static __device__ __forceinline__ uint16_t encode(float d) {
    return d != d ? kNan : (uint16_t)(__float2int_rn(d * kScale) + kZero);
  }
  static __device__ __forceinline__ float decode(uint16_t c) {
    return c == kNan ? __int_as_float(0x7fffffff) : (float)((int)c - kZero) * (1.f / kScale);
  }
};
template <>
struct Derivative<f16> : Derivative<bf16> {};

struct EpilogueParams {
  const void* bias;      // [N] or null
  const void* residual;  // [M, N] or null, row stride ldr
  void* out;             // [M, N], row stride N
  void* act_grad;        // Derivative<T>::Code [M, N], or null
  int64_t ldr;
  int32_t act;
  bool bias_f32;
  bool vec;  // out, residual, act_grad: 16-byte aligned rows
};

template <typename T>
struct alignas(16) Vec16 {
  T v[16 / sizeof(T)];
};

// Writes one 32 x 32 block of sums held in shared memory (row stride 33): rows
// m0.., columns n0.. below n1.  With `vec` four (16-bit) or eight (fp32)
// neighbouring lanes share a row and move 16 bytes each; else one lane per
// column.
template <typename T>
__device__ __forceinline__ void store_block(const float* stage, const EpilogueParams& e, int64_t m0, int64_t M,
                                            int64_t n0, int64_t n1, int64_t N, int lane) {
  using D = Derivative<T>;
  using Code = typename D::Code;
  if (e.vec) {
    constexpr int V = 16 / sizeof(T), kLanes = 32 / V, kRows = 32 / kLanes;
    const int c = (lane % kLanes) * V;
    const int64_t n = n0 + c;
    if (n >= n1) return;
    float bias[V];
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = e.bias ? load_mixed<T>(e.bias, n + i, e.bias_f32) : 0.f;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += kRows) {
      const int r = r0 + lane / kLanes;
      const int64_t m = m0 + r;
      if (m >= M) return;
      Vec16<T> res, out;
      Vec16<Code> d;
      if (e.residual) res = *reinterpret_cast<const Vec16<T>*>(static_cast<const T*>(e.residual) + m * e.ldr + n);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float dv, o = activate<T>(stage[r * 33 + c + i] + bias[i], e.act, dv);
        if (e.residual) o += to_f(res.v[i]);
        out.v[i] = from_f<T>(o);
        d.v[i] = D::encode(dv);
      }
      *reinterpret_cast<Vec16<T>*>(static_cast<T*>(e.out) + m * N + n) = out;
      if (e.act_grad) *reinterpret_cast<Vec16<Code>*>(static_cast<Code*>(e.act_grad) + m * N + n) = d;
    }
  } else {
    const int64_t n = n0 + lane;
    if (n >= n1) return;
    const float bias = e.bias ? load_mixed<T>(e.bias, n, e.bias_f32) : 0.f;
    for (int r = 0; r < 32 && m0 + r < M; ++r) {
      const int64_t m = m0 + r;
      float dv, o = activate<T>(stage[r * 33 + lane] + bias, e.act, dv);
      if (e.residual) o += to_f(static_cast<const T*>(e.residual)[m * e.ldr + n]);
      static_cast<T*>(e.out)[m * N + n] = from_f<T>(o);
      if (e.act_grad) static_cast<Code*>(e.act_grad)[m * N + n] = D::encode(dv);
    }
  }
}

// The raw sums of one piece of the k range.
__device__ __forceinline__ void store_partial(const float* stage, float* partial, int64_t m0, int64_t M, int64_t n0,
                                              int64_t n1, int64_t N, int lane) {
  const int64_t n = n0 + lane;
  if (n >= n1) return;
  for (int r = 0; r < 32 && m0 + r < M; ++r) partial[(m0 + r) * N + n] = stage[r * 33 + lane];
}

}  // namespace nnue_ls

// What happens to a finished sum z before it leaves the chip:
//   out = act(z + bias) + residual,  and act'(z) for the backward.
#pragma once

#include <type_traits>

#include "ls_common.cuh"

namespace nnue_ls {

enum Activation : int { kNone = 0, kRelu = 1, kCrelu = 2, kSqrCrelu = 3, kSilu = 4, kGelu = 5, kActivations = 6 };

// act(z) and act'(z).  A clamp passes the gradient on the closed interval, its
// bounds included, as the feature transformer's epilogue does; relu's is 0 at 0.
//
// gelu(z) = z Phi(z), Phi(z) = erfc(-z / sqrt 2) / 2.  For 16-bit results, with
// u = |z| / sqrt 2 and t = 1 / (1 + 0.45 u), erfc(u) = exp(-u^2) P(t): P is the
// polynomial of degree 6 without constant term whose largest relative error
// against exp(u^2) erfc(u) on u in [0, 14] is least (a linear program over its
// coefficients; 9.5e-6), so the lower tail keeps its digits too.  The
// exponential is the density's, needed for the derivative anyway.  fp32 results
// take erfcf and logistic: the short exponential's error grows with |z| (25 units
// at z = -20).
// The hardware's own reciprocal and power of two (2^-22 relative, subnormals
// flushed), for 16-bit results.
__device__ __forceinline__ float short_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float short_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

template <typename T, int ACT>
__device__ __forceinline__ float activate(float z, float& d) {
  constexpr bool kShort = sizeof(T) == 2;
  if constexpr (ACT == kRelu) {
    d = z > 0.f ? 1.f : 0.f;
    return z > 0.f || z != z ? z : 0.f;
  } else if constexpr (ACT == kCrelu || ACT == kSqrCrelu) {
    const float c = z != z ? z : fminf(fmaxf(z, 0.f), 1.f);
    const bool inside = z >= 0.f && z <= 1.f;
    d = inside ? (ACT == kCrelu ? 1.f : 2.f * z) : 0.f;
    return ACT == kCrelu ? c : c * c;
  } else if constexpr (ACT == kSilu) {
    const float s = kShort ? short_rcp(1.f + short_exp2(-1.44269504f * z)) : logistic(z);
    d = s * (1.f + z * (1.f - s));
    return z * s;
  } else if constexpr (ACT == kGelu) {
    float phi, bell;
    if constexpr (kShort) {
      const float t = short_rcp(fmaf(0.45f * 0.70710678f, fabsf(z), 1.f));
      bell = short_exp2(-0.72134752f * z * z);
      float p = fmaf(t, -0.135856772f, 0.292236458f);
      p = fmaf(t, p, 0.0894653538f);
      p = fmaf(t, p, 0.248474505f);
      p = fmaf(t, p, 0.251702836f);
      p = fmaf(t, p, 0.253968126f);
      const float tail = 0.5f * t * p * bell;
      phi = z < 0.f ? tail : 1.f - tail;
    } else {
      bell = expf(-0.5f * z * z);
      phi = 0.5f * erfcf(-0.70710678118654752f * z);
    }
    d = fmaf(z * 0.39894228040143268f, bell, phi);
    return z * phi;
  } else {
    d = 1.f;
    return z;
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
  // Adding 1.5 * 2^23 leaves the rounded integer in the low bits; a NaN result has them all set.
  static __device__ __forceinline__ uint16_t encode(float d) {
    return (uint16_t)__float_as_uint(fmaf(d, kScale, 12582912.f + kZero));
  }
  static __device__ __forceinline__ float decode(uint16_t c) {
    const float v = (__uint_as_float(0x4b000000u | c) - (8388608.f + kZero)) * (1.f / kScale);
    return c == kNan ? __int_as_float(0x7fffffff) : v;
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

template <typename T, int V>
struct alignas(sizeof(T) * V) VecT {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void round_all(const float (&v)[V], VecT<T, V>& out) {
  if constexpr (sizeof(T) == 2) {  // two per instruction
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      if constexpr (std::is_same<T, bf16>::value)
        *reinterpret_cast<__nv_bfloat162*>(&out.v[j]) = __floats2bfloat162_rn(v[j], v[j + 1]);
      else
        *reinterpret_cast<__half2*>(&out.v[j]) = __floats2half2_rn(v[j], v[j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) out.v[j] = v[j];
  }
}

// Calls fn with the activation as a constant.
template <typename F>
__device__ __forceinline__ void with_activation(int act, const F& fn) {
  switch (act) {
    case kRelu: fn(std::integral_constant<int, kRelu>{}); break;
    case kCrelu: fn(std::integral_constant<int, kCrelu>{}); break;
    case kSqrCrelu: fn(std::integral_constant<int, kSqrCrelu>{}); break;
    case kSilu: fn(std::integral_constant<int, kSilu>{}); break;
    case kGelu: fn(std::integral_constant<int, kGelu>{}); break;
    default: fn(std::integral_constant<int, kNone>{}); break;
  }
}

// A warp's 32 x 32 block of sums on its way from one row per lane to rows
// shared by neighbouring lanes: 16-byte pieces in shared memory, a row's
// pieces exchanged by the row's low bits so that neither side meets a bank
// twice.
struct Block32 {
  float4* s;
  __device__ __forceinline__ void put(const float (&v)[32], int lane) {
    __syncwarp();  // the previous block has been read
#pragma unroll
    for (int j = 0; j < 8; ++j)
      s[lane * 8 + (j ^ (lane & 7))] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    __syncwarp();
  }
  template <int V>
  __device__ __forceinline__ void get(int row, int col, float (&v)[V]) const {  // col: a multiple of V >= 4
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const float4 t = s[row * 8 + ((col / 4 + j) ^ (row & 7))];
      v[4 * j] = t.x, v[4 * j + 1] = t.y, v[4 * j + 2] = t.z, v[4 * j + 3] = t.w;
    }
  }
  __device__ __forceinline__ float get1(int row, int col) const {
    return reinterpret_cast<const float*>(s)[row * 32 + (((col >> 2) ^ (row & 7)) << 2) + (col & 3)];
  }
};

// One block's writer: the first `rows` rows from m0, columns n0.. below n1.
// With `vec` four (16-bit) or eight (fp32) neighbouring lanes share a row and
// move 16 bytes each; else one lane per column.  The first residual is asked
// for at construction, before the sums are waited for.
template <typename T>
struct BlockWriter {
  using D = Derivative<T>;
  using Code = typename D::Code;
  static constexpr int V = 16 / sizeof(T), kLanes = 32 / V, kRows = 32 / kLanes;
  const EpilogueParams& e;
  int64_t m0, n, N;
  int rows, lane, row, col;
  bool inside;
  VecT<T, V> first;

  __device__ __forceinline__ BlockWriter(const EpilogueParams& e_, int64_t m0_, int rows_, int64_t n0, int64_t n1,
                                         int64_t N_, int lane_)
      : e(e_), m0(m0_), N(N_), rows(rows_), lane(lane_) {
    row = e.vec ? lane / kLanes : 0;
    col = e.vec ? (lane % kLanes) * V : lane;
    n = n0 + col;
    inside = n < n1 && row < rows;
    if (e.vec && e.residual && inside)
      first = *reinterpret_cast<const VecT<T, V>*>(static_cast<const T*>(e.residual) + (m0 + row) * e.ldr + n);
  }

  template <int ACT, bool RES, bool GRAD>
  __device__ __forceinline__ void write_vec(const Block32& block) const {
    T* out_p = static_cast<T*>(e.out) + (m0 + row) * N + n;
    Code* grad_p = static_cast<Code*>(e.act_grad) + (m0 + row) * N + n;
    const T* res_p = static_cast<const T*>(e.residual) + (m0 + row) * e.ldr + n;
    VecT<T, V> next = first;
    float bias[V];
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = e.bias ? load_mixed<T>(e.bias, n + j, e.bias_f32) : 0.f;
#pragma unroll 1
    for (int r = row; r < rows; r += kRows) {
      const VecT<T, V> res = next;
      if (RES) {
        res_p += kRows * e.ldr;
        if (r + kRows < rows) next = *reinterpret_cast<const VecT<T, V>*>(res_p);  // one step ahead
      }
      float z[V];
      block.get<V>(r, col, z);
      VecT<T, V> out;
      VecT<Code, V> d;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float dv;
        z[j] = activate<T, ACT>(z[j] + bias[j], dv);
        if (RES) z[j] += to_f(res.v[j]);
        if (GRAD) d.v[j] = D::encode(dv);
      }
      round_all(z, out);
      *reinterpret_cast<VecT<T, V>*>(out_p) = out;
      out_p += kRows * N;
      if (GRAD) {
        *reinterpret_cast<VecT<Code, V>*>(grad_p) = d;
        grad_p += kRows * N;
      }
    }
  }

  template <int ACT>
  __device__ __forceinline__ void write_single(const Block32& block) const {
    const bool with_res = e.residual, with_grad = ACT != kNone && e.act_grad;
    const float bias = e.bias ? load_mixed<T>(e.bias, n, e.bias_f32) : 0.f;
    T* out_p = static_cast<T*>(e.out) + m0 * N + n;
    Code* grad_p = static_cast<Code*>(e.act_grad) + m0 * N + n;
    const T* res_p = static_cast<const T*>(e.residual) + m0 * e.ldr + n;
#pragma unroll 1
    for (int r = 0; r < rows; r += 4) {
      T res[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (with_res && r + i < rows) res[i] = res_p[i * e.ldr];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float dv, o = activate<T, ACT>(block.get1(r + i, lane) + bias, dv);
        if (with_res) o += to_f(res[i]);
        if (r + i < rows) {
          out_p[i * N] = from_f<T>(o);
          if (with_grad) grad_p[i * N] = D::encode(dv);
        }
      }
      out_p += 4 * N;
      grad_p += 4 * N;
      res_p += 4 * e.ldr;
    }
  }

  __device__ __forceinline__ void write(const Block32& block) const {
    if (!inside) return;
    with_activation(e.act, [&](auto a) {
      constexpr int ACT = decltype(a)::value;
      if (!e.vec) {
        write_single<ACT>(block);
      } else if (e.act_grad && ACT != kNone) {
        e.residual ? write_vec<ACT, true, ACT != kNone>(block) : write_vec<ACT, false, ACT != kNone>(block);
      } else {
        e.residual ? write_vec<ACT, true, false>(block) : write_vec<ACT, false, false>(block);
      }
    });
  }
};

// A block of the fp32 kernel, which holds running sums in registers: the
// parameters come from their copy in shared memory, which leaves it fewer spills
// than reading them as kernel parameters (65536 x 1040 x 1024, GELU and residual:
// 797 us against 829; as a call of its own 820).
static __device__ __forceinline__ void store_block_f32(float4* block, const EpilogueParams* shared, int64_t m0,
                                                       int rows, int64_t n0, int64_t n1, int64_t N, int lane) {
  const EpilogueParams e = *shared;
  BlockWriter<float>(e, m0, rows, n0, n1, N, lane).write(Block32{block});
}

// The raw sums of one piece of the k range; vec: N is a multiple of 4.
__device__ __forceinline__ void store_partial(const Block32& block, float* partial, bool vec, int64_t m0, int rows,
                                              int64_t n0, int64_t n1, int64_t N, int lane) {
  if (vec) {
    const int c = (lane & 7) * 4;
    if (n0 + c >= n1) return;
    float* out = partial + m0 * N + n0 + c;
#pragma unroll
    for (int r = lane >> 3; r < 32; r += 4) {
      float z[4];
      block.get<4>(r, c, z);
      if (r < rows) *reinterpret_cast<float4*>(out + r * N) = make_float4(z[0], z[1], z[2], z[3]);
    }
  } else {
    if (n0 + lane >= n1) return;
    float* out = partial + m0 * N + n0 + lane;
    for (int r = 0; r < rows; ++r) out[r * N] = block.get1(r, lane);
  }
}

}  // namespace nnue_ls

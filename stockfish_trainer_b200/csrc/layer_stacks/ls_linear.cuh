// The memory-bound passes around the linear layer's matrix products: operands
// brought into the products' layout, the output gradient times act'(z) with
// its column sums, the join of a product whose k range was cut into pieces.
#pragma once

#include "ls_common.cuh"
#include "ls_epilogue.cuh"

namespace nnue_ls {

// The three bf16 planes of V fp32 values: each takes what is left, rounded to
// its 8 bits, so their sum is the value.  Rounding to nearest, not cutting off:
// what is left then has either sign and half the size, so that the products of
// planes that are not formed (ls_gemm.cuh) lie below half a unit of the value's
// product and have either sign; cut off, they reached four units, all of one
// sign.  An infinity or NaN stays in the first plane, and a value that would
// round to infinity is cut off there.  bf16 has no steps below 2^-133: below
// 2^-110 (7.7e-34) the last plane is rounded to them and the sum is the value to
// 2^-134 only.
template <int V>
__device__ __forceinline__ void split_planes(const float (&v)[V], uint16_t (&q)[3][V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float r = v[i];
    const bool finite = (__float_as_uint(r) & 0x7f800000u) != 0x7f800000u;
    if (!finite) {
      q[0][i] = r != r ? 0x7fff : (uint16_t)(__float_as_uint(r) >> 16);
      q[1][i] = q[2][i] = 0;
      continue;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint16_t top = __bfloat16_as_ushort(__float2bfloat16_rn(r));
      if (k == 0 && (top & 0x7fff) == 0x7f80) top = (uint16_t)(__float_as_uint(r) >> 16);
      q[k][i] = top;
      r -= __uint_as_float((uint32_t)top << 16);
    }
  }
}

template <int V>
struct alignas(2 * V) Pack16 {
  uint16_t v[V];
};

// Stores V neighbouring values in the products' layout: T itself, or planes
// `plane` elements apart.
template <typename T, int V>
__device__ __forceinline__ void store_operand(void* dst, int64_t at, int64_t plane, const float (&v)[V]) {
  if constexpr (sizeof(T) == 4) {
    uint16_t q[3][V];
    split_planes(v, q);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      Pack16<V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) o.v[i] = q[k][i];
      *reinterpret_cast<Pack16<V>*>(static_cast<uint16_t*>(dst) + k * plane + at) = o;
    }
  } else {
    struct alignas(2 * V) Out {
      T v[V];
    } o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = from_f<T>(v[i]);
    *reinterpret_cast<Out*>(static_cast<T*>(dst) + at) = o;
  }
}

// Up to two matrices brought into the products' layout by one launch: [rows,
// cols] with row stride ld -> rows of ldo (a multiple of 8) values; a thread
// moves 8 values.  vec: rows start on 16-byte boundaries.
struct PackJob {
  const void* src;
  void* dst;
  int64_t ld, rows, cols, ldo;
  bool vec;
};
struct PackJobs {
  PackJob job[2];
  int64_t end[2];  // threads' work items up to each job's end
};
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const PackJobs jobs) {
  for (int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x; item < jobs.end[1]; item += (int64_t)gridDim.x * 256) {
    const bool second = item >= jobs.end[0];
    const PackJob& j = second ? jobs.job[1] : jobs.job[0];
    const int64_t i = second ? item - jobs.end[0] : item, groups = j.ldo / 8;
    const int64_t r = i / groups, c = (i - r * groups) * 8;
    const T* src = static_cast<const T*>(j.src) + r * j.ld + c;
    float v[8];
    if (j.vec && c + 8 <= j.cols) {
      constexpr int W = 16 / sizeof(T);
#pragma unroll
      for (int k = 0; k < 8; k += W) {
        const auto t = *reinterpret_cast<const VecT<T, W>*>(src + k);
#pragma unroll
        for (int q = 0; q < W; ++q) v[k + q] = to_f(t.v[q]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = c + k < j.cols ? to_f(src[k]) : 0.f;
    }
    store_operand<T, 8>(j.dst, r * j.ldo + c, j.rows * j.ldo, v);
  }
}

// Few rows (at most MT): a warp per output column reads that column's
// weights once, 16 bytes a lane (VEC), and keeps MT sums; x comes from the L1.
// Bound by the latency of one pass over W; a tensor-core tile would be nearly
// empty and its k range would have to be cut and joined in a second launch.
// 1 x 1040 x 256 fp32 takes 2.7 us, against 14.6 us in three launches on tiles.
template <typename T, int MT, bool VEC>
__global__ void __launch_bounds__(256) few_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w,
                                                       int64_t ldw, int M, int64_t N, int64_t K,
                                                       const EpilogueParams e) {
  using D = Derivative<T>;
  constexpr int V = VEC ? 16 / sizeof(T) : 1;
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= N) return;
  float acc[MT] = {};
#pragma unroll 2
  for (int64_t k = lane * V; k < K; k += 32 * V) {
    const auto wv = *reinterpret_cast<const VecT<T, V>*>(w + n * ldw + k);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m < M) {
        const auto xv = *reinterpret_cast<const VecT<T, V>*>(x + m * ldx + k);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[m] = fmaf(to_f(xv.v[j]), to_f(wv.v[j]), acc[m]);
      }
    }
  }
  // each step halves the rows a lane carries; in the end lane l holds row l / (32 / MT)
  int o = 16;
#pragma unroll
  for (int c = MT; c > 1; c /= 2) {
#pragma unroll
    for (int i = 0; i < c / 2; ++i) {
      const bool upper = lane & o;
      const float send = upper ? acc[i] : acc[i + c / 2], keep = upper ? acc[i + c / 2] : acc[i];
      acc[i] = keep + __shfl_xor_sync(kFull, send, o);
    }
    o /= 2;
  }
  float z = acc[0];
  for (; o > 0; o /= 2) z += __shfl_xor_sync(kFull, z, o);
  constexpr int kSpan = 32 / MT;
  const int m = lane / kSpan;
  if (lane % kSpan || m >= M) return;
  if (e.bias) z += load_mixed<T>(e.bias, n, e.bias_f32);
  with_activation(e.act, [&](auto act) {
    float d, out = activate<T, decltype(act)::value>(z, d);
    if (e.residual) out += to_f(static_cast<const T*>(e.residual)[m * e.ldr + n]);
    static_cast<T*>(e.out)[m * N + n] = from_f<T>(out);
    if (e.act_grad) static_cast<typename D::Code*>(e.act_grad)[m * N + n] = D::encode(d);
  });
}

// dz = g * act'(z), written in the products' layout when dst is given, and per
// block the fp32 column sums of the unrounded dz over a range of rows: into
// `partial`, or where one block is high enough for all rows, rounded into
// `total`.
// A block is `tx` groups of V columns wide and 256 / tx rows high (its last few
// threads may have nothing to do).
template <typename T, int V>
__global__ void __launch_bounds__(256) dz_kernel(const T* __restrict__ g, int64_t ldg,
                                                 const typename Derivative<T>::Code* __restrict__ act_grad,
                                                 void* __restrict__ dst, int64_t ldo, float* __restrict__ partial,
                                                 void* __restrict__ total, bool total_f32, int64_t M, int64_t N,
                                                 int64_t rows_per_block, int tx) {
  using D = Derivative<T>;
  using Code = typename D::Code;
  __shared__ float red[256 * V];
  const int x = threadIdx.x % tx, y = threadIdx.x / tx, ty = 256 / tx;
  const int64_t n = ((int64_t)blockIdx.x * tx + x) * V;
  const int64_t m1 = min(M, ((int64_t)blockIdx.y + 1) * rows_per_block);
  float sum[V] = {};
  if (n < N && y < ty) {
#pragma unroll 4
    for (int64_t m = (int64_t)blockIdx.y * rows_per_block + y; m < m1; m += ty) {
      const auto t = *reinterpret_cast<const VecT<T, V>*>(g + m * ldg + n);
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = to_f(t.v[i]);
      if (act_grad) {
        const auto d = *reinterpret_cast<const VecT<Code, V>*>(act_grad + m * N + n);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= D::decode(d.v[i]);
      }
      if (dst) store_operand<T, V>(dst, m * ldo + n, M * ldo, v);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += v[i];
    }
  }
  if (!partial && !total) return;
#pragma unroll
  for (int i = 0; i < V; ++i) red[i * 256 + threadIdx.x] = sum[i];
  __syncthreads();
  if (y == 0 && n < N) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      for (int j = 1; j < ty; ++j) sum[i] += red[i * 256 + j * tx + x];
      if (total) store_mixed<T>(total, n + i, total_f32, sum[i]);
      else partial[(int64_t)blockIdx.y * N + n + i] = sum[i];
    }
  }
}

// out[n] = sum over parts of partial[part, n], in a fixed order: 8 rows of
// threads take every eighth part, then their sums are added in turn.
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

// z = sum over pieces, in piece order, then the epilogue.  VEC: N is a multiple
// of 4 and rows are aligned; a thread takes 4 columns.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ partial, int splits, int64_t M, int64_t N,
                                                   EpilogueParams e) {
  using D = Derivative<T>;
  using Code = typename D::Code;
  constexpr int V = VEC ? 4 : 1;
  const int64_t groups = N / V, total = M * groups, MN = M * N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / groups, n = (i - m * groups) * V;
    float z[V] = {};
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
      const auto t = *reinterpret_cast<const VecT<float, V>*>(partial + s * MN + m * N + n);
#pragma unroll
      for (int j = 0; j < V; ++j) z[j] += t.v[j];
    }
    VecT<T, V> out, res;
    VecT<Code, V> d;
    if (e.residual) res = *reinterpret_cast<const VecT<T, V>*>(static_cast<const T*>(e.residual) + m * e.ldr + n);
    with_activation(e.act, [&](auto act) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (e.bias) z[j] += load_mixed<T>(e.bias, n + j, e.bias_f32);
        float dv, o = activate<T, decltype(act)::value>(z[j], dv);
        if (e.residual) o += to_f(res.v[j]);
        out.v[j] = from_f<T>(o);
        d.v[j] = D::encode(dv);
      }
    });
    *reinterpret_cast<VecT<T, V>*>(static_cast<T*>(e.out) + m * N + n) = out;
    if (e.act_grad) *reinterpret_cast<VecT<Code, V>*>(static_cast<Code*>(e.act_grad) + m * N + n) = d;
  }
}

}  // namespace nnue_ls

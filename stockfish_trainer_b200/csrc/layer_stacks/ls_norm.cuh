// Norms before and after a residual block, fused with the block's gate and
// residual scale:
//   n = norm(f) * post_weight + post_bias        (the norm after the block)
//   y = scale * x + gate * n                     (gate: none, one per row, or elementwise; through a sigmoid or not)
//   h = norm(y) * pre_weight + pre_bias          (the norm before the next block)
// norm(v) = (v - m) / sqrt(mean((v - m)^2) + eps), m = mean(v) for layer norm
// and 0 for rms norm.  Without f: y = x.  Without post_weight: n = f.
#pragma once

#include "ls_common.cuh"

namespace nnue_ls {

enum GateMode : int { kGateNone = 0, kGateRow = 1, kGateFull = 2 };

struct NormParams {
  const void *x, *f, *gate;
  const void *post_weight, *post_bias, *scale, *pre_weight, *pre_bias;  // [width]; null = absent
  void *y, *h;
  float4* stats;  // per row: mean and 1/std of f, mean and 1/std of y
  const void *grad_y, *grad_h;
  void *grad_x, *grad_f, *grad_gate;
  float* partial;  // backward: [blocks, 5, width] column sums (post_weight, post_bias, scale, pre_weight, pre_bias)
  int64_t rows;
  int width;
  float scale_value, eps;
  int gate_mode;
  bool gate_sigmoid, gate_f32, params_f32;
};

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + expf(-v)); }

// One row of the forward's inputs, element by element; used by every pass.
template <typename T>
struct NormRow {
  const NormParams& p;
  const T *x, *f, *g;
  float row_gate, mean_f, rstd_f;
  __device__ NormRow(const NormParams& p_, int64_t row) : p(p_), mean_f(0.f), rstd_f(1.f) {
    x = static_cast<const T*>(p.x) + row * p.width;
    f = static_cast<const T*>(p.f) + (p.f ? row * p.width : 0);
    g = static_cast<const T*>(p.gate) + (p.gate_mode == kGateFull ? row * p.width : 0);
    row_gate = 1.f;
    if (p.gate_mode == kGateRow) {
      row_gate = load_mixed<T>(p.gate, row, p.gate_f32);
      if (p.gate_sigmoid) row_gate = sigmoid(row_gate);
    }
  }
  __device__ float param(const void* v, int c) const { return load_mixed<T>(v, c, p.params_f32); }
  __device__ float scale(int c) const { return p.scale ? param(p.scale, c) : p.scale_value; }
  __device__ float gate(int c) const {
    if (p.gate_mode != kGateFull) return row_gate;
    const float v = to_f(g[c]);
    return p.gate_sigmoid ? sigmoid(v) : v;
  }
  __device__ float f_hat(int c) const { return (to_f(f[c]) - mean_f) * rstd_f; }
  __device__ float branch(int c) const {
    if (!p.post_weight) return to_f(f[c]);
    float n = f_hat(c) * param(p.post_weight, c);
    return p.post_bias ? n + param(p.post_bias, c) : n;
  }
  __device__ float y(int c) const {
    const float v = to_f(x[c]);
    return p.f ? scale(c) * v + gate(c) * branch(c) : v;
  }
};

// Mean (layer norm) and 1/std of a row whose element c is value(c).
template <bool CENTER, typename F>
__device__ __forceinline__ void row_stats(const F& value, int width, float eps, float* scratch, float& mean,
                                          float& rstd) {
  float v[1];
  mean = 0.f;
  if (CENTER) {
    v[0] = 0.f;
    for (int c = threadIdx.x; c < width; c += blockDim.x) v[0] += value(c);
    block_sum(v, scratch);
    mean = v[0] / width;
  }
  v[0] = 0.f;
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    const float d = value(c) - mean;
    v[0] += d * d;
  }
  block_sum(v, scratch);
  rstd = rsqrtf(v[0] / width + eps);
}

// One block per row, any width; the row is read again for each pass.
template <typename T, bool CENTER>
__global__ void __launch_bounds__(256) norm_forward_kernel(NormParams p) {
  __shared__ float scratch[32];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    NormRow<T> r(p, row);
    float mean_y = 0.f, rstd_y = 1.f;
    if (p.f && p.post_weight)
      row_stats<CENTER>([&](int c) { return to_f(r.f[c]); }, p.width, p.eps, scratch, r.mean_f, r.rstd_f);
    if (p.pre_weight) row_stats<CENTER>([&](int c) { return r.y(c); }, p.width, p.eps, scratch, mean_y, rstd_y);
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      const float y = r.y(c);
      if (p.y) static_cast<T*>(p.y)[row * p.width + c] = from_f<T>(y);
      if (p.h) {
        float h = (y - mean_y) * rstd_y * r.param(p.pre_weight, c);
        if (p.pre_bias) h += r.param(p.pre_bias, c);
        static_cast<T*>(p.h)[row * p.width + c] = from_f<T>(h);
      }
    }
    if (p.stats && threadIdx.x == 0) p.stats[row] = make_float4(r.mean_f, r.rstd_f, mean_y, rstd_y);
  }
}

// With d = the gradient of y (its own plus the norm's before the next block):
//   d = dy + rstd_y * (u - mean(u) - y_hat * mean(u * y_hat)),  u = dh * pre_weight   (mean(u) for layer norm only)
//   dx = scale * d;  dgate = d * n (summed over the row for a row gate; times s(1-s) through a sigmoid)
//   df = rstd_f * (v - mean(v) - f_hat * mean(v * f_hat)),      v = gate * d * post_weight
// and, summed over rows: post_weight += gate * d * f_hat, post_bias += gate * d, scale += d * x,
// pre_weight += dh * y_hat, pre_bias += dh.
// y is formed again from x, f and the gate: x has to be read for the scale's gradient anyway, and the y that the
// forward wrote is rounded to 16 bits, which would show in the fp32 sums.
// Each block owns a slice of `partial` and each thread its columns of it.
template <typename T, bool CENTER>
__global__ void __launch_bounds__(256) norm_backward_kernel(NormParams p) {
  __shared__ float scratch[64];
  const int W = p.width;
  const float inv = 1.f / W;
  float* part = p.partial ? p.partial + (int64_t)blockIdx.x * 5 * W : nullptr;
  if (part)
    for (int c = threadIdx.x; c < 5 * W; c += blockDim.x) part[c] = 0.f;
  __syncthreads();
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    NormRow<T> r(p, row);
    const float4 st = p.stats[row];
    r.mean_f = st.x;
    r.rstd_f = st.y;
    const T* gy = static_cast<const T*>(p.grad_y) + (p.grad_y ? row * W : 0);
    const T* gh = static_cast<const T*>(p.grad_h) + (p.grad_h ? row * W : 0);
    const bool pre = p.grad_h && p.pre_weight;
    auto y_hat = [&](int c) { return (r.y(c) - st.z) * st.w; };
    float s[2] = {0.f, 0.f};
    if (pre) {
      for (int c = threadIdx.x; c < W; c += blockDim.x) {
        const float u = to_f(gh[c]) * r.param(p.pre_weight, c);
        s[0] += u * y_hat(c);
        if (CENTER) s[1] += u;
      }
      block_sum(s, scratch);
    }
    const float c1 = s[0] * inv, c2 = s[1] * inv;
    auto d_of = [&](int c) {
      float d = p.grad_y ? to_f(gy[c]) : 0.f;
      if (pre) {
        const float u = to_f(gh[c]) * r.param(p.pre_weight, c);
        d += st.w * (u - c2 - y_hat(c) * c1);
      }
      return d;
    };
    float q[3] = {0.f, 0.f, 0.f};
    if (p.f) {
      for (int c = threadIdx.x; c < W; c += blockDim.x) {
        const float d = d_of(c);
        if (p.post_weight) {
          const float v = r.gate(c) * d * r.param(p.post_weight, c);
          q[0] += v * r.f_hat(c);
          if (CENTER) q[1] += v;
        }
        if (p.gate_mode == kGateRow) q[2] += d * r.branch(c);
      }
      float t[2] = {q[0], q[1]};
      block_sum(t, scratch);
      float t2[1] = {q[2]};
      block_sum(t2, scratch);
      q[0] = t[0];
      q[1] = t[1];
      q[2] = t2[0];
    }
    const float c3 = q[0] * inv, c4 = q[1] * inv;
    for (int c = threadIdx.x; c < W; c += blockDim.x) {
      const float d = d_of(c);
      const int64_t o = row * W + c;
      if (p.grad_x) static_cast<T*>(p.grad_x)[o] = from_f<T>(p.f ? r.scale(c) * d : d);
      float gn = 0.f;
      if (p.f) {
        const float gate = r.gate(c);
        gn = gate * d;
        if (p.grad_f) {
          float df = gn;
          if (p.post_weight) df = r.rstd_f * (gn * r.param(p.post_weight, c) - c4 - r.f_hat(c) * c3);
          static_cast<T*>(p.grad_f)[o] = from_f<T>(df);
        }
        if (p.grad_gate && p.gate_mode == kGateFull) {
          float dg = d * r.branch(c);
          if (p.gate_sigmoid) dg *= gate * (1.f - gate);
          static_cast<T*>(p.grad_gate)[o] = from_f<T>(dg);
        }
      }
      if (part) {
        if (p.f && p.post_weight) {
          part[c] += gn * r.f_hat(c);
          if (p.post_bias) part[W + c] += gn;
        }
        if (p.f && p.scale) part[2 * W + c] += d * to_f(r.x[c]);
        if (pre) {
          part[3 * W + c] += to_f(gh[c]) * y_hat(c);
          if (p.pre_bias) part[4 * W + c] += to_f(gh[c]);
        }
      }
    }
    if (p.grad_gate && p.gate_mode == kGateRow && threadIdx.x == 0) {
      float dg = q[2];
      if (p.gate_sigmoid) dg *= r.row_gate * (1.f - r.row_gate);
      store_mixed<T>(p.grad_gate, row, p.gate_f32, dg);
    }
  }
}

// Totals of the backward's column sums over blocks, in block order within each
// of a block's 8 rows of threads; out[i] null = not wanted.
struct NormTotals {
  void* out[5];
};
template <typename T>
__global__ void __launch_bounds__(256) norm_totals_kernel(const float* __restrict__ partial, int blocks, int width,
                                                          NormTotals t, bool out_f32) {
  __shared__ float red[8][33];
  const int which = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  if (!t.out[which]) return;
  float sum = 0.f;
  if (c < width)
    for (int b = threadIdx.y; b < blocks; b += 8) sum += partial[((int64_t)b * 5 + which) * width + c];
  red[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    for (int i = 1; i < 8; ++i) sum += red[i][threadIdx.x];
    store_mixed<T>(t.out[which], c, out_f32, sum);
  }
}

}  // namespace nnue_ls

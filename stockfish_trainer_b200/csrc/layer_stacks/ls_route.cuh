// Router of the layer stacks: softmax over the experts' logits, the k largest
// (ties to the lowest index) with their gates, per-expert counts and the
// balance loss
//   loss = E / (k n^2) * sum_e counts_e * sum_b p[b, e]
// over the n rows that count: rows marked valid with at least one logit other
// than -inf.  Rows that do not count have indices -1, gates 0 and no gradient.
#pragma once

#include "ls_common.cuh"

namespace nnue_ls {

constexpr int kMaxExperts = 1024;

struct RouteParams {
  const void* logits;     // [rows, experts], row stride ld
  const uint8_t* valid;   // [rows] or null
  int64_t* indices;       // [rows, k]
  float* gates;           // [rows, k]
  float* partial_p;       // [blocks, experts]
  int32_t* partial_count; // [blocks, experts + 1]; the last one counts the rows
  int64_t* counts;        // [experts]
  float* loss;            // the balance loss
  float* unit;            // E / (k n^2), kept for the backward
  const float* grad_gates;
  const float* grad_loss;
  void* grad_logits;
  int64_t rows, ld;
  int experts, k, blocks;
  bool renormalize;
};

// One warp's row: lane l holds experts l, l + 32, ...
template <typename T, int V>
struct RouteRow {
  float l[V], p[V];
  bool counts;
  __device__ __forceinline__ void load(const RouteParams& r, int64_t row, int lane) {
    const T* src = static_cast<const T*>(r.logits) + row * r.ld;
    const float ninf = __int_as_float(0xff800000);
    bool open = false;
    float m = ninf;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 32 * i;
      l[i] = e < r.experts ? to_f(src[e]) : ninf;
      open |= l[i] != ninf;
      m = fmaxf(m, l[i]);
    }
    counts = __any_sync(kFull, open) && (!r.valid || r.valid[row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    if (m == ninf) m = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = counts ? expf(l[i] - m) : 0.f;
      sum += p[i];
    }
    sum = warp_sum(sum);
    const float inv = counts ? 1.f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] *= inv;
  }
};

template <typename T, int V>
__global__ void __launch_bounds__(256) route_forward_kernel(RouteParams r) {
  __shared__ float sp[8][33];
  __shared__ int sc[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float ninf = __int_as_float(0xff800000);
  float total_p[V];
  int total_c[V], rows = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) total_p[i] = 0.f, total_c[i] = 0;
  for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < r.rows; row += (int64_t)gridDim.x * 8) {
    RouteRow<T, V> w;
    w.load(r, row, lane);
    rows += w.counts;
    float sum = 0.f, my_gate = 0.f;
    int my_index = -1;
#pragma unroll
    for (int i = 0; i < V; ++i) total_p[i] += w.p[i];
    for (int j = 0; j < r.k; ++j) {
      float best = ninf, prob = 0.f;
      int at = kMaxExperts;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (w.counts && w.l[i] > best) best = w.l[i], prob = w.p[i], at = lane + 32 * i;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float b = __shfl_xor_sync(kFull, best, o), q = __shfl_xor_sync(kFull, prob, o);
        const int a = __shfl_xor_sync(kFull, at, o);
        if (b > best || (b == best && a < at)) best = b, prob = q, at = a;
      }
      const bool taken = at < kMaxExperts;
      if (taken) sum += prob;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at == lane + 32 * i) total_c[i]++, w.l[i] = ninf;
      if (lane == (j & 31)) my_gate = prob, my_index = taken ? at : -1;
      if ((j & 31) == 31 || j == r.k - 1) {
        if (lane <= (j & 31)) {
          const int64_t o = row * r.k + (j & ~31) + lane;
          r.indices[o] = my_index;
          r.gates[o] = my_gate;
        }
      }
    }
    if (r.renormalize && sum != 0.f) {
      __syncwarp();
      for (int j = lane; j < r.k; j += 32) r.gates[row * r.k + j] /= sum;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    sp[warp][lane] = total_p[i];
    sc[warp][lane] = total_c[i];
    __syncthreads();
    if (warp == 0 && lane + 32 * i < r.experts) {
      float a = 0.f;
      int c = 0;
      for (int j = 0; j < 8; ++j) a += sp[j][lane], c += sc[j][lane];
      r.partial_p[(int64_t)blockIdx.x * r.experts + lane + 32 * i] = a;
      r.partial_count[(int64_t)blockIdx.x * (r.experts + 1) + lane + 32 * i] = c;
    }
    __syncthreads();
  }
  if (lane == 0) sc[warp][0] = rows;
  __syncthreads();
  if (threadIdx.x == 0) {
    int c = 0;
    for (int j = 0; j < 8; ++j) c += sc[j][0];
    r.partial_count[(int64_t)blockIdx.x * (r.experts + 1) + r.experts] = c;
  }
}

// One block: totals over the forward's blocks, then the loss.
__global__ void __launch_bounds__(256) route_totals_kernel(RouteParams r) {
  __shared__ float scratch[32];
  float part[1] = {0.f};
  for (int e = threadIdx.x; e < r.experts; e += blockDim.x) {
    float p = 0.f;
    int64_t c = 0;
    for (int b = 0; b < r.blocks; ++b) {
      p += r.partial_p[(int64_t)b * r.experts + e];
      c += r.partial_count[(int64_t)b * (r.experts + 1) + e];
    }
    r.counts[e] = c;
    part[0] += p * (float)c;
  }
  block_sum(part, scratch);
  if (threadIdx.x == 0) {
    int64_t n = 0;
    for (int b = 0; b < r.blocks; ++b) n += r.partial_count[(int64_t)b * (r.experts + 1) + r.experts];
    const float nf = (float)(n > 0 ? n : 1);
    const float unit = ((float)r.experts / (float)r.k / nf) / nf;
    *r.unit = unit;
    *r.loss = unit * part[0];
  }
}

// d logits = unit * dloss * p * (counts - sum_e counts_e p_e) + the gates' part:
// renormalised, on chosen entries g * (dg - sum g dg); else
// on chosen entries g * dg, and -p * sum g dg on all.
template <typename T, int V>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteParams r) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float c[V];
  const float coef = r.grad_loss ? *r.unit * *r.grad_loss : 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane + 32 * i;
    c[i] = e < r.experts ? (float)r.counts[e] * coef : 0.f;
  }
  for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < r.rows; row += (int64_t)gridDim.x * 8) {
    RouteRow<T, V> w;
    w.load(r, row, lane);
    float dot = 0.f, extra[V];
#pragma unroll
    for (int i = 0; i < V; ++i) dot += w.p[i] * c[i], extra[i] = 0.f;
    dot = warp_sum(dot);
    if (r.grad_gates && w.counts) {
      float inner = 0.f;
      for (int j = 0; j < r.k; ++j) {
        const int64_t o = row * r.k + j;
        if (r.indices[o] >= 0) inner += r.gates[o] * r.grad_gates[o];
      }
      for (int j = 0; j < r.k; ++j) {
        const int64_t o = row * r.k + j;
        const int64_t at = r.indices[o];
        if (at < 0) continue;
        if (at >= r.experts) {
          if (lane == 0) flag_error(kErrBadIndex);
          continue;
        }
        const float g = r.gates[o] * (r.grad_gates[o] - (r.renormalize ? inner : 0.f));
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (at == lane + 32 * i) extra[i] += g;
      }
      if (!r.renormalize) dot += inner;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 32 * i;
      if (e < r.experts)
        static_cast<T*>(r.grad_logits)[row * r.experts + e] = from_f<T>(w.counts ? w.p[i] * (c[i] - dot) + extra[i] : 0.f);
    }
  }
}

}  // namespace nnue_ls

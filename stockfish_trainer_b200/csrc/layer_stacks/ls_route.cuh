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
  bool vec, vec_out;      // rows of logits / grad_logits lie on 16-byte boundaries, whole 16-byte pieces
};

// A row belongs to G neighbouring lanes; lane g of them holds experts g * V ..
// g * V + V - 1.  What bounds this operator is latency: a row is a few dozen
// bytes, so small rows are packed 32 / G to a warp and every value stays in a
// register.
template <typename T, int V, int G>
struct RouteRow {
  float l[V], p[V];
  bool counts;

  static __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o /= 2) v += __shfl_xor_sync(kFull, v, o);
    return v;
  }
  // Every lane of the warp calls this; rows beyond the last do not count.
  __device__ __forceinline__ void load(const RouteParams& r, int64_t row, int g) {
    const float ninf = __int_as_float(0xff800000);
    const bool real = row < r.rows;
    const T* src = static_cast<const T*>(r.logits) + (real ? row : 0) * r.ld;
    bool open = false;
    float m = ninf;
    if (r.vec) {
      constexpr int W = 16 / sizeof(T) < V ? 16 / sizeof(T) : V;
      struct alignas(sizeof(T) * W) Vec {
        T v[W];
      };
#pragma unroll
      for (int i = 0; i < V; i += W) {
        const int e = g * V + i;
        if (real && e < r.experts) {  // a multiple of W of them
          const Vec t = *reinterpret_cast<const Vec*>(src + e);
#pragma unroll
          for (int j = 0; j < W; ++j) l[i + j] = to_f(t.v[j]);
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) l[i + j] = ninf;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = real && g * V + i < r.experts ? to_f(src[g * V + i]) : ninf;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      open |= l[i] != ninf;
      m = fmaxf(m, l[i]);
    }
    int any = open;
#pragma unroll
    for (int o = G / 2; o > 0; o /= 2) {
      m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
      any |= __shfl_xor_sync(kFull, any, o);
    }
    counts = any && (!r.valid || r.valid[row]);  // `any` implies a real row
    if (m == ninf) m = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = counts ? expf(l[i] - m) : 0.f;
      sum += p[i];
    }
    sum = group_sum(sum);
    const float inv = counts ? 1.f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] *= inv;
  }
};

// Warps of a forward block: their sums meet in shared memory.
__host__ __device__ constexpr int route_warps(int v, int g) { return v * g > 256 ? 4 : 8; }

// Totals over `parts` partial sums; then the loss.  One block, a part per warp
// and 32 experts at a time, parts in a fixed order.
__device__ __forceinline__ void route_totals(const RouteParams& r, int parts) {
  __shared__ float sp[32][33];
  __shared__ long long sc[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, rows = blockDim.x >> 5;
  float weighted = 0.f;  // thread y == 0: its experts' counts * p
  for (int e0 = 0; e0 < r.experts + 1; e0 += 32) {  // the last "expert" is the number of rows
    const int e = e0 + x;
    float p = 0.f;
    long long c = 0;
    if (e <= r.experts) {
#pragma unroll 10
      for (int b = y; b < parts; b += rows) {
        if (e < r.experts) p += r.partial_p[(int64_t)b * r.experts + e];
        c += r.partial_count[(int64_t)b * (r.experts + 1) + e];
      }
    }
    sp[y][x] = p;
    sc[y][x] = c;
    __syncthreads();
    if (y == 0) {
      for (int i = 1; i < rows; ++i) p += sp[i][x], c += sc[i][x];
      if (e < r.experts) {
        r.counts[e] = c;
        weighted += p * (float)c;
      }
      if (e == r.experts) sc[0][32] = c;
    }
    __syncthreads();
  }
  if (y == 0) {
    weighted = warp_sum(weighted);
    if (x == 0) {
      const long long n = sc[0][32];
      const float nf = (float)(n > 0 ? n : 1);
      const float unit = ((float)r.experts / (float)r.k / nf) / nf;
      *r.unit = unit;
      *r.loss = unit * weighted;
    }
  }
}

constexpr int kRouteKept = 8;  // choices whose gates wait in registers for their sum

template <typename T, int V, int G>
__global__ void __launch_bounds__(256) route_forward_kernel(const RouteParams r) {
  constexpr int kRows = 32 / G;  // rows per warp
  constexpr int kWarps = route_warps(V, G);
  __shared__ float sp[kWarps][V * G];
  __shared__ int sc[kWarps][V * G + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane % G;
  const float ninf = __int_as_float(0xff800000);
  float total_p[V];
  int total_c[V], rows = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) total_p[i] = 0.f, total_c[i] = 0;
  // whole warps take part in every step: the row of the warp's first lane decides
  for (int64_t first = ((int64_t)blockIdx.x * kWarps + warp) * kRows; first < r.rows;
       first += (int64_t)gridDim.x * kWarps * kRows) {
    const int64_t row = first + lane / G;
    RouteRow<T, V, G> w;
    w.load(r, row, g);
    if (g == 0) rows += w.counts;
#pragma unroll
    for (int i = 0; i < V; ++i) total_p[i] += w.p[i];
    float sum = 0.f, kept[kRouteKept];
#pragma unroll 1
    for (int j0 = 0; j0 < r.k; j0 += kRouteKept) {
#pragma unroll
      for (int jj = 0; jj < kRouteKept; ++jj) {
        const int j = j0 + jj;
        if (j >= r.k) break;
        float best = ninf, prob = 0.f;
        int at = kMaxExperts;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (w.counts && w.l[i] > best) best = w.l[i], prob = w.p[i], at = g * V + i;
#pragma unroll
        for (int o = G / 2; o > 0; o /= 2) {
          const float b = __shfl_xor_sync(kFull, best, o), q = __shfl_xor_sync(kFull, prob, o);
          const int a = __shfl_xor_sync(kFull, at, o);
          if (b > best || (b == best && a < at)) best = b, prob = q, at = a;
        }
        const bool taken = at < kMaxExperts;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (at == g * V + i) total_c[i]++, w.l[i] = ninf;
        sum += prob;
        kept[jj] = prob;
        if (g == 0 && row < r.rows) {
          r.indices[row * r.k + j] = taken ? at : -1;
          if (!r.renormalize || r.k > kRouteKept) r.gates[row * r.k + j] = prob;
        }
      }
    }
    if (r.renormalize && g == 0 && row < r.rows) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;  // a NaN sum stays one
      if (r.k <= kRouteKept) {
#pragma unroll
        for (int jj = 0; jj < kRouteKept; ++jj)
          if (jj < r.k) r.gates[row * r.k + jj] = kept[jj] * inv;
      } else {
        for (int j = 0; j < r.k; ++j) r.gates[row * r.k + j] *= inv;  // this lane's own stores
      }
    }
  }
  // over the warp's rows, then over the block's warps
#pragma unroll
  for (int o = 16; o >= G; o /= 2) {
    rows += __shfl_xor_sync(kFull, rows, o);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      total_p[i] += __shfl_xor_sync(kFull, total_p[i], o);
      total_c[i] += __shfl_xor_sync(kFull, total_c[i], o);
    }
  }
  if (lane < G) {
#pragma unroll
    for (int i = 0; i < V; ++i) sp[warp][g * V + i] = total_p[i], sc[warp][g * V + i] = total_c[i];
    if (g == 0) sc[warp][V * G] = rows;
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= r.experts; e += 32 * kWarps) {
    float p = 0.f;
    int c = 0;
    const bool is_rows = e == r.experts;
    for (int j = 0; j < kWarps; ++j) {
      if (!is_rows) p += sp[j][e];
      c += sc[j][is_rows ? V * G : e];
    }
    if (!is_rows) r.partial_p[(int64_t)blockIdx.x * r.experts + e] = p;
    r.partial_count[(int64_t)blockIdx.x * (r.experts + 1) + e] = c;
  }
  if (gridDim.x == 1) {  // few rows: no second launch
    __syncthreads();
    route_totals(r, 1);
  }
}

__global__ void __launch_bounds__(1024) route_totals_kernel(const RouteParams r) { route_totals(r, r.blocks); }

// d logits = unit * dloss * p * (counts - sum_e counts_e p_e) + the gates' part:
// renormalised, on chosen entries g * (dg - sum g dg); else on chosen entries
// g * dg, and -p * sum g dg on all.
template <typename T, int V, int G>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteParams r) {
  constexpr int kRows = 32 / G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane % G;
  float c[V];
  const float coef = r.grad_loss ? *r.unit * *r.grad_loss : 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = g * V + i < r.experts ? (float)r.counts[g * V + i] * coef : 0.f;
  for (int64_t first = ((int64_t)blockIdx.x * 8 + warp) * kRows; first < r.rows;
       first += (int64_t)gridDim.x * 8 * kRows) {
    const int64_t row = first + lane / G;
    RouteRow<T, V, G> w;
    w.load(r, row, g);
    float dot = 0.f, out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) dot += w.p[i] * c[i];
    dot = RouteRow<T, V, G>::group_sum(dot);
    float inner = 0.f;
    const bool gated = r.grad_gates && w.counts;
    if (gated) {
#pragma unroll 4
      for (int j = 0; j < r.k; ++j) {
        const int64_t o = row * r.k + j;
        if (r.indices[o] >= 0) inner += r.gates[o] * r.grad_gates[o];
      }
      if (!r.renormalize) dot += inner;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = w.counts ? w.p[i] * (c[i] - dot) : 0.f;
    if (gated) {
#pragma unroll 4
      for (int j = 0; j < r.k; ++j) {
        const int64_t o = row * r.k + j, at = r.indices[o];
        if (at < 0) continue;
        if (at >= r.experts) {
          if (g == 0) flag_error(kErrBadIndex);
          continue;
        }
        const float add = r.gates[o] * (r.grad_gates[o] - (r.renormalize ? inner : 0.f));
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (at == g * V + i) out[i] += add;
      }
    }
    if (row >= r.rows) continue;
    T* dst = static_cast<T*>(r.grad_logits) + row * r.experts;
    if (r.vec_out) {
      constexpr int W = 16 / sizeof(T) < V ? 16 / sizeof(T) : V;
      struct alignas(sizeof(T) * W) Vec {
        T v[W];
      };
#pragma unroll
      for (int i = 0; i < V; i += W) {
        if (g * V + i >= r.experts) continue;
        Vec t;
#pragma unroll
        for (int j = 0; j < W; ++j) t.v[j] = from_f<T>(out[i + j]);
        *reinterpret_cast<Vec*>(dst + g * V + i) = t;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (g * V + i < r.experts) dst[g * V + i] = from_f<T>(out[i]);
    }
  }
}

}  // namespace nnue_ls

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
  float4* stats;  // per row: mean of f and 1 / its deviation; the same of y
  const void *grad_y, *grad_h;
  void *grad_x, *grad_f, *grad_gate;
  float* partial;  // backward: [blocks, 5, width] column sums (post_weight, post_bias, scale, pre_weight, pre_bias)
  int64_t rows;
  int width;
  float scale_value, eps;
  int gate_mode;
  bool gate_sigmoid, gate_f32, params_f32;
};

// As an elementwise gate of T; a gate per row is always taken as fp32's.  The short
// exponential's error grows with |v| (25 units of fp32 at v = -20), which 16-bit results do not show.
template <typename T>
__device__ __forceinline__ float sigmoid(float v) {
  return sizeof(T) == 2 ? __fdividef(1.f, 1.f + __expf(-v)) : logistic(v);
}

// 1 / sqrt(v) to about one unit: the hardware's estimate and a Newton step.
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = rsqrtf(v), e = fmaf(-v * r, r, 1.f);
  return v > 0.f && isfinite(r) ? fmaf(0.5f * r, e, r) : r;
}

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
      if (p.gate_sigmoid) row_gate = logistic(row_gate);
    }
  }
  __device__ float param(const void* v, int c) const { return load_mixed<T>(v, c, p.params_f32); }
  __device__ float scale(int c) const { return p.scale ? param(p.scale, c) : p.scale_value; }
  __device__ float gate(int c) const {
    if (p.gate_mode != kGateFull) return row_gate;
    const float v = to_f(g[c]);
    return p.gate_sigmoid ? sigmoid<T>(v) : v;
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

// Mean (layer norm) and 1 / deviation of a row whose element c is value(c).
template <bool CENTER, typename F>
__device__ __forceinline__ void row_stats(const F& value, int width, float eps, float* scratch, float& mean,
                                          float& rstd) {
  float v[1];
  mean = 0.f;
  if (CENTER) {
    v[0] = 0.f;
#pragma unroll 4
    for (int c = threadIdx.x; c < width; c += blockDim.x) v[0] += value(c);
    block_sum(v, scratch);
    mean = v[0] / width;
  }
  v[0] = 0.f;
#pragma unroll 4
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    const float d = value(c) - mean;
    v[0] += d * d;
  }
  block_sum(v, scratch);
  rstd = inv_sqrt(v[0] / width + eps);
}

// One block per row, any width; the row is read again for each pass.
template <typename T, bool CENTER>
__global__ void __launch_bounds__(512) norm_forward_kernel(NormParams p) {
  __shared__ float scratch[32];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    NormRow<T> r(p, row);
    float mean_y = 0.f, rstd_y = 1.f;
    if (p.f && p.post_weight)
      row_stats<CENTER>([&](int c) { return to_f(r.f[c]); }, p.width, p.eps, scratch, r.mean_f, r.rstd_f);
    if (p.pre_weight) row_stats<CENTER>([&](int c) { return r.y(c); }, p.width, p.eps, scratch, mean_y, rstd_y);
#pragma unroll 4
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
// The products with y_hat and f_hat are formed as (y - mean) * (mean(u * (y - mean)) * rstd^2): the two terms of a
// difference that can cancel then share fewer roundings.
// y is formed again from x, f and the gate: x has to be read for the scale's gradient anyway, and the y that the
// forward wrote is rounded to 16 bits, which would show in the fp32 sums.
// Each block owns a slice of `partial` and each thread its columns of it.
template <typename T, bool CENTER>
__global__ void __launch_bounds__(512) norm_backward_kernel(NormParams p) {
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
    const float rstd_y = st.w;
    const T* gy = static_cast<const T*>(p.grad_y) + (p.grad_y ? row * W : 0);
    const T* gh = static_cast<const T*>(p.grad_h) + (p.grad_h ? row * W : 0);
    const bool pre = p.grad_h && p.pre_weight;
    auto y_cen = [&](int c) { return r.y(c) - st.z; };
    float s[2] = {0.f, 0.f};
    if (pre) {
#pragma unroll 4
      for (int c = threadIdx.x; c < W; c += blockDim.x) {
        const float u = to_f(gh[c]) * r.param(p.pre_weight, c);
        s[0] += u * y_cen(c);
        if (CENTER) s[1] += u;
      }
      block_sum(s, scratch);
    }
    const float c1 = s[0] * inv * (rstd_y * rstd_y), c2 = s[1] * inv;
    auto d_of = [&](int c) {
      float d = p.grad_y ? to_f(gy[c]) : 0.f;
      if (pre) {
        const float u = to_f(gh[c]) * r.param(p.pre_weight, c);
        d += rstd_y * (u - c2 - y_cen(c) * c1);
      }
      return d;
    };
    float q[3] = {0.f, 0.f, 0.f};
    if (p.f) {
#pragma unroll 4
      for (int c = threadIdx.x; c < W; c += blockDim.x) {
        const float d = d_of(c);
        if (p.post_weight) {
          const float v = r.gate(c) * d * r.param(p.post_weight, c);
          q[0] += v * (to_f(r.f[c]) - st.x);
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
    const float c3 = q[0] * inv * (st.y * st.y), c4 = q[1] * inv;
#pragma unroll 4
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
          if (p.post_weight) df = r.rstd_f * (gn * r.param(p.post_weight, c) - c4 - (to_f(r.f[c]) - st.x) * c3);
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
          part[3 * W + c] += to_f(gh[c]) * (y_cen(c) * rstd_y);
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

// ---- rows held in registers -----------------------------------------------------
// The kernels above read a row once per pass, for any width.  Up to 4096 columns
// the ones below read it once: a block works on R rows at a time and a thread
// owns eight columns of them (as 16-byte pieces, or single ones where rows are
// not aligned).  A thread's columns are the same in every row, so the
// parameters are read once and the sums over rows are plain registers until
// the block's last row; R rows share each barrier.

// V values of a row at column c.
template <typename T, int V>
struct RowVec {
  struct alignas(sizeof(T) * V) Raw {
    T v[V];
  };
  Raw raw;
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    raw = *reinterpret_cast<const Raw*>(static_cast<const T*>(base) + at);
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f(raw.v[i]); }
  // All values; two 16-bit ones at a time, an instruction each.
  __device__ __forceinline__ void unpack(float* out) const {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
      const unsigned* words = reinterpret_cast<const unsigned*>(&raw);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if constexpr (std::is_same<T, bf16>::value) {
          out[2 * i] = __uint_as_float(words[i] << 16);
          out[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
        } else {
          const float2 t = __half22float2(*reinterpret_cast<const __half2*>(words + i));
          out[2 * i] = t.x, out[2 * i + 1] = t.y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = to_f(raw.v[i]);
    }
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_row(void* base, int64_t at, const float (&v)[V]) {
  typename RowVec<T, V>::Raw o;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    unsigned* words = reinterpret_cast<unsigned*>(&o);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, bf16>::value)
        *reinterpret_cast<__nv_bfloat162*>(words + i) = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      else
        *reinterpret_cast<__half2*>(words + i) = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = from_f<T>(v[i]);
  }
  *reinterpret_cast<typename RowVec<T, V>::Raw*>(static_cast<T*>(base) + at) = o;
}
// V values of a parameter; `absent` where there is none.
template <typename T, int V>
__device__ __forceinline__ void load_param(const void* p, int c, bool f32, float absent, float (&v)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = absent;
  } else if (f32) {
    if constexpr (V >= 4) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + c + i));
        v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __ldg(static_cast<const float*>(p) + c + i);
    }
  } else {
    RowVec<T, V> t;
    t.load(p, c);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = t[i];
  }
}

// Sums K values (a power of two) over the block; every thread gets the totals.
// Within a warp each step of the exchange halves the number of values a lane
// carries; between warps the sums meet in shared memory, taken in warp order.
// Two halves of `scratch` in turn make one barrier enough.
template <int K>
struct BlockSum {
  static constexpr int kSpan = 32 / K;  // neighbouring lanes that end with the same value
  float* scratch;                       // 2 * 32 * K floats
  int turn = 0;
  __device__ __forceinline__ void operator()(float (&v)[K]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int o = 16;
#pragma unroll
    for (int n = K; n > 1; n /= 2) {
#pragma unroll
      for (int i = 0; i < n / 2; ++i) {
        const bool upper = lane & o;
        const float send = upper ? v[i] : v[i + n / 2], keep = upper ? v[i + n / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(kFull, send, o);
      }
      o /= 2;
    }
    float sum = v[0];
#pragma unroll
    for (int q = kSpan / 2; q > 0; q /= 2) sum += __shfl_xor_sync(kFull, sum, q);
    if (warps > 1) {
      float* s = scratch + turn * 32 * K;
      turn ^= 1;
      const int k = lane / kSpan, sub = lane % kSpan;
      if (sub == 0) s[warp * K + k] = sum;
      __syncthreads();
      sum = 0.f;
      for (int w = sub; w < warps; w += kSpan) sum += s[w * K + k];
#pragma unroll
      for (int q = kSpan / 2; q > 0; q /= 2) sum += __shfl_xor_sync(kFull, sum, q);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = __shfl_sync(kFull, sum, k * kSpan);
  }
};

__host__ __device__ constexpr int pow2_at_least(int n) { return n <= 1 ? 1 : 2 * pow2_at_least((n + 1) / 2); }

// A thread's columns: kColumns of them, V neighbouring ones at a time; a warp's
// are neighbours, so that a thread's lie a constant apart.
constexpr int kColumns = 8;
template <typename T, int V>
struct Columns {
  static constexpr int kNV = kColumns / V;
  __device__ __forceinline__ static int at(int i) {
    return (int)(threadIdx.x & ~31u) * kColumns + ((int)(threadIdx.x & 31) + 32 * i) * V;
  }
  __device__ __forceinline__ static void store(void* base, int64_t row, int width, const float (&v)[kColumns]) {
    T* dst = static_cast<T*>(base) + row * width;
#pragma unroll
    for (int i = 0; i < kNV; ++i)
      if (at(i) < width) {
        float t[V];
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = v[i * V + j];
        store_row<T, V>(dst, at(i), t);
      }
  }
  __device__ __forceinline__ static void params(const void* p, int width, bool f32, float absent,
                                                float (&v)[kColumns]) {
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      float t[V];
#pragma unroll
      for (int j = 0; j < V; ++j) t[j] = 0.f;
      if (at(i) < width) load_param<T, V>(p, at(i), f32, absent, t);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = t[j];
    }
  }
};

// The rows to come, on their way from HBM to shared memory while earlier ones
// are worked on: STAGES rounds of R rows, read again by every pass over a row
// instead of held in registers.  Arrays: x, f, gate, grad_y, grad_h.
//
// Rows of 16-byte pieces (V > 1): a thread copies its own columns into slots of
// its own, so that nobody waits for anybody.  Other rows (V == 1): the R rows of
// a round are one run of memory, copied as the aligned 16-byte pieces that cover
// it, whoever needs them, with a barrier before they are read; a row then starts
// at any byte of shared memory (16384 x 4095 bf16, forward and backward: 594 us;
// with single values loaded straight into registers 774 us).
enum RowArray : int { kX = 0, kF = 1, kGate = 2, kGradY = 3, kGradH = 4 };

// Bytes of one array's rows in one round, for rows that are not 16-byte pieces.
__host__ __device__ constexpr int run_bytes(int rows, int width, int size) { return (rows * width * size + 46) & ~15; }

template <typename T, int V, int R, bool FULL, bool BACKWARD, int STAGES>
struct RowRing {
  using C = Columns<T, V>;
  using Raw = typename RowVec<T, V>::Raw;
  static constexpr int kArrays = 2 + FULL + 2 * BACKWARD, kNV = C::kNV;
  __host__ __device__ static constexpr int index(int a) { return a <= kGate ? a : a - !FULL; }
  char* smem;
  const T* base[5];
  int width, rows, stage = 0;
  const T* run[V == 1 ? kArrays : 1];  // V == 1: the round's rows in shared memory

  __device__ __forceinline__ RowRing(const NormParams& p, void* ring) {
    smem = static_cast<char*>(ring);
    base[kX] = static_cast<const T*>(p.x);
    base[kF] = static_cast<const T*>(p.f);
    base[kGate] = static_cast<const T*>(FULL ? p.gate : nullptr);
    base[kGradY] = static_cast<const T*>(BACKWARD ? p.grad_y : nullptr);
    base[kGradH] = static_cast<const T*>(BACKWARD ? p.grad_h : nullptr);
    width = p.width;
    rows = (int)p.rows;
    if constexpr (V > 1) {  // what is never copied reads as zero
#pragma unroll
      for (int i = 0; i < STAGES * R; ++i)
#pragma unroll
        for (int v = 0; v < kNV; ++v)
#pragma unroll
          for (int a = 0; a < 5; ++a)
            if (index(a) < kArrays && a != (FULL ? -1 : kGate) && (C::at(v) >= width || !has(a)))
              *reinterpret_cast<uint4*>(slot(i / R, i % R, index(a), v)) = uint4{};
    }
  }
  __device__ __forceinline__ bool has(int a) const {
    return !(a == kGate && !FULL) && !(a >= kGradY && !BACKWARD) && (a == kX || base[a]);
  }
  __device__ __forceinline__ Raw* slot(int st, int r, int i, int v) const {
    const int warp_stage = (int)(threadIdx.x >> 5) * STAGES + st, lane = (int)(threadIdx.x & 31);
    return reinterpret_cast<Raw*>(smem) + warp_stage * (R * kArrays * kNV * 32) + lane + ((r * kArrays + i) * kNV + v) * 32;
  }
  __device__ __forceinline__ char* run_at(int st, int i) const {
    return smem + (st * kArrays + i) * run_bytes(R, width, (int)sizeof(T));
  }
  __device__ __forceinline__ static void copy(void* dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(dst)),
                 "l"(src), "r"(bytes)
                 : "memory");
  }
  __device__ __forceinline__ void issue(int row0, int st) const {
    if (row0 < rows) {
      if constexpr (V > 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int64_t row = (int64_t)min(row0 + r, rows - 1) * width;  // beyond the last row: read, not used
#pragma unroll
          for (int v = 0; v < kNV; ++v) {
            const int c = C::at(v);
            if (c >= width) continue;
#pragma unroll
            for (int a = 0; a < 5; ++a)
              if (has(a)) copy(slot(st, r, index(a), v), base[a] + row + c, 16);
          }
        }
      } else {
        const int64_t first = (int64_t)row0 * width, last = (int64_t)min(row0 + R, rows) * width;
#pragma unroll
        for (int a = 0; a < 5; ++a) {
          if (!has(a)) continue;
          char* dst = run_at(st, index(a));
          const uintptr_t lo = reinterpret_cast<uintptr_t>(base[a]), hi = lo + (int64_t)rows * width * sizeof(T),
                          from = (lo + first * sizeof(T)) & ~uintptr_t(15), to = lo + last * sizeof(T);
          const int pieces = (int)((to - from + 15) / 16);
          for (int i = (int)threadIdx.x; i < pieces; i += (int)blockDim.x) {
            const uintptr_t at = from + 16 * (int64_t)i;
            if (at >= lo) {
              copy(dst + 16 * i, reinterpret_cast<const void*>(at), (int)min((uintptr_t)16, hi - at));
            } else {  // the tensor starts inside this piece
              const int skip = (int)(lo - at) / (int)sizeof(T);
              const int64_t have = (int64_t)rows * width;
              for (int k = skip; k < 16 / (int)sizeof(T); ++k)
                if (k - skip < have) reinterpret_cast<T*>(dst)[k] = base[a][k - skip];
            }
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void start(int row0, int stride) {
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(row0 + i * stride, i);
  }
  // The rows from row0 on are there; those of STAGES - 1 rounds later are asked for.
  __device__ __forceinline__ void next(int row0, int stride) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    // the slots written now were last read in the round before: by this thread, or before the barrier
    if (V == 1) __syncthreads();
    const int64_t ahead = row0 + (int64_t)(STAGES - 1) * stride;
    issue(ahead < rows ? (int)ahead : rows, stage == 0 ? STAGES - 1 : stage - 1);
    if constexpr (V == 1) {
#pragma unroll
      for (int a = 0; a < 5; ++a)
        if (has(a)) {
          const uintptr_t at = reinterpret_cast<uintptr_t>(base[a]) + (int64_t)row0 * width * sizeof(T);
          run[index(a)] = reinterpret_cast<const T*>(run_at(stage, index(a)) + (at & 15));
        }
    }
  }
  __device__ __forceinline__ void done() {
    if (++stage == STAGES) stage = 0;
  }
  // The thread's values of array A in row r of the round; zero where there are none.
  template <int A>
  __device__ __forceinline__ void get(int r, float (&out)[kColumns]) const {
#pragma unroll
    for (int v = 0; v < kNV; ++v) {
      RowVec<T, V> raw;
      if constexpr (V > 1) {
        raw.raw = *slot(stage, r, index(A), v);
      } else {
        raw.raw = Raw{};
        if (has(A) && C::at(v) < width) raw.raw.v[0] = run[index(A)][r * width + C::at(v)];
      }
      raw.unpack(out + v * V);
    }
  }
};

// The gate of a row's columns.
template <typename T, bool FULL, typename Ring>
__device__ __forceinline__ void gates(const NormParams& p, const Ring& ring, int r, float row_gate,
                                      float (&g)[kColumns]) {
  if constexpr (FULL) {
    ring.template get<kGate>(r, g);
    if (p.gate_sigmoid) {
#pragma unroll
      for (int k = 0; k < kColumns; ++k) g[k] = sigmoid<T>(g[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kColumns; ++k) g[k] = row_gate;
  }
}
template <bool MORE, typename C>
__device__ __forceinline__ void scales(const NormParams& p, float (&sc)[kColumns]) {
  if (MORE) {
    C::params(p.scale, p.width, p.params_f32, p.scale_value, sc);
  } else {
#pragma unroll
    for (int k = 0; k < kColumns; ++k) sc[k] = p.scale_value;
  }
}
template <typename T>
__device__ __forceinline__ float load_row_gate(const NormParams& p, int row) {
  if (p.gate_mode != kGateRow) return 1.f;
  const float g = load_mixed<T>(p.gate, row, p.gate_f32);
  return p.gate_sigmoid ? logistic(g) : g;
}

// The forward's calls without biases or a learned scale fit 64 registers, so
// that an SM holds 1024 threads instead of 512 (before other savings: 65536 x
// 1040 bf16 159 us against 181, 16384 x 4096 bf16 123 against 166).  With them
// 16-bit rows fit 80, for 768 (65536 x 1040 bf16 layer norm 202 us against 234);
// fp32 rows are better two at a time with 512 (262 us against 288).
__host__ __device__ constexpr int norm_forward_threads(int v, bool both, bool more) {
  return v == 1 || !both ? 512 : !more ? 1024 : v == 8 ? 768 : 512;
}
// The backward's fit 96, for 640 threads: four blocks of 1040 columns instead of
// three, two of 2056 instead of one (forward and backward, 65536 x 1040 fp32 472
// us against 515, bf16 326 against 341, 16384 x 2056 fp32 260 against 360; 4096
// columns, where one block fits either way, bf16 317 against 306).
__host__ __device__ constexpr int norm_backward_threads(int v, bool both, bool more) {
  return v > 1 && both && !more ? 640 : 512;
}

// BOTH: the call has f with its norm and the norm after it.  MORE: it may have
// biases or a learned scale.  Without BOTH what is there is looked up.
// The busiest unit on 16-bit rows is instruction issue (60-70% of its slots at 16
// to 32 warps an SM), so a thread takes eight columns:
// what a row costs besides its columns (addresses, copies, the exchange of sums)
// is shared by eight instead of four.  65536 x 1040, row gate, rms norms:
// forward fp32 184 us (90% of the HBM copy rate over its four arrays), bf16 120
// (69%); backward fp32 273 us (91% over its six), bf16 196 (64%).  With four
// columns a thread the bf16 figures were 186 and 472 us.
template <typename T, int V, int R, bool CENTER, bool FULL, bool BOTH, bool MORE, int STAGES>
__global__ void __launch_bounds__(norm_forward_threads(V, BOTH, MORE), 1) norm_forward_rows_kernel(const NormParams p) {
  using C = Columns<T, V>;
  constexpr int N = kColumns;
  extern __shared__ float4 norm_ring[];
  __shared__ float scratch[2 * 32 * R];
  BlockSum<R> total{scratch};
  const bool has_f = BOTH || p.f, post = BOTH || p.post_weight, pre = BOTH || p.h;
  const int W = p.width, rows = (int)p.rows, stride = (int)gridDim.x * R;
  const float inv = 1.f / W;
  float w[N], b[N], sc[N], pw[N], pb[N];
  C::params(p.post_weight, W, p.params_f32, 1.f, w);
  C::params(MORE ? p.post_bias : nullptr, W, p.params_f32, 0.f, b);
  scales<MORE, C>(p, sc);
  C::params(p.pre_weight, W, p.params_f32, 1.f, pw);
  C::params(MORE ? p.pre_bias : nullptr, W, p.params_f32, 0.f, pb);
  RowRing<T, V, R, FULL, false, STAGES> ring(p, norm_ring);
  ring.start((int)blockIdx.x * R, stride);
  for (int row0 = (int)blockIdx.x * R; row0 < rows; row0 += stride) {
    ring.next(row0, stride);
    float gate[R], mean_f[R], rstd_f[R], mean_y[R], rstd_y[R], s[R], y[R][N], v[N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      gate[r] = FULL ? 1.f : load_row_gate<T>(p, min(row0 + r, rows - 1));
      mean_f[r] = mean_y[r] = 0.f;
      rstd_f[r] = rstd_y[r] = 1.f;
    }
    if (post) {
      if (CENTER) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          ring.template get<kF>(r, v);
          s[r] = 0.f;
#pragma unroll
          for (int k = 0; k < N; ++k) s[r] += v[k];
        }
        total(s);
#pragma unroll
        for (int r = 0; r < R; ++r) mean_f[r] = s[r] * inv;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ring.template get<kF>(r, v);
        s[r] = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float d = CENTER ? (C::at(k / V) < W ? v[k] - mean_f[r] : 0.f) : v[k];
          s[r] = fmaf(d, d, s[r]);
        }
      }
      total(s);
#pragma unroll
      for (int r = 0; r < R; ++r) rstd_f[r] = inv_sqrt(s[r] * inv + p.eps);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ring.template get<kX>(r, y[r]);
      if (has_f) {
        ring.template get<kF>(r, v);
        if (FULL || MORE) {
          float g[N];
          gates<T, FULL>(p, ring, r, gate[r], g);
#pragma unroll
          for (int k = 0; k < N; ++k)
            y[r][k] = fmaf(g[k], fmaf((CENTER ? v[k] - mean_f[r] : v[k]) * rstd_f[r], w[k], b[k]), sc[k] * y[r][k]);
        } else {
          const float gr = gate[r] * rstd_f[r];
#pragma unroll
          for (int k = 0; k < N; ++k) y[r][k] = fmaf((CENTER ? v[k] - mean_f[r] : v[k]) * gr, w[k], sc[k] * y[r][k]);
        }
      }
      if ((BOTH || p.y) && row0 + r < rows) C::store(p.y, row0 + r, W, y[r]);  // without f it may be wanted too
    }
    if (pre) {
      if (CENTER) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          s[r] = 0.f;
#pragma unroll
          for (int k = 0; k < N; ++k) s[r] += C::at(k / V) < W ? y[r][k] : 0.f;
        }
        total(s);
#pragma unroll
        for (int r = 0; r < R; ++r) mean_y[r] = s[r] * inv;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[r] = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float d = CENTER ? (C::at(k / V) < W ? y[r][k] - mean_y[r] : 0.f) : y[r][k];
          s[r] = fmaf(d, d, s[r]);
        }
      }
      total(s);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        rstd_y[r] = inv_sqrt(s[r] * inv + p.eps);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float u = (CENTER ? y[r][k] - mean_y[r] : y[r][k]) * rstd_y[r];
          y[r][k] = MORE ? fmaf(u, pw[k], pb[k]) : u * pw[k];
        }
        if (row0 + r < rows) C::store(p.h, row0 + r, W, y[r]);
      }
    }
    if (p.stats && threadIdx.x == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row0 + r < rows) p.stats[row0 + r] = make_float4(mean_f[r], rstd_f[r], mean_y[r], rstd_y[r]);
    }
    ring.done();
  }
}

template <typename T, int V, int R, bool CENTER, bool FULL, bool BOTH, bool MORE, int STAGES>
__global__ void __launch_bounds__(norm_backward_threads(V, BOTH, MORE), 1) norm_backward_rows_kernel(const NormParams p) {
  using C = Columns<T, V>;
  constexpr int N = kColumns, N1 = 1 + CENTER, N2 = 1 + CENTER + MORE, K1 = R * N1, K2 = pow2_at_least(R * N2);
  extern __shared__ float4 norm_ring[];
  __shared__ float scratch[2 * 32 * (K1 + K2)];
  BlockSum<K1> total1{scratch};
  BlockSum<K2> total2{scratch + 2 * 32 * K1};
  const bool has_f = BOTH || p.f, post = BOTH || p.post_weight, pre = BOTH || (p.grad_h && p.pre_weight);
  const int W = p.width, rows = (int)p.rows, stride = (int)gridDim.x * R;
  const float inv = 1.f / W;
  float w[N], b[N], sc[N], pw[N];
  float sum_post[N] = {}, sum_post_bias[N] = {}, sum_scale[N] = {}, sum_pre[N] = {}, sum_pre_bias[N] = {};
  C::params(p.post_weight, W, p.params_f32, 1.f, w);
  C::params(MORE ? p.post_bias : nullptr, W, p.params_f32, 0.f, b);
  scales<MORE, C>(p, sc);
  C::params(p.pre_weight, W, p.params_f32, 0.f, pw);
  RowRing<T, V, R, FULL, true, STAGES> ring(p, norm_ring);
  ring.start((int)blockIdx.x * R, stride);
  // the rows' statistics and gates come a round ahead, in registers
  float4 st[R], st_next[R];
  float gate[R], gate_next[R];
  auto ahead = [&](int row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = min(row0 + r, rows - 1);
      st_next[r] = __ldg(p.stats + row);
      gate_next[r] = FULL ? 1.f : load_row_gate<T>(p, row);
    }
  };
  if ((int)blockIdx.x * R < rows) ahead((int)blockIdx.x * R);
  for (int row0 = (int)blockIdx.x * R; row0 < rows; row0 += stride) {
    ring.next(row0, stride);
#pragma unroll
    for (int r = 0; r < R; ++r) st[r] = st_next[r], gate[r] = gate_next[r];
    ahead(min(row0 + stride, rows - 1));
    float d[R][N], s[K1], q[K2];  // d: y - mean, then the gradient of y
    float gates_of_row[FULL && R == 1 ? N : 1];  // taken once; two rows' would not fit the registers
    auto gates_of = [&](int r, float (&g)[N]) {
      if constexpr (FULL && R == 1) {
#pragma unroll
        for (int k = 0; k < N; ++k) g[k] = gates_of_row[k];
      } else {
        gates<T, FULL>(p, ring, r, gate[r], g);
      }
    };
    if constexpr (FULL && R == 1) {
      if (has_f) gates<T, FULL>(p, ring, 0, 1.f, gates_of_row);
    }
    if (pre) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float gh[N], v[N], g[N];
        ring.template get<kX>(r, d[r]);
        ring.template get<kGradH>(r, gh);
        if (has_f) {
          ring.template get<kF>(r, v);
          if (FULL || MORE) {
            gates_of(r, g);
#pragma unroll
            for (int k = 0; k < N; ++k)
              d[r][k] = fmaf(g[k], fmaf((CENTER ? v[k] - st[r].x : v[k]) * st[r].y, w[k], b[k]), sc[k] * d[r][k]);
          } else {
            const float gr = gate[r] * st[r].y;
#pragma unroll
            for (int k = 0; k < N; ++k) d[r][k] = fmaf((CENTER ? v[k] - st[r].x : v[k]) * gr, w[k], sc[k] * d[r][k]);
          }
        }
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          if (CENTER) d[r][k] -= st[r].z;
          const float u = gh[k] * pw[k];
          s0 = fmaf(u, d[r][k], s0);
          if (CENTER) s1 += u;
        }
        s[r * N1] = s0;
        if (CENTER) s[r * N1 + 1] = s1;
        if (row0 + r < rows) {  // a row beyond the last one adds nothing
#pragma unroll
          for (int k = 0; k < N; ++k) {
            sum_pre[k] = fmaf(gh[k], d[r][k] * st[r].w, sum_pre[k]);
            if (MORE) sum_pre_bias[k] += gh[k];
          }
        }
      }
      total1(s);
    }
#pragma unroll
    for (int i = R * N2; i < K2; ++i) q[i] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = row0 + r < rows;
      float v[N], dx[N], q0 = 0.f, q1 = 0.f, q2 = 0.f;
      ring.template get<kGradY>(r, dx);
      if (pre) {
        const float c1 = s[r * N1] * inv * (st[r].w * st[r].w), c2 = CENTER ? s[r * N1 + CENTER] * inv : 0.f;
        ring.template get<kGradH>(r, v);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float u = v[k] * pw[k];
          dx[k] = fmaf(st[r].w, fmaf(-d[r][k], c1, CENTER ? u - c2 : u), dx[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) d[r][k] = dx[k], dx[k] *= sc[k];
      if (p.grad_x && live) C::store(p.grad_x, row0 + r, W, dx);
      if (has_f) {
        // a gate per row is taken out of the row's sums: gr of it stays in front
        const float gr = gate[r] * st[r].y;
        float g[N];
        ring.template get<kF>(r, v);
        if (FULL) gates_of(r, g);
        if (MORE) ring.template get<kX>(r, dx);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float gn = FULL ? g[k] * d[r][k] : d[r][k], fc = CENTER ? v[k] - st[r].x : v[k], u = gn * w[k];
          q0 = fmaf(u, fc, q0);  // u as below: what cancels there is rounded alike
          if (CENTER) q1 += u;
          if (MORE && !FULL) q2 = fmaf(gn, b[k], q2);
          if (live) {
            sum_post[k] = fmaf(gn * fc, gr, sum_post[k]);
            if (MORE) {
              sum_post_bias[k] = fmaf(gn, gate[r], sum_post_bias[k]);
              sum_scale[k] = fmaf(d[r][k], dx[k], sum_scale[k]);
            }
          }
        }
      }
      q[r * N2] = q0;
      if (CENTER) q[r * N2 + CENTER] = q1;
      if (MORE) q[r * N2 + N2 - 1] = q2;
    }
    if (has_f) {
      total2(q);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row0 + r < rows) {
          const float c3 = post ? q[r * N2] * inv * (st[r].y * st[r].y) : 0.f,
                      c4 = CENTER && post ? q[r * N2 + CENTER] * inv : 0.f, gr = gate[r] * st[r].y;
          float v[N], g[N], df[N];
          ring.template get<kF>(r, v);
          if (FULL) gates_of(r, g);
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (CENTER) v[k] -= st[r].x;
          if (p.grad_f) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
              const float gn = FULL ? g[k] * d[r][k] : d[r][k];
              df[k] = gr * fmaf(-v[k], c3, gn * w[k] - c4);
            }
            C::store(p.grad_f, row0 + r, W, df);
          }
          if (FULL) {
            if (p.grad_gate) {
#pragma unroll
              for (int k = 0; k < N; ++k) {
                df[k] = d[r][k] * fmaf(v[k] * st[r].y, w[k], b[k]);
                if (p.gate_sigmoid) df[k] *= g[k] * (1.f - g[k]);
              }
              C::store(p.grad_gate, row0 + r, W, df);
            }
          } else if (p.grad_gate && threadIdx.x == 0) {
            const float gt = gate[r], dq = fmaf(q[r * N2], st[r].y, MORE ? q[r * N2 + N2 - 1] : 0.f);
            store_mixed<T>(p.grad_gate, row0 + r, p.gate_f32, p.gate_sigmoid ? dq * gt * (1.f - gt) : dq);
          }
        }
      }
    }
    ring.done();
  }
  if (!p.partial) return;
  float* part = p.partial + (int64_t)blockIdx.x * 5 * W;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = C::at(k / V) + k % V;
    if (C::at(k / V) >= W) continue;
    part[c] = sum_post[k];
    part[3 * W + c] = sum_pre[k];
    if (MORE) {
      part[W + c] = sum_post_bias[k];
      part[2 * W + c] = sum_scale[k];
      part[4 * W + c] = sum_pre_bias[k];
    }
  }
}

// Totals of the backward's column sums over blocks: 32 rows of threads take
// every 32nd block, then their sums are added in turn; out[i] null = not wanted.
struct NormTotals {
  void* out[5];
};
template <typename T>
__global__ void __launch_bounds__(1024) norm_totals_kernel(const float* __restrict__ partial, int blocks, int width,
                                                           NormTotals t, bool out_f32) {
  __shared__ float red[32][33];
  const int which = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  if (!t.out[which]) return;
  float sum = 0.f;
  if (c < width)
#pragma unroll 4
    for (int b = threadIdx.y; b < blocks; b += 32) sum += partial[((int64_t)b * 5 + which) * width + c];
  red[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    for (int i = 1; i < 32; ++i) sum += red[i][threadIdx.x];
    store_mixed<T>(t.out[which], c, out_f32, sum);
  }
}

}  // namespace nnue_ls

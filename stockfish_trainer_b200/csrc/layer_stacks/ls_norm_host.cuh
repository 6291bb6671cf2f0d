// Host side of the norms around a residual block: checks, which kernel a call
// takes, the launches.
#pragma once

#include <algorithm>
#include <type_traits>

#include "ls_host.cuh"
#include "ls_norm.cuh"

namespace nnue_ls {
namespace {

NormParams norm_params(const nnue_ls_norm& a) {
  NormParams p{};
  p.x = a.x;
  p.f = a.f;
  p.gate = a.gate;
  p.post_weight = a.post_weight;
  p.post_bias = a.post_bias;
  p.scale = a.scale;
  p.pre_weight = a.pre_weight;
  p.pre_bias = a.pre_bias;
  p.y = a.y;
  p.h = a.h;
  p.stats = reinterpret_cast<float4*>(a.stats);
  p.grad_y = a.grad_y;
  p.grad_h = a.grad_h;
  p.grad_x = a.grad_x;
  p.grad_f = a.grad_f;
  p.grad_gate = a.grad_gate;
  p.rows = a.rows;
  p.width = a.width;
  p.scale_value = a.scale_value;
  p.eps = a.eps;
  p.gate_mode = a.gate_mode;
  p.gate_sigmoid = a.gate_sigmoid != 0;
  p.gate_f32 = a.gate_dtype == NNUE_LS_F32;
  p.params_f32 = a.params_dtype == NNUE_LS_F32;
  return p;
}

bool wants_params(const nnue_ls_norm& a) {
  return a.grad_post_weight || a.grad_post_bias || a.grad_scale || a.grad_pre_weight || a.grad_pre_bias;
}

// Whether every tensor and parameter can be read 16 bytes (parameters: 16 or
// fewer) at a time.
template <typename T>
bool norm_vectors(const nnue_ls_norm& a) {
  const void* all[] = {a.x, a.f, a.gate_mode == kGateFull ? a.gate : nullptr, a.post_weight, a.post_bias, a.scale,
                       a.pre_weight, a.pre_bias, a.y, a.h, a.grad_y, a.grad_h, a.grad_x, a.grad_f,
                       a.gate_mode == kGateFull ? a.grad_gate : nullptr};
  for (const void* p : all)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return a.width % (int)(16 / sizeof(T)) == 0;
}

// Which kernel a call takes.  Up to 2048 columns, four per thread: rows of up to
// 1152 columns get 288 threads a block, whose registers hold more rows at once.
// Wider rows are read once per pass.
struct RowPlan {
  bool vec;
  int threads;  // 0: the kernel for any width
  bool narrow() const { return vec && threads <= 288; }
};
constexpr int kRowsForward = 4;

template <typename T>
RowPlan plan_norm(const nnue_ls_norm& a) {
  RowPlan r{norm_vectors<T>(a), 0};
  const int64_t threads = ceil_div(a.width, 128) * 32;
  if (threads <= 512) r.threads = (int)threads;
  return r;
}
// rows at a time: what 168 registers a thread hold twice over (narrow) or 128 once
template <typename T>
constexpr int rows_backward(bool narrow, bool full) { return narrow && sizeof(T) == 2 && !full ? 4 : 2; }

template <typename T>
int64_t norm_backward_blocks(const nnue_ls_norm& a, const RowPlan& r) {
  const int64_t rows = std::max<int64_t>(a.rows, 1);
  if (!r.threads) return std::min<int64_t>(rows, kNumSMs * 4);
  const int per_sm = (r.narrow() ? 288 : 512) / r.threads;  // as the registers allow
  return std::min<int64_t>(ceil_div(rows, rows_backward<T>(r.narrow(), a.gate_mode == kGateFull)), (int64_t)kNumSMs * std::min(per_sm, 8));
}

// fn(center, full) with both as constants.
template <typename F>
void with_flags(bool center, bool full, const F& fn) {
  using Yes = std::true_type;
  using No = std::false_type;
  if (center) full ? fn(Yes{}, Yes{}) : fn(Yes{}, No{});
  else full ? fn(No{}, Yes{}) : fn(No{}, No{});
}

}  // namespace

template <typename T>
int norm_forward(const nnue_ls_norm& a, cudaStream_t s) {
  const NormParams p = norm_params(a);
  const RowPlan r = plan_norm<T>(a);
  const bool center = a.kind == NNUE_LS_NORM_LAYER;
  count_launch();
  if (!r.threads) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, kNumSMs * 8);
    if (center) norm_forward_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else norm_forward_kernel<T, false><<<grid, 256, 0, s>>>(p);
    return check_launch("norm_forward");
  }
  // as many blocks as stay on the SMs together, each looping over rows
  const int per_sm = std::min(16, 576 / r.threads);
  const unsigned grid =
      (unsigned)std::min<int64_t>(ceil_div(a.rows, kRowsForward), (int64_t)kNumSMs * std::max(1, per_sm));
  with_flags(center, a.gate_mode == kGateFull, [&](auto c, auto f) {
    constexpr bool C = decltype(c)::value, F = decltype(f)::value;
    if (r.narrow()) norm_forward_rows_kernel<T, 4, kRowsForward, C, F, 288, 2><<<grid, r.threads, 0, s>>>(p);
    else if (r.vec) norm_forward_rows_kernel<T, 4, kRowsForward, C, F, 512, 1><<<grid, r.threads, 0, s>>>(p);
    else norm_forward_rows_kernel<T, 1, kRowsForward, C, F, 512, 1><<<grid, r.threads, 0, s>>>(p);
  });
  return check_launch("norm_forward");
}

template <typename T>
size_t norm_backward_bytes(const nnue_ls_norm& a) {
  return wants_params(a) ? align256((size_t)norm_backward_blocks<T>(a, plan_norm<T>(a)) * 5 * a.width * 4) : 0;
}

template <typename T>
int norm_backward(const nnue_ls_norm& a, void* workspace, cudaStream_t s) {
  NormParams p = norm_params(a);
  const bool params = wants_params(a), center = a.kind == NNUE_LS_NORM_LAYER;
  p.partial = params ? static_cast<float*>(workspace) : nullptr;
  const RowPlan r = plan_norm<T>(a);
  const unsigned grid = (unsigned)norm_backward_blocks<T>(a, r);
  count_launch();
  if (!r.threads) {
    if (center) norm_backward_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else norm_backward_kernel<T, false><<<grid, 256, 0, s>>>(p);
  } else {
    with_flags(center, a.gate_mode == kGateFull, [&](auto c, auto f) {
      constexpr bool C = decltype(c)::value, F = decltype(f)::value;
      if (r.narrow()) norm_backward_rows_kernel<T, 4, rows_backward<T>(true, F), C, F, true, 288><<<grid, r.threads, 0, s>>>(p);
      else if (r.vec) norm_backward_rows_kernel<T, 4, 2, C, F, false, 512><<<grid, r.threads, 0, s>>>(p);
      else norm_backward_rows_kernel<T, 1, 2, C, F, false, 512><<<grid, r.threads, 0, s>>>(p);
    });
  }
  if (params) {
    const NormTotals out{{a.grad_post_weight, a.grad_post_bias, a.grad_scale, a.grad_pre_weight, a.grad_pre_bias}};
    count_launch();
    norm_totals_kernel<T><<<dim3((unsigned)ceil_div(a.width, 32), 5), dim3(32, 32), 0, s>>>(
        p.partial, (int)grid, a.width, out, p.params_f32);
  }
  return check_launch("norm_backward");
}

}  // namespace nnue_ls

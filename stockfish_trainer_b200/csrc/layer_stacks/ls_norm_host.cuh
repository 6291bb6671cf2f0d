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

// Which kernel a call takes.  Up to 4096 columns, four per thread; the fewer
// threads a row takes, the more registers each has, for more rows at once.
// Wider rows are read once per pass (65536 x 1040 fp32 forward and backward:
// 0.57 ms by rows, 2.1 ms by passes).
enum RowClass : int { kNarrow = 0, kMiddle = 1, kWide = 2, kAnyWidth = 3 };
struct RowPlan {
  bool vec;
  int threads, cls;
};

template <typename T>
RowPlan plan_norm(const nnue_ls_norm& a) {
  const int64_t threads = ceil_div(a.width, 128) * 32;
  const bool vec = norm_vectors<T>(a);
  const int cls = threads <= 288 && vec ? kNarrow : threads <= 512 ? kMiddle : threads <= 1024 ? kWide : kAnyWidth;
  return RowPlan{vec, (int)std::min<int64_t>(threads, 1024), cls};
}

// Rows at a time, rounds in flight, and blocks per SM, so that registers and
// 227 KB of shared memory hold them.
template <typename T, int CLASS, bool FULL, bool BACKWARD>
struct RowShape {
  static constexpr int kThreads = CLASS == kNarrow ? 288 : CLASS == kMiddle ? 512 : 1024;
  static constexpr int kRows = BACKWARD ? (CLASS == kNarrow && sizeof(T) == 2 ? 4 : CLASS == kWide ? 1 : 2)
                               : CLASS == kWide || (sizeof(T) == 4 && FULL) ? 2
                                                                           : 4;
  static constexpr int kSlot = (int)sizeof(T) * 4 * kRows * (2 + FULL + 2 * BACKWARD);  // bytes per thread and round
  static constexpr int kBlocks = CLASS == kNarrow ? 2 : 1;
  static constexpr int kFit = 220 * 1024 / kBlocks / (kSlot * kThreads);
  static constexpr int kStages = kFit > 4 ? 4 : kFit;
  static_assert(kStages >= 2, "a round on its way while one is worked on");
};

int norm_blocks_per_sm(const RowPlan& r) {
  return std::min(16, std::max(1, (r.cls == kNarrow ? 576 : r.cls == kMiddle ? 512 : 1024) / r.threads));
}

template <typename T>
int64_t norm_backward_blocks(const nnue_ls_norm& a, const RowPlan& r) {
  const int64_t rows = std::max<int64_t>(a.rows, 1);
  if (r.cls == kAnyWidth) return std::min<int64_t>(rows, kNumSMs * 4);
  const int at_once = r.cls == kNarrow   ? RowShape<T, kNarrow, false, true>::kRows
                      : r.cls == kMiddle ? RowShape<T, kMiddle, false, true>::kRows
                                         : RowShape<T, kWide, false, true>::kRows;
  return std::min<int64_t>(ceil_div(rows, at_once), (int64_t)kNumSMs * norm_blocks_per_sm(r));
}

// Launches with the ring's shared memory, `slots` of them per thread.
template <typename K>
int launch_norm_rows(K kernel, unsigned grid, const RowPlan& r, size_t slot_bytes, const NormParams& p, cudaStream_t s) {
  const size_t smem = slot_bytes * r.threads;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return fail(NNUE_LS_ERR_CUDA, "norm: %s", cudaGetErrorString(e));
  }
  kernel<<<grid, r.threads, smem, s>>>(p);
  return NNUE_LS_OK;
}

// fn(center, full, both) with all as constants.
template <typename F>
int with_flags(bool center, bool full, bool both, const F& fn) {
  auto pick = [](bool v, const auto& next) { return v ? next(std::true_type{}) : next(std::false_type{}); };
  return pick(center, [&](auto c) {
    return pick(full, [&](auto f) { return pick(both, [&](auto b) { return fn(c, f, b); }); });
  });
}

}  // namespace

template <typename T>
int norm_forward(const nnue_ls_norm& a, cudaStream_t s) {
  const NormParams p = norm_params(a);
  const RowPlan r = plan_norm<T>(a);
  const bool center = a.kind == NNUE_LS_NORM_LAYER;
  count_launch();
  if (r.cls == kAnyWidth) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, kNumSMs * 8);
    if (center) norm_forward_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else norm_forward_kernel<T, false><<<grid, 256, 0, s>>>(p);
    return check_launch("norm_forward");
  }
  // as many blocks as stay on the SMs together, each looping over rows
  auto blocks = [&](int at_once) {
    return (unsigned)std::min<int64_t>(ceil_div(a.rows, at_once), (int64_t)kNumSMs * norm_blocks_per_sm(r));
  };
  const bool both = a.f && a.post_weight && a.h;
  const int rc = with_flags(center, a.gate_mode == kGateFull, both, [&](auto c, auto f, auto b2) {
    constexpr bool C = decltype(c)::value, F = decltype(f)::value, B = decltype(b2)::value;
    auto go = [&](auto cls) {
      constexpr int K = decltype(cls)::value;
      using H = RowShape<T, K, F, false>;
      if (r.vec)
        return launch_norm_rows(norm_forward_rows_kernel<T, 4, H::kRows, C, F, B, H::kStages, H::kThreads, H::kBlocks>,
                                blocks(H::kRows), r, H::kSlot * H::kStages, p, s);
      if constexpr (K == kNarrow) return NNUE_LS_OK;  // a row off 16 bytes is never of this class
      else
        return launch_norm_rows(norm_forward_rows_kernel<T, 1, H::kRows, C, F, B, 0, H::kThreads, 1>, blocks(H::kRows),
                                r, 0, p, s);
    };
    if (r.cls == kNarrow) return go(std::integral_constant<int, kNarrow>{});
    if (r.cls == kMiddle) return go(std::integral_constant<int, kMiddle>{});
    return go(std::integral_constant<int, kWide>{});
  });
  if (rc) return rc;
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
  if (r.cls == kAnyWidth) {
    if (center) norm_backward_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else norm_backward_kernel<T, false><<<grid, 256, 0, s>>>(p);
  } else {
    const bool both = a.f && a.post_weight && a.pre_weight && a.grad_h;
    const int rc = with_flags(center, a.gate_mode == kGateFull, both, [&](auto c, auto f, auto b2) {
      constexpr bool C = decltype(c)::value, F = decltype(f)::value, B = decltype(b2)::value;
      auto go = [&](auto cls) {
        constexpr int K = decltype(cls)::value;
        using H = RowShape<T, K, F, true>;
        if (r.vec)
          return launch_norm_rows(
              norm_backward_rows_kernel<T, 4, H::kRows, C, F, B, H::kStages, H::kThreads, H::kBlocks>, grid, r,
              H::kSlot * H::kStages, p, s);
        if constexpr (K == kNarrow) return NNUE_LS_OK;
        else
          return launch_norm_rows(norm_backward_rows_kernel<T, 1, H::kRows, C, F, B, 0, H::kThreads, 1>, grid, r, 0, p,
                                  s);
      };
      if (r.cls == kNarrow) return go(std::integral_constant<int, kNarrow>{});
      if (r.cls == kMiddle) return go(std::integral_constant<int, kMiddle>{});
      return go(std::integral_constant<int, kWide>{});
    });
    if (rc) return rc;
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

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
  p.scale_value = a.f ? a.scale_value : 1.f;  // without a block y is x
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

// Which kernel a call takes.  Up to 4096 columns, eight per thread; wider rows
// are read once per pass (forward and backward of 16384 rows in fp32: 0.49 ms
// for 4096 columns by rows, 1.53 ms for 4104 by passes; bf16 0.30 and 1.61 ms).
struct RowPlan {
  bool vec;
  int threads;  // 0: any width
};
constexpr int kMostRowThreads = 512;

template <typename T>
RowPlan plan_norm(const nnue_ls_norm& a) {
  const int64_t threads = ceil_div(a.width, 32 * kColumns) * 32;
  return RowPlan{norm_vectors<T>(a), threads <= kMostRowThreads ? (int)threads : 0};
}

// Rows at a time and rounds in flight: the slots of an SM's THREADS take at most
// 220 KB.  The backward takes two rows at a time only where they come as
// 16-byte pieces of 16-bit values; elsewhere two rows do not fit the registers.
template <typename T, int V, bool FULL, bool BACKWARD, int THREADS>
struct RowShape {
  static constexpr int kRows = V < 8 && (BACKWARD || THREADS == 1024) ? 1 : 2;
  static constexpr int kSlot = (int)sizeof(T) * kColumns * kRows * (2 + FULL + 2 * BACKWARD);  // bytes per thread
  static constexpr int kFit = 220 * 1024 / (kSlot * THREADS);
  static constexpr int kStages = kFit > 4 ? 4 : kFit;
  static_assert(kStages >= 2, "a round on its way while one is worked on");
  static constexpr size_t ring_bytes(int threads, int width) {
    const int arrays = 2 + FULL + 2 * BACKWARD;
    return (size_t)kStages * (V > 1 ? kSlot * threads : arrays * run_bytes(kRows, width, (int)sizeof(T)));
  }
  static constexpr size_t kMostBytes = ring_bytes(kMostRowThreads, kMostRowThreads * kColumns);
};

// As many blocks of `rows` rows as stay on the SMs together at `threads` each, looping over rows.
int64_t norm_row_blocks(const nnue_ls_norm& a, const RowPlan& r, int rows, int threads) {
  return std::min<int64_t>(ceil_div(std::max<int64_t>(a.rows, 1), rows), (int64_t)kNumSMs * (threads / r.threads));
}
// At most so many blocks in the backward.
int64_t norm_backward_blocks(const nnue_ls_norm& a, const RowPlan& r) {
  if (!r.threads) return std::min<int64_t>(std::max<int64_t>(a.rows, 1), kNumSMs * 4);
  return norm_row_blocks(a, r, 1, norm_backward_threads(4, true, false));
}

template <auto kernel, typename Shape>
int launch_norm_rows(int64_t grid, const RowPlan& r, const NormParams& p, cudaStream_t s) {
  const size_t smem = Shape::ring_bytes(r.threads, p.width);
  if (smem > 40 * 1024)  // 48 KB without asking, the kernels' own 3 KB at most included
    if (int rc = allow_shared<kernel>("norm", Shape::kMostBytes)) return rc;
  kernel<<<(unsigned)grid, r.threads, smem, s>>>(p);
  return NNUE_LS_OK;
}

// fn(center, full, both, more) with all as constants; more without both is looked up too.
template <typename F>
int with_flags(bool center, bool full, bool both, bool more, const F& fn) {
  auto pick = [](bool v, const auto& next) { return v ? next(std::true_type{}) : next(std::false_type{}); };
  return pick(center, [&](auto c) {
    return pick(full, [&](auto f) {
      if (!both) return fn(c, f, std::false_type{}, std::true_type{});
      return pick(more, [&](auto m) { return fn(c, f, std::true_type{}, m); });
    });
  });
}
bool has_more(const nnue_ls_norm& a) {
  return a.post_bias || a.scale || a.pre_bias || a.grad_post_bias || a.grad_scale || a.grad_pre_bias;
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
    if (center) norm_forward_kernel<T, true><<<grid, 512, 0, s>>>(p);
    else norm_forward_kernel<T, false><<<grid, 512, 0, s>>>(p);
    return check_launch("norm_forward");
  }
  const bool both = a.f && a.post_weight && a.h;
  const int rc = with_flags(center, a.gate_mode == kGateFull, both, has_more(a), [&](auto c, auto f, auto b, auto m) {
    constexpr bool C = decltype(c)::value, F = decltype(f)::value, B = decltype(b)::value, M = decltype(m)::value;
    auto launch = [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      constexpr int kThreads = norm_forward_threads(V, B, M);
      using H = RowShape<T, V, F, false, kThreads>;
      return launch_norm_rows<norm_forward_rows_kernel<T, V, H::kRows, C, F, B, M, H::kStages>, H>(
          norm_row_blocks(a, r, H::kRows, kThreads), r, p, s);
    };
    return r.vec ? launch(std::integral_constant<int, 16 / sizeof(T)>{}) : launch(std::integral_constant<int, 1>{});
  });
  if (rc) return rc;
  return check_launch("norm_forward");
}

template <typename T>
size_t norm_backward_bytes(const nnue_ls_norm& a) {
  return wants_params(a) ? align256((size_t)norm_backward_blocks(a, plan_norm<T>(a)) * 5 * a.width * 4) : 0;
}

template <typename T>
int norm_backward(const nnue_ls_norm& a, void* workspace, cudaStream_t s) {
  NormParams p = norm_params(a);
  const bool params = wants_params(a), center = a.kind == NNUE_LS_NORM_LAYER;
  p.partial = params ? static_cast<float*>(workspace) : nullptr;
  const RowPlan r = plan_norm<T>(a);
  int64_t grid = norm_backward_blocks(a, r);
  count_launch();
  if (!r.threads) {
    if (center) norm_backward_kernel<T, true><<<(unsigned)grid, 512, 0, s>>>(p);
    else norm_backward_kernel<T, false><<<(unsigned)grid, 512, 0, s>>>(p);
  } else {
    const bool both = a.f && a.post_weight && a.pre_weight && a.grad_h;
    const int rc = with_flags(center, a.gate_mode == kGateFull, both, has_more(a), [&](auto c, auto f, auto b, auto m) {
      constexpr bool C = decltype(c)::value, F = decltype(f)::value, B = decltype(b)::value, M = decltype(m)::value;
      auto launch = [&](auto vec) {
        constexpr int V = decltype(vec)::value;
        constexpr int kThreads = norm_backward_threads(V, B, M);
        using H = RowShape<T, V, F, true, kThreads>;
        grid = norm_row_blocks(a, r, H::kRows, kThreads);
        return launch_norm_rows<norm_backward_rows_kernel<T, V, H::kRows, C, F, B, M, H::kStages>, H>(grid, r, p, s);
      };
      return r.vec ? launch(std::integral_constant<int, 16 / sizeof(T)>{}) : launch(std::integral_constant<int, 1>{});
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

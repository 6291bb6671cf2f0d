// C ABI of the layer-stack operators for B200 (sm_100a).
// Declarations and contracts: include/nnue_ls.h.
//
// One translation unit: the kernels live in the *.cuh files included here.

#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "../../../include/nnue_ls.h"
#include "ls_common.cuh"
#include "ls_linear.cuh"
#include "ls_norm.cuh"
#include "ls_route.cuh"

namespace nnue_ls {
namespace {

thread_local char g_last_error[512];
std::atomic<unsigned long long> g_launches{0};

inline void count_launch(unsigned n = 1) { g_launches.fetch_add(n, std::memory_order_relaxed); }

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

int check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? NNUE_LS_OK : fail(NNUE_LS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr size_t align256(size_t n) { return (n + 255) / 256 * 256; }
constexpr int64_t kMaxDim = INT32_MAX;

bool bad_dtype(int t) { return t < NNUE_LS_F32 || t > NNUE_LS_F16; }

int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
  if (need == 0) return NNUE_LS_OK;
  if (!ws || have < need) return fail(NNUE_LS_ERR_WORKSPACE, "%s: workspace has %zu bytes, needs %zu", what, have, need);
  if (reinterpret_cast<uintptr_t>(ws) % 256) return fail(NNUE_LS_ERR_WORKSPACE, "%s: workspace not 256-byte aligned", what);
  return NNUE_LS_OK;
}

// Calls fn(T{}) with the element type of `dtype`.
template <typename F>
void with_type(int dtype, const F& fn) {
  if (dtype == NNUE_LS_F32) fn(float{});
  else if (dtype == NNUE_LS_BF16) fn(bf16{});
  else fn(f16{});
}

// ---- linear ----------------------------------------------------------------
int check_linear(const char* what, const nnue_ls_linear* a) {
  if (!a) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
  if (a->rows < 0 || a->inputs < 1 || a->outputs < 1)
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: need rows >= 0, inputs >= 1, outputs >= 1", what);
  if (a->rows > kMaxDim || a->inputs > kMaxDim || a->outputs > kMaxDim)
    return fail(NNUE_LS_ERR_UNSUPPORTED, "%s: sizes must be below 2^31", what);
  if (bad_dtype(a->dtype) || (a->bias_dtype != a->dtype && a->bias_dtype != NNUE_LS_F32))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: bad element type", what);
  if (a->activation < 0 || a->activation >= kActivations)
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, a->activation);
  return NNUE_LS_OK;
}

struct BackwardPlan {
  size_t dz, partial, total;
  int64_t parts, rows_per_part;
};

BackwardPlan plan_backward(const nnue_ls_linear& a) {
  BackwardPlan p{};
  const int64_t columns = ceil_div(a.outputs, 32);
  p.parts = std::max<int64_t>(1, std::min(ceil_div(a.rows, 64), ceil_div(kNumSMs * 8, columns)));
  p.rows_per_part = std::max<int64_t>(1, ceil_div(a.rows, p.parts));
  p.dz = a.activation == NNUE_LS_ACT_NONE ? 0 : align256((size_t)a.rows * a.outputs * (a.dtype == NNUE_LS_F32 ? 4 : 2));
  p.partial = a.grad_bias ? align256((size_t)p.parts * a.outputs * 4) : 0;
  p.total = p.dz + p.partial;
  return p;
}

template <typename T>
void simple_gemm(const T* a, int64_t sam, int64_t sak, const T* b, int64_t sbn, int64_t sbk, int64_t M, int64_t N,
                 int64_t K, const LinearEpilogue& e, cudaStream_t s) {
  count_launch();
  const dim3 grid((unsigned)ceil_div(M, kTile), (unsigned)ceil_div(N, kTile));
  simple_gemm_kernel<T><<<grid, 256, 0, s>>>(a, sam, sak, b, sbn, sbk, M, N, K, e);
}

// ---- norm --------------------------------------------------------------------
int check_norm(const char* what, const nnue_ls_norm* a) {
  if (!a) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
  if (a->rows < 0 || a->width < 1) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: need rows >= 0 and width >= 1", what);
  if (a->rows > kMaxDim || a->width > NNUE_LS_NORM_MAX_WIDTH)
    return fail(NNUE_LS_ERR_UNSUPPORTED, "%s: width must be at most %d", what, NNUE_LS_NORM_MAX_WIDTH);
  if (bad_dtype(a->dtype) || (a->params_dtype != a->dtype && a->params_dtype != NNUE_LS_F32) ||
      (a->gate_dtype != a->dtype && a->gate_dtype != NNUE_LS_F32))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: bad element type", what);
  if (a->kind != NNUE_LS_NORM_RMS && a->kind != NNUE_LS_NORM_LAYER)
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: unknown norm kind %d", what, a->kind);
  if (a->gate_mode < kGateNone || a->gate_mode > kGateFull)
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: unknown gate mode %d", what, a->gate_mode);
  if (a->rows > 0 && !a->f && (a->gate_mode != kGateNone || a->post_weight || a->scale))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: a gate, scale or norm after the block needs f", what);
  if ((a->post_bias && !a->post_weight) || (a->pre_bias && !a->pre_weight))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: a norm's bias needs its weight", what);
  if (!(a->eps >= 0.f)) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", what);
  if (a->rows > 0 && (!a->x || (a->gate_mode != kGateNone && !a->gate)))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  return NNUE_LS_OK;
}

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

int64_t norm_backward_blocks(const nnue_ls_norm& a) { return std::min<int64_t>(std::max<int64_t>(a.rows, 1), kNumSMs * 4); }

// ---- route -------------------------------------------------------------------
int check_route(const char* what, const nnue_ls_route* a) {
  if (!a) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
  if (a->rows < 0 || a->experts < 1 || a->k < 1 || a->k > a->experts)
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: need rows >= 0 and 1 <= k <= experts", what);
  if (a->rows > kMaxDim || a->experts > NNUE_LS_MAX_EXPERTS)
    return fail(NNUE_LS_ERR_UNSUPPORTED, "%s: at most %d experts", what, NNUE_LS_MAX_EXPERTS);
  if (bad_dtype(a->dtype)) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: bad element type", what);
  if (a->rows > 0 && (!a->logits || a->ld < a->experts || !a->indices || !a->gates))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: null pointer or row stride below experts", what);
  if (!a->counts || !a->loss) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  return NNUE_LS_OK;
}

int64_t route_blocks(const nnue_ls_route& a) {
  return std::min<int64_t>(std::max<int64_t>(1, ceil_div(a.rows, 8)), kNumSMs * 2);
}

RouteParams route_params(const nnue_ls_route& a) {
  RouteParams r{};
  r.logits = a.logits;
  r.valid = a.valid;
  r.indices = a.indices;
  r.gates = a.gates;
  r.counts = a.counts;
  r.loss = a.loss;
  r.unit = a.loss + 1;
  r.grad_gates = a.grad_gates;
  r.grad_loss = a.grad_loss;
  r.grad_logits = a.grad_logits;
  r.rows = a.rows;
  r.ld = a.ld;
  r.experts = a.experts;
  r.k = a.k;
  r.blocks = (int)route_blocks(a);
  r.renormalize = a.renormalize != 0;
  return r;
}

template <typename T>
void launch_route(const RouteParams& r, bool backward, cudaStream_t s) {
  count_launch();
#define NNUE_LS_ROUTE(V)                                                      \
  if (r.experts <= 32 * V) {                                                  \
    if (backward) route_backward_kernel<T, V><<<r.blocks, 256, 0, s>>>(r);    \
    else route_forward_kernel<T, V><<<r.blocks, 256, 0, s>>>(r);              \
    return;                                                                   \
  }
  NNUE_LS_ROUTE(1)
  NNUE_LS_ROUTE(2)
  NNUE_LS_ROUTE(4)
  NNUE_LS_ROUTE(8)
  NNUE_LS_ROUTE(32)
#undef NNUE_LS_ROUTE
}

}  // namespace
}  // namespace nnue_ls

using namespace nnue_ls;

extern "C" {

int nnue_ls_version(void) { return 100; }

const char* nnue_ls_last_error(void) { return g_last_error; }

uint64_t nnue_ls_launch_count(void) { return g_launches.load(); }

int nnue_ls_device_errors(uint32_t* flags, int clear) {
  if (!flags) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "device_errors: null pointer");
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(flags, g_device_errors, sizeof(*flags));
  const unsigned zero = 0;
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(g_device_errors, &zero, sizeof(zero));
  return e == cudaSuccess ? NNUE_LS_OK : fail(NNUE_LS_ERR_CUDA, "device_errors: %s", cudaGetErrorString(e));
}

size_t nnue_ls_linear_forward_workspace_size(const nnue_ls_linear*) { return 0; }

int nnue_ls_linear_forward(const nnue_ls_linear* a, void*, size_t, void* stream) {
  if (int rc = check_linear("linear_forward", a)) return rc;
  if (a->rows == 0) return NNUE_LS_OK;
  if (!a->x || !a->weight || !a->out) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_forward: null pointer");
  if (a->ldx < a->inputs || a->ldw < a->inputs || (a->residual && a->ldr < a->outputs))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_forward: row stride below the row length");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  LinearEpilogue e{a->bias, a->residual, a->out, a->act_grad, a->ldr, a->outputs, a->activation,
                   a->bias_dtype == NNUE_LS_F32};
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    simple_gemm<T>(static_cast<const T*>(a->x), a->ldx, 1, static_cast<const T*>(a->weight), a->ldw, 1, a->rows,
                   a->outputs, a->inputs, e, s);
  });
  return check_launch("linear_forward");
}

size_t nnue_ls_linear_backward_workspace_size(const nnue_ls_linear* a) {
  return check_linear("linear_backward", a) ? 0 : plan_backward(*a).total;
}

int nnue_ls_linear_backward(const nnue_ls_linear* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_linear("linear_backward", a)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->rows > 0) {
    if (!a->grad_out || (a->activation != NNUE_LS_ACT_NONE && !a->act_grad) || (a->grad_x && !a->weight) ||
        (a->grad_weight && !a->x))
      return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_backward: null pointer");
    if (a->ldg < a->outputs || (a->grad_x && a->ldw < a->inputs) || (a->grad_weight && a->ldx < a->inputs))
      return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_backward: row stride below the row length");
  }
  const BackwardPlan p = plan_backward(*a);
  if (int rc = check_workspace("linear_backward", workspace, workspace_bytes, p.total)) return rc;
  char* ws = static_cast<char*>(workspace);
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    const T* dz = static_cast<const T*>(a->grad_out);
    int64_t lddz = a->ldg;
    float* partial = p.partial ? reinterpret_cast<float*>(ws + p.dz) : nullptr;
    if (p.dz || partial) {
      T* out = p.dz ? reinterpret_cast<T*>(ws) : nullptr;
      count_launch();
      dz_bias_kernel<T><<<dim3((unsigned)ceil_div(a->outputs, 32), (unsigned)p.parts), dim3(32, 8), 0, s>>>(
          dz, lddz, p.dz ? static_cast<const T*>(a->act_grad) : nullptr, out, partial, a->rows, a->outputs,
          p.rows_per_part);
      if (p.dz) dz = out, lddz = a->outputs;
    }
    if (partial) {
      count_launch();
      column_total_kernel<T><<<(unsigned)ceil_div(a->outputs, 32), dim3(32, 8), 0, s>>>(
          partial, p.parts, a->outputs, a->grad_bias, a->bias_dtype == NNUE_LS_F32);
    }
    LinearEpilogue e{};
    if (a->grad_x && a->rows > 0) {
      e.out = a->grad_x;
      e.ldo = a->inputs;
      simple_gemm<T>(dz, lddz, 1, static_cast<const T*>(a->weight), 1, a->ldw, a->rows, a->inputs, a->outputs, e, s);
    }
    if (a->grad_weight) {
      e.out = a->grad_weight;
      e.ldo = a->inputs;
      simple_gemm<T>(dz, 1, lddz, static_cast<const T*>(a->x), 1, a->ldx, a->outputs, a->inputs, a->rows, e, s);
    }
  });
  return check_launch("linear_backward");
}

int nnue_ls_norm_forward(const nnue_ls_norm* a, void* stream) {
  if (int rc = check_norm("norm_forward", a)) return rc;
  if (a->rows == 0) return NNUE_LS_OK;
  if ((a->f && !a->y) || (a->pre_weight && !a->h) || (a->h && !a->pre_weight))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "norm_forward: null pointer, or h without pre_weight");
  const NormParams p = norm_params(*a);
  const unsigned grid = (unsigned)std::min<int64_t>(a->rows, kNumSMs * 8);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    count_launch();
    if (a->kind == NNUE_LS_NORM_LAYER) norm_forward_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else norm_forward_kernel<T, false><<<grid, 256, 0, s>>>(p);
  });
  return check_launch("norm_forward");
}

size_t nnue_ls_norm_backward_workspace_size(const nnue_ls_norm* a) {
  if (check_norm("norm_backward", a) || !wants_params(*a)) return 0;
  return align256((size_t)norm_backward_blocks(*a) * 5 * a->width * 4);
}

int nnue_ls_norm_backward(const nnue_ls_norm* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_norm("norm_backward", a)) return rc;
  if (a->rows > 0 && !a->stats) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "norm_backward: null pointer");
  if (a->rows > 0 && !a->f && (a->grad_f || a->grad_gate || a->grad_post_weight || a->grad_post_bias || a->grad_scale))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "norm_backward: gradients of a branch that is absent");
  if (int rc = check_workspace("norm_backward", workspace, workspace_bytes, nnue_ls_norm_backward_workspace_size(a)))
    return rc;
  NormParams p = norm_params(*a);
  const bool params = wants_params(*a);
  p.partial = params ? static_cast<float*>(workspace) : nullptr;
  const unsigned grid = (unsigned)norm_backward_blocks(*a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    count_launch();
    if (a->kind == NNUE_LS_NORM_LAYER) norm_backward_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else norm_backward_kernel<T, false><<<grid, 256, 0, s>>>(p);
    if (params) {
      const NormTotals out{{a->grad_post_weight, a->grad_post_bias, a->grad_scale, a->grad_pre_weight, a->grad_pre_bias}};
      count_launch();
      norm_totals_kernel<T><<<dim3((unsigned)ceil_div(a->width, 32), 5), dim3(32, 8), 0, s>>>(
          p.partial, (int)grid, a->width, out, p.params_f32);
    }
  });
  return check_launch("norm_backward");
}

size_t nnue_ls_route_forward_workspace_size(const nnue_ls_route* a) {
  if (check_route("route_forward", a)) return 0;
  return align256((size_t)route_blocks(*a) * (2 * a->experts + 1) * 4);
}

int nnue_ls_route_forward(const nnue_ls_route* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_route("route_forward", a)) return rc;
  if (int rc = check_workspace("route_forward", workspace, workspace_bytes, nnue_ls_route_forward_workspace_size(a)))
    return rc;
  RouteParams r = route_params(*a);
  r.partial_p = static_cast<float*>(workspace);
  r.partial_count = reinterpret_cast<int32_t*>(r.partial_p + (int64_t)r.blocks * r.experts);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  with_type(a->dtype, [&](auto t) { launch_route<decltype(t)>(r, false, s); });
  count_launch();
  route_totals_kernel<<<1, 256, 0, s>>>(r);
  return check_launch("route_forward");
}

int nnue_ls_route_backward(const nnue_ls_route* a, void* stream) {
  if (int rc = check_route("route_backward", a)) return rc;
  if (a->rows == 0) return NNUE_LS_OK;
  if (!a->grad_logits) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "route_backward: null pointer");
  const RouteParams r = route_params(*a);
  with_type(a->dtype, [&](auto t) { launch_route<decltype(t)>(r, true, static_cast<cudaStream_t>(stream)); });
  return check_launch("route_backward");
}

}  // extern "C"

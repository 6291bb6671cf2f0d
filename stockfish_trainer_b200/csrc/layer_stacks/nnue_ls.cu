// C ABI of the layer-stack operators for B200 (sm_100a).
// Declarations and contracts: include/nnue_ls.h.
//
// Checks of arguments; the operators are compiled in files of their own.

#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "../../../include/nnue_ls.h"
#include "ls_common.cuh"
#include "ls_host.cuh"

namespace nnue_ls {

static thread_local char g_last_error[512];
static std::atomic<unsigned long long> g_launches{0};
static std::atomic<uint64_t> g_wait_limit_ns{4000000000ull};

void count_launch() { g_launches.fetch_add(1, std::memory_order_relaxed); }
uint64_t wait_limit_ns() { return g_wait_limit_ns.load(std::memory_order_relaxed); }

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

namespace {

// Whether some pointer (null is fine) is not on a multiple of `to` bytes: a power of two.
bool off_boundary(size_t to, std::initializer_list<const void*> pointers) {
  uintptr_t all = 0;
  for (const void* p : pointers) all |= reinterpret_cast<uintptr_t>(p);
  return (all & (to - 1)) != 0;
}
size_t bytes_of(int dtype) { return dtype == NNUE_LS_F32 ? 4 : 2; }

// ---- linear ----------------------------------------------------------------
int check_linear(const char* what, const nnue_ls_linear* a) {
  if (!a) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
  if (a->rows < 0 || a->inputs < 1 || a->outputs < 1)
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: need rows >= 0, inputs >= 1, outputs >= 1", what);
  if (a->rows > kMaxDim || a->inputs > kMaxDim || a->outputs > kMaxDim)
    return fail(NNUE_LS_ERR_UNSUPPORTED, "%s: sizes must be below 2^30", what);
  if (bad_dtype(a->dtype) || (a->bias_dtype != a->dtype && a->bias_dtype != NNUE_LS_F32))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: bad element type", what);
  if (a->activation < 0 || a->activation > NNUE_LS_ACT_GELU)
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, a->activation);
  if (off_boundary(bytes_of(a->dtype), {a->x, a->weight, a->residual, a->out, a->act_grad, a->grad_out, a->grad_x,
                                        a->grad_weight}) ||
      off_boundary(bytes_of(a->bias_dtype), {a->bias, a->grad_bias}))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  if (off_boundary(256, {a->x_packed, a->weight_packed}))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: x_packed or weight_packed not 256-byte aligned", what);
  return NNUE_LS_OK;
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
  if (a->gate_mode < NNUE_LS_GATE_NONE || a->gate_mode > NNUE_LS_GATE_FULL)
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: unknown gate mode %d", what, a->gate_mode);
  if (a->rows > 0 && !a->f && (a->gate_mode != NNUE_LS_GATE_NONE || a->post_weight || a->scale))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: a gate, scale or norm after the block needs f", what);
  if ((a->post_bias && !a->post_weight) || (a->pre_bias && !a->pre_weight))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: a norm's bias needs its weight", what);
  if (!(a->eps >= 0.f)) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", what);
  if (a->rows > 0 && (!a->x || (a->gate_mode != NNUE_LS_GATE_NONE && !a->gate)))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  const bool row_gate = a->gate_mode == NNUE_LS_GATE_ROW;
  if (off_boundary(bytes_of(a->dtype), {a->x, a->f, a->y, a->h, a->grad_y, a->grad_h, a->grad_x, a->grad_f}) ||
      off_boundary(bytes_of(row_gate ? a->gate_dtype : a->dtype), {a->gate, a->grad_gate}) ||
      off_boundary(bytes_of(a->params_dtype),
                   {a->post_weight, a->post_bias, a->scale, a->pre_weight, a->pre_bias, a->grad_post_weight,
                    a->grad_post_bias, a->grad_scale, a->grad_pre_weight, a->grad_pre_bias}))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  if (off_boundary(16, {a->stats})) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: stats not 16-byte aligned", what);
  return NNUE_LS_OK;
}

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
  if (off_boundary(bytes_of(a->dtype), {a->logits, a->grad_logits}) || off_boundary(8, {a->indices, a->counts}) ||
      off_boundary(4, {a->gates, a->loss, a->grad_gates, a->grad_loss}))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its elements", what);
  return NNUE_LS_OK;
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
  *flags = 0;
  if (e == cudaSuccess) e = linear_device_errors<float>(flags, clear != 0);
  if (e == cudaSuccess) e = linear_device_errors<bf16>(flags, clear != 0);
  if (e == cudaSuccess) e = linear_device_errors<f16>(flags, clear != 0);
  if (e == cudaSuccess) e = route_device_errors(flags, clear != 0);
  return e == cudaSuccess ? NNUE_LS_OK : fail(NNUE_LS_ERR_CUDA, "device_errors: %s", cudaGetErrorString(e));
}

uint64_t nnue_ls_set_wait_limit(uint64_t ns) { return g_wait_limit_ns.exchange(ns); }

size_t nnue_ls_linear_saved_layout(const nnue_ls_linear* a, int32_t parts, int64_t offsets[3]) {
  if (!offsets) return 0;
  offsets[0] = offsets[1] = offsets[2] = -1;
  if (check_linear("linear_saved_layout", a) || a->rows == 0) return 0;
  return with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    const size_t bytes[3] = {
        parts & 1 && a->activation != NNUE_LS_ACT_NONE ? (size_t)a->rows * a->outputs * sizeof(T) : 0,
        parts & 2 ? linear_packed_bytes<T>(*a, false) : 0, parts & 4 ? linear_packed_bytes<T>(*a, true) : 0};
    size_t total = 0;
    for (int i = 0; i < 3; ++i) {
      if (!bytes[i]) continue;
      offsets[i] = (int64_t)total;
      total += align256(bytes[i]);
    }
    return total;
  });
}

size_t nnue_ls_linear_forward_workspace_size(const nnue_ls_linear* a) {
  if (check_linear("linear_forward", a) || a->rows == 0) return 0;
  return with_type(a->dtype, [&](auto t) { return linear_forward_bytes<decltype(t)>(*a); });
}

int nnue_ls_linear_forward(const nnue_ls_linear* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_linear("linear_forward", a)) return rc;
  if (a->rows == 0) return NNUE_LS_OK;
  if (!a->x || !a->weight || !a->out) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_forward: null pointer");
  if (a->ldx < a->inputs || a->ldw < a->inputs || (a->residual && a->ldr < a->outputs))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_forward: row stride below the row length");
  return with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    if ((a->x_packed && !linear_packed_bytes<T>(*a, false)) || (a->weight_packed && !linear_packed_bytes<T>(*a, true)))
      return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_forward: a buffer for an operand that is read as it lies");
    if (int rc = check_workspace("linear_forward", workspace, workspace_bytes, linear_forward_bytes<T>(*a))) return rc;
    return linear_forward<T>(*a, static_cast<char*>(workspace), static_cast<cudaStream_t>(stream));
  });
}

size_t nnue_ls_linear_backward_workspace_size(const nnue_ls_linear* a) {
  if (check_linear("linear_backward", a)) return 0;
  return with_type(a->dtype, [&](auto t) { return linear_backward_bytes<decltype(t)>(*a); });
}

int nnue_ls_linear_backward(const nnue_ls_linear* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_linear("linear_backward", a)) return rc;
  if (a->rows > 0) {
    if (!a->grad_out || (a->activation != NNUE_LS_ACT_NONE && !a->act_grad) || (a->grad_x && !a->weight && !a->weight_packed) ||
        (a->grad_weight && !a->x && !a->x_packed))
      return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_backward: null pointer");
    if (a->ldg < a->outputs || (a->grad_x && !a->weight_packed && a->ldw < a->inputs) || (a->grad_weight && !a->x_packed && a->ldx < a->inputs))
      return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "linear_backward: row stride below the row length");
  }
  return with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    if (int rc = check_workspace("linear_backward", workspace, workspace_bytes, linear_backward_bytes<T>(*a))) return rc;
    return linear_backward<T>(*a, static_cast<char*>(workspace), static_cast<cudaStream_t>(stream));
  });
}

int nnue_ls_norm_forward(const nnue_ls_norm* a, void* stream) {
  if (int rc = check_norm("norm_forward", a)) return rc;
  if (a->rows == 0) return NNUE_LS_OK;
  if ((a->f && !a->y) || (a->pre_weight && !a->h) || (a->h && !a->pre_weight))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "norm_forward: null pointer, or h without pre_weight");
  return with_type(a->dtype,
                   [&](auto t) { return norm_forward<decltype(t)>(*a, static_cast<cudaStream_t>(stream)); });
}

size_t nnue_ls_norm_backward_workspace_size(const nnue_ls_norm* a) {
  if (check_norm("norm_backward", a)) return 0;
  return with_type(a->dtype, [&](auto t) { return norm_backward_bytes<decltype(t)>(*a); });
}

int nnue_ls_norm_backward(const nnue_ls_norm* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_norm("norm_backward", a)) return rc;
  if (a->rows > 0 && !a->stats) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "norm_backward: null pointer");
  if (a->rows > 0 && !a->f && (a->grad_f || a->grad_gate || a->grad_post_weight || a->grad_post_bias || a->grad_scale))
    return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "norm_backward: gradients of a branch that is absent");
  return with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    if (int rc = check_workspace("norm_backward", workspace, workspace_bytes, norm_backward_bytes<T>(*a))) return rc;
    return norm_backward<T>(*a, workspace, static_cast<cudaStream_t>(stream));
  });
}

size_t nnue_ls_route_forward_workspace_size(const nnue_ls_route* a) {
  return check_route("route_forward", a) ? 0 : route_forward_bytes(*a);
}

int nnue_ls_route_forward(const nnue_ls_route* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_route("route_forward", a)) return rc;
  if (int rc = check_workspace("route_forward", workspace, workspace_bytes, route_forward_bytes(*a))) return rc;
  return with_type(
      a->dtype, [&](auto t) { return route_forward<decltype(t)>(*a, workspace, static_cast<cudaStream_t>(stream)); });
}

int nnue_ls_route_backward(const nnue_ls_route* a, void* stream) {
  if (int rc = check_route("route_backward", a)) return rc;
  if (a->rows == 0) return NNUE_LS_OK;
  if (!a->grad_logits) return fail(NNUE_LS_ERR_INVALID_ARGUMENT, "route_backward: null pointer");
  return with_type(a->dtype,
                   [&](auto t) { return route_backward<decltype(t)>(*a, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"

// Host helpers shared by the operators' launch code: errors, launch counting.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "../../../include/nnue_ls.h"

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

bool bad_dtype(int t) { return t < NNUE_LS_F32 || t > NNUE_LS_F16; }

int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
  if (need == 0) return NNUE_LS_OK;
  if (!ws || have < need)
    return fail(NNUE_LS_ERR_WORKSPACE, "%s: workspace has %zu bytes, needs %zu", what, ws ? have : (size_t)0, need);
  if (reinterpret_cast<uintptr_t>(ws) % 256)
    return fail(NNUE_LS_ERR_WORKSPACE, "%s: workspace not 256-byte aligned", what);
  return NNUE_LS_OK;
}

// Calls fn(T{}) with the element type of `dtype`.
template <typename F>
auto with_type(int dtype, const F& fn) {
  if (dtype == NNUE_LS_F32) return fn(float{});
  if (dtype == NNUE_LS_BF16) return fn(bf16{});
  return fn(f16{});
}

}  // namespace
}  // namespace nnue_ls

// Host helpers shared by the operators' launch code: errors, launch counting.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../../include/nnue_ls.h"
#include "ls_common.cuh"

namespace nnue_ls {

// One per library (nnue_ls.cu).
void count_launch();
uint64_t wait_limit_ns();  // of a matrix kernel's waits
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int check_launch(const char* what);  // the last launch's error, if any

namespace {

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr size_t align256(size_t n) { return (n + 255) / 256 * 256; }

constexpr int64_t kMaxDim = (1 << 30) - 1;

inline bool bad_dtype(int t) { return t < NNUE_LS_F32 || t > NNUE_LS_F16; }

inline int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
  if (need == 0) return NNUE_LS_OK;
  if (!ws || have < need)
    return fail(NNUE_LS_ERR_WORKSPACE, "%s: workspace has %zu bytes, needs %zu", what, ws ? have : (size_t)0, need);
  if (reinterpret_cast<uintptr_t>(ws) % 256)
    return fail(NNUE_LS_ERR_WORKSPACE, "%s: workspace not 256-byte aligned", what);
  return NNUE_LS_OK;
}

// Allows `kernel` up to `most` bytes of dynamic shared memory, once per device: the limit is the kernel's on that device,
// whoever calls it, so no call may set it to its own need.
template <auto kernel>
int allow_shared(const char* what, size_t most) {
  static std::atomic<uint64_t> ready{0};  // one bit per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch(what);
  if (dev < 64 && ready.load(std::memory_order_acquire) >> dev & 1) return NNUE_LS_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  if (e != cudaSuccess) return fail(NNUE_LS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
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

// The operators' entry points per element type, each compiled in a file of its
// own (linear_*.cu, norm_*.cu; route.cu), and the device error words of those files.
template <typename T>
size_t linear_packed_bytes(const nnue_ls_linear& a, bool weight);
template <typename T>
size_t linear_forward_bytes(const nnue_ls_linear& a);
template <typename T>
int linear_forward(const nnue_ls_linear& a, char* ws, cudaStream_t s);
template <typename T>
size_t linear_backward_bytes(const nnue_ls_linear& a);
template <typename T>
int linear_backward(const nnue_ls_linear& a, char* ws, cudaStream_t s);
template <typename T>
cudaError_t linear_device_errors(unsigned* flags, bool clear);
template <typename T>
int norm_forward(const nnue_ls_norm& a, cudaStream_t s);
template <typename T>
size_t norm_backward_bytes(const nnue_ls_norm& a);
template <typename T>
int norm_backward(const nnue_ls_norm& a, void* workspace, cudaStream_t s);
size_t route_forward_bytes(const nnue_ls_route& a);
template <typename T>
int route_forward(const nnue_ls_route& a, void* workspace, cudaStream_t s);
template <typename T>
int route_backward(const nnue_ls_route& a, cudaStream_t s);
cudaError_t route_device_errors(unsigned* flags, bool clear);

}  // namespace nnue_ls

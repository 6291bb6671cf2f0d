// The router: how rows are spread over lanes and blocks, and the launches.
#include <algorithm>

#include "ls_host.cuh"
#include "ls_route.cuh"

namespace nnue_ls {
namespace {

int lanes_per_row(int experts) {
  int g = 1;
  while (g < 32 && g * 8 < experts) g *= 2;
  return g;
}

// Two blocks per SM at most; one block, which forms the totals itself, for up
// to two rounds of its rows (8 experts: 24 rows 4.3 us and 512 rows 6.2 us in one
// launch; 520 rows in two 4.0 and 2.5 us, and the second launch's gap).
int64_t route_blocks(const nnue_ls_route& a) {
  const int64_t per_block = a.experts > 256 ? 4 : 256 / lanes_per_row(a.experts), need = ceil_div(a.rows, per_block);
  return need <= 2 ? 1 : std::min<int64_t>(need, kNumSMs * 2);
}

template <typename T>
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
  const int w = std::min<int>(16 / sizeof(T), 8);
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  r.vec = a.experts % w == 0 && a.ld % w == 0 && aligned(a.logits);
  r.vec_out = a.experts % w == 0 && aligned(a.grad_logits);
  return r;
}

template <typename T, int V, int G>
void launch_route(const RouteParams& r, bool backward, cudaStream_t s) {
  if (backward) {
    const int64_t blocks = std::min<int64_t>(ceil_div(r.rows, 256 / G), kNumSMs * 8);
    route_backward_kernel<T, V, G><<<(unsigned)blocks, 256, 0, s>>>(r);
  } else {
    route_forward_kernel<T, V, G><<<r.blocks, 32 * route_warps(V, G), 0, s>>>(r);
  }
}

template <typename T>
void launch_route(const RouteParams& r, bool backward, cudaStream_t s) {
  count_launch();
  if (r.experts > 256) return launch_route<T, 32, 32>(r, backward, s);
  switch (lanes_per_row(r.experts)) {
    case 1: return launch_route<T, 8, 1>(r, backward, s);
    case 2: return launch_route<T, 8, 2>(r, backward, s);
    case 4: return launch_route<T, 8, 4>(r, backward, s);
    case 8: return launch_route<T, 8, 8>(r, backward, s);
    case 16: return launch_route<T, 8, 16>(r, backward, s);
    default: return launch_route<T, 8, 32>(r, backward, s);
  }
}

}  // namespace

size_t route_forward_bytes(const nnue_ls_route& a) {
  return align256((size_t)route_blocks(a) * (2 * a.experts + 1) * 4);
}

template <typename T>
int route_forward(const nnue_ls_route& a, void* workspace, cudaStream_t s) {
  RouteParams r = route_params<T>(a);
  r.partial_p = static_cast<float*>(workspace);
  r.partial_count = reinterpret_cast<int32_t*>(r.partial_p + (int64_t)r.blocks * r.experts);
  launch_route<T>(r, false, s);
  if (r.blocks > 1) {
    count_launch();
    route_totals_kernel<<<1, 1024, 0, s>>>(r);
  }
  return check_launch("route_forward");
}

template <typename T>
int route_backward(const nnue_ls_route& a, cudaStream_t s) {
  launch_route<T>(route_params<T>(a), true, s);
  return check_launch("route_backward");
}

cudaError_t route_device_errors(unsigned* flags, bool clear) { return read_device_errors(flags, clear); }

template int route_forward<float>(const nnue_ls_route&, void*, cudaStream_t);
template int route_forward<bf16>(const nnue_ls_route&, void*, cudaStream_t);
template int route_forward<f16>(const nnue_ls_route&, void*, cudaStream_t);
template int route_backward<float>(const nnue_ls_route&, cudaStream_t);
template int route_backward<bf16>(const nnue_ls_route&, cudaStream_t);
template int route_backward<f16>(const nnue_ls_route&, cudaStream_t);

}  // namespace nnue_ls

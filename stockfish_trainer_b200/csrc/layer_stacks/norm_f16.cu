// The norms around a residual block on f16 tensors.
#include "ls_norm_host.cuh"

namespace nnue_ls {
template int norm_forward<f16>(const nnue_ls_norm&, cudaStream_t);
template size_t norm_backward_bytes<f16>(const nnue_ls_norm&);
template int norm_backward<f16>(const nnue_ls_norm&, void*, cudaStream_t);
}  // namespace nnue_ls

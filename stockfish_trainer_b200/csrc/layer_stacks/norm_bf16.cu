// The norms around a residual block on bf16 tensors.
#include "ls_norm_host.cuh"

namespace nnue_ls {
template int norm_forward<bf16>(const nnue_ls_norm&, cudaStream_t);
template size_t norm_backward_bytes<bf16>(const nnue_ls_norm&);
template int norm_backward<bf16>(const nnue_ls_norm&, void*, cudaStream_t);
}  // namespace nnue_ls

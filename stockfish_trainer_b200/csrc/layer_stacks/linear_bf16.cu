// The linear layer on bf16 tensors.
#include "ls_linear_host.cuh"

namespace nnue_ls {
template size_t linear_packed_bytes<bf16>(const nnue_ls_linear&, bool);
template size_t linear_forward_bytes<bf16>(const nnue_ls_linear&);
template int linear_forward<bf16>(const nnue_ls_linear&, char*, cudaStream_t);
template size_t linear_backward_bytes<bf16>(const nnue_ls_linear&);
template int linear_backward<bf16>(const nnue_ls_linear&, char*, cudaStream_t);
template cudaError_t linear_device_errors<bf16>(unsigned*, bool);
}  // namespace nnue_ls

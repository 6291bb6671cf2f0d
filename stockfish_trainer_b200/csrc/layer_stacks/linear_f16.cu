// The linear layer on f16 tensors.
#include "ls_linear_host.cuh"

namespace nnue_ls {
template size_t linear_packed_bytes<f16>(const nnue_ls_linear&, bool);
template size_t linear_forward_bytes<f16>(const nnue_ls_linear&);
template int linear_forward<f16>(const nnue_ls_linear&, char*, cudaStream_t);
template size_t linear_backward_bytes<f16>(const nnue_ls_linear&);
template int linear_backward<f16>(const nnue_ls_linear&, char*, cudaStream_t);
template cudaError_t linear_device_errors<f16>(unsigned*, bool);
}  // namespace nnue_ls

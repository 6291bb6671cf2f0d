// The linear layer on fp32 tensors.
#include "ls_linear_host.cuh"

namespace nnue_ls {
template size_t linear_packed_bytes<float>(const nnue_ls_linear&, bool);
template size_t linear_forward_bytes<float>(const nnue_ls_linear&);
template int linear_forward<float>(const nnue_ls_linear&, char*, cudaStream_t);
template size_t linear_backward_bytes<float>(const nnue_ls_linear&);
template int linear_backward<float>(const nnue_ls_linear&, char*, cudaStream_t);
template cudaError_t linear_device_errors<float>(unsigned*, bool);
}  // namespace nnue_ls

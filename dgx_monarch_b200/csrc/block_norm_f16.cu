// The block norm's row kernels for fp16 tensors.
#include "block_norm.cuh"

namespace dgxm {

template int bn_launch<false, __half>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);
template int bn_launch<true, __half>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);

}  // namespace dgxm

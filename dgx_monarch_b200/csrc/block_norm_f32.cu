// The block norm's row kernels for fp32 tensors.
#include "block_norm.cuh"

namespace dgxm {

template int bn_launch<false, float>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);
template int bn_launch<true, float>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);

}  // namespace dgxm

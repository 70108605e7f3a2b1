// The block norm's row kernels for bf16 tensors.
#include "block_norm.cuh"

namespace dgxm {

template int bn_launch<false, __nv_bfloat16>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);
template int bn_launch<true, __nv_bfloat16>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);

}  // namespace dgxm

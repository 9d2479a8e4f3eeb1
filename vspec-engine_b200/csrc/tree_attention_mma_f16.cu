// tree_attention_mma_f16.cu -- the warp-MMA tree attention kernels over f16 pages.
#include "tree_attention_mma.cuh"

namespace vb200 {

template cudaError_t tree_mma_launch<kTreeF16>(const TreeParams&, int, cudaStream_t);

}  // namespace vb200

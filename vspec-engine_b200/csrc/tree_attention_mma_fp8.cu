// tree_attention_mma_fp8.cu -- the warp-MMA tree attention kernels over fp8 pages.
#include "tree_attention_mma.cuh"

namespace vb200 {

template cudaError_t tree_mma_launch<kTreeFp8>(const TreeParams&, int, cudaStream_t);

}  // namespace vb200

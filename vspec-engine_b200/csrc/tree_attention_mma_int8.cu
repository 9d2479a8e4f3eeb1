// tree_attention_mma_int8.cu -- the warp-MMA tree attention kernels over int8 pages.
#include "tree_attention_mma.cuh"

namespace vb200 {

template cudaError_t tree_mma_launch<kTreeInt8>(const TreeParams&, int, cudaStream_t);

}  // namespace vb200

// tree_attention_tc_int8.cu -- the tcgen05 tree attention kernels over int8 pages.
#include "tree_attention_tc.cuh"

namespace vb200 {

template cudaError_t tree_tc_launch<kTreeInt8>(const TcParams&, int, cudaStream_t);

}  // namespace vb200

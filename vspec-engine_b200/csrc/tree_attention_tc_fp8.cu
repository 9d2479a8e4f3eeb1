// tree_attention_tc_fp8.cu -- the tcgen05 tree attention kernels over fp8 pages.
#include "tree_attention_tc.cuh"

namespace vb200 {

template cudaError_t tree_tc_launch<kTreeFp8>(const TcParams&, int, cudaStream_t);

}  // namespace vb200

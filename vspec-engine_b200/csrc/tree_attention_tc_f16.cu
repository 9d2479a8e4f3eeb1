// tree_attention_tc_f16.cu -- the tcgen05 tree attention kernels over f16 pages.
#include "tree_attention_tc.cuh"

namespace vb200 {

template cudaError_t tree_tc_launch<kTreeF16>(const TcParams&, int, cudaStream_t);

}  // namespace vb200

// The kernels of kan_block_ring.cuh for a bfloat16 stream.
#include "kan_block_ring.cuh"

namespace kanb200 {

template cudaError_t ring_forward<__nv_bfloat16>(const kanb200_block_args&, const RingPlan&, cudaStream_t);
template cudaError_t ring_backward<__nv_bfloat16>(const kanb200_block_args&, const RingPlan&, const BackwardSlabs&, cudaStream_t);

}  // namespace kanb200

// The kernels of kan_block_ring.cuh for a float64 stream.
#include "kan_block_ring.cuh"

namespace kanb200 {

template cudaError_t ring_forward<double>(const kanb200_block_args&, const RingPlan&, cudaStream_t);
template cudaError_t ring_backward<double>(const kanb200_block_args&, const RingPlan&, const BackwardSlabs&, cudaStream_t);

}  // namespace kanb200

// Launcher interface of the operators around a KAN layer (kan_block.cu, kan_pack.cu): the norm in front of it, the
// gated residual connection behind it, and 8-bit checkpoints.  The argument structure is that of the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/kan_b200.h"

namespace kanb200 {

constexpr int kActNone = KANB200_ACT_NONE, kActSigmoid = KANB200_ACT_SIGMOID, kActSilu = KANB200_ACT_SILU;
constexpr int kNormNone = KANB200_NORM_NONE, kNormRms = KANB200_NORM_RMS, kNormLayer = KANB200_NORM_LAYER;
constexpr int kPackNone = KANB200_PACK_NONE, kPackInt8 = KANB200_PACK_INT8, kPackE4m3 = KANB200_PACK_E4M3;
constexpr int kPackGroup = KANB200_PACK_GROUP;

int block_columns_at_once(const kanb200_block_args& a, bool backward);
cudaError_t block_forward(const kanb200_block_args& a, cudaStream_t st);
size_t block_backward_workspace(const kanb200_block_args& a);
cudaError_t block_backward(const kanb200_block_args& a, void* ws, size_t ws_bytes, cudaStream_t st);

cudaError_t pack_activation(int dtype, int format, const void* x, int64_t x_stride, void* codes, void* scales,
                            int64_t rows, int64_t width, cudaStream_t st);
cudaError_t unpack_activation(int dtype, int format, const void* codes, const void* scales, void* x, int64_t rows,
                              int64_t width, cudaStream_t st);

}  // namespace kanb200

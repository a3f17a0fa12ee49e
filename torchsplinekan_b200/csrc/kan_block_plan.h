// How a call of kan_block.cu is spread over the GPU: host decisions, read by the kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "kan_block.h"

namespace kanb200 {

constexpr int kSms = 148;

// Sums over rows that the backward returns, one slab each.
enum { kSumScale, kSumPostWeight, kSumPostBias, kSumNextWeight, kSumNextBias, kColumnSums };

struct BackwardSlabs {
    void* column[kColumnSums];       // [slab rows, width] each; NULL = not needed
    void* gate;                      // [items, width]: per-item sums of dgate (the output itself with one item per span)
};

// Rows are dealt out as items of `chunk` consecutive rows.  With a shared gate an item stays within the rows of one gate
// row (a span), so that its gate is read once and its share of dgate leaves as one slab row.
struct RowSplit {
    bool shared;
    int64_t span, per_span, items;   // rows per gate row, items per span
    int chunk;
};

struct RingPlan : RowSplit {
    int64_t teams;                   // of the launch
    int lanes;                       // 8, 16 or 32
    int warps;                       // of a team, in one block (lanes == 32)
    int teams_per_block, cluster;
    int threads, blocks, stages, stage_bytes;
    int at_dout, at_dh, at_x, at_next_stats, at_y, at_gate, at_post_stats;      // backward: tensors within a stage
    bool vec, big;
};

// Registers: 256-thread blocks may use 128 (two to an SM), larger ones 64 (float64: 128, half as many threads).
template <typename S> constexpr int ring_max_threads(bool big) {
    return !big ? 256 : std::is_same<S, double>::value ? 512 : 1024;
}

template <typename S> cudaError_t ring_forward(const kanb200_block_args& a, const RingPlan& p, cudaStream_t st);
template <typename S>
cudaError_t ring_backward(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st);

}  // namespace kanb200

// How a call of kan_block.cu is spread over the GPU: host decisions, read by the kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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
    int lanes;                       // 4, 8, 16 or 32
    int warps;                       // of a team, in one block (lanes == 32)
    int teams_per_block, cluster;
    int threads, blocks, stages, stage_bytes;
    bool vec, big;
};

// Chunks of four columns per thread.  More share the cost of a row among more elements, fewer leave registers for the sums
// that are parameter gradients (20 V floats behind a branch, 8 V behind a norm alone).
constexpr int ring_chunks(bool backward, bool branch, bool f64) { return backward && branch ? (f64 ? 1 : 2) : f64 ? 2 : 4; }
// Threads of a block and blocks to an SM, which bound the registers: 512 threads to an SM may use 128 each.
constexpr int ring_threads(bool big) { return big ? 512 : 256; }
constexpr int ring_blocks(bool backward, bool branch, bool big, bool f64) {
    return big ? 1 : backward || branch || f64 ? 2 : 3;
}

// Bytes of one tensor in a stage of the ring: elements of less than 4 bytes that cannot be copied four at a time are not
// there.  Values that may come as codes need room for either.
constexpr int ring_bytes(int element, bool vec, int chunks, int threads) {
    return vec || element >= 4 ? 4 * element * chunks * threads : 0;
}
constexpr int ring_kept_bytes(int element, bool vec, int chunks, int threads, int branch) {
    return ring_bytes(element, vec, chunks, threads) > (4 + branch) * chunks * threads
               ? ring_bytes(element, vec, chunks, threads) : (4 + branch) * chunks * threads;
}
// A stage of the backward; what is not part of every call comes last.
template <bool NEXT, bool BRANCH, int V, int T, bool VEC, int S, int B> struct BackwardStage {
    static constexpr int dh = 0;
    static constexpr int x = dh + (NEXT ? ring_bytes(B, VEC, V, T) : 0);
    static constexpr int next_stats = x + (NEXT ? ring_kept_bytes(S, VEC, V, T, B) : 0);
    static constexpr int y = next_stats + (NEXT ? 2 * B * T : 0);
    static constexpr int post_stats = y + (BRANCH ? ring_kept_bytes(B, VEC, V, T, B) : 0);
    static constexpr int dout = post_stats + (BRANCH ? 2 * B * T : 0);
    static constexpr int gate = dout + ring_bytes(S, VEC, V, T);
    static constexpr int end = gate + ring_kept_bytes(B, VEC, V, T, B);
};

template <typename S> cudaError_t ring_forward(const kanb200_block_args& a, const RingPlan& p, cudaStream_t st);
template <typename S>
cudaError_t ring_backward(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st);

}  // namespace kanb200

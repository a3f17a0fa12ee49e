// How a call of kan_block.cu is spread over the GPU: host decisions, read by the kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kan_block.h"

namespace kanb200 {

constexpr int kSms = 148;
// Dynamic shared memory of a ring kernel's block: 228 KB of an SM less 1 KB per block and the kernel's own 768 bytes.
constexpr int kSharedBytes = 227 * 1024 - 768;

// Sums over rows that the backward returns, one slab each.
enum { kSumScale, kSumPostWeight, kSumPostBias, kSumNextWeight, kSumNextBias, kColumnSums };

struct BackwardSlabs {
    void* column[kColumnSums];       // [slab rows, width] each; NULL = not needed
    void* gate;                      // [teams + gate rows, width]: dgate of the part of a gate row's span that team t takes, at
                                     // row t + (gate row); NULL = no shared gate, or dgate not needed
};

// Teams take at most rows_per_team rows each: with a shared gate consecutive ones, otherwise every teams-th.
struct RowSplit {
    bool shared;                     // gate_rows rows share a gate row
    uint32_t rows_per_team;
    int64_t teams;                   // with a shared gate: those that have rows
};

enum { kFull, kVector, kScalar };    // how a thread reaches its columns, see Columns

struct RingPlan : RowSplit {
    int lanes;                       // 4, 8, 16 or 32
    int warps;                       // of a team, in one block (lanes == 32)
    int teams_per_block, cluster;
    int threads, blocks, stages, stage_bytes, parameter_bytes;
    bool many;                       // chunks
    int mode;                        // kFull, kVector or kScalar
    bool big;
};

// Chunks of four columns per thread.  More share the cost of a row among more elements, fewer leave registers.
//   * The forward behind a branch holds its parameters in registers with few chunks (rows that 8 warps cover that way) and
//     reads them from memory with many (wider rows; larger blocks with few chunks left SMs half empty: gated forward of
//     8176 x 2052, 190 us).
//   * The backward behind a branch holds the sums that are parameter gradients (20 V values): few chunks always (with many the
//     8-bit gated backward of 16384 x 2048 spilled and took 278 us instead of 243).
//   * A norm alone takes many.
constexpr int ring_chunks(bool many, bool f64) { return many && !f64 ? 4 : 2; }
// Threads of a block and blocks to an SM, which bound the registers: 512 threads to an SM may use 128 each.  (Float64: one
// block of 256, whose threads may use 255; wide rows take a cluster of those, as a larger block's ring and parameters would
// not fit an SM's shared memory.)
constexpr int ring_threads(bool big) { return big ? 512 : 256; }
constexpr int ring_blocks(bool big, bool f64) { return big || f64 ? 1 : 2; }

// Bytes of one tensor in a stage of the ring: elements of less than 4 bytes that cannot be copied four at a time are not
// there.  Values that may come as codes need room for either.
constexpr int ring_bytes(int element, bool vec, int chunks, int threads) {
    return vec || element >= 4 ? 4 * element * chunks * threads : 0;
}
constexpr int ring_scale_bytes(int chunks, int threads, int branch) { return chunks * threads / 4 * branch; }
constexpr int ring_stats_bytes(int threads, int branch) { return 2 * threads / 4 * branch; }        // a team has 4 lanes at least
constexpr int ring_kept_bytes(int element, bool vec, int chunks, int threads, int branch) {
    const int values = ring_bytes(element, vec, chunks, threads);
    const int codes = 4 * chunks * threads + ring_scale_bytes(chunks, threads, branch);
    return values > codes ? values : codes;
}
// A stage of the backward; what is not part of every call comes last.
template <bool NEXT, bool BRANCH, int V, int T, bool VEC, int S, int B> struct BackwardStage {
    static constexpr int dh = 0;
    static constexpr int x = dh + (NEXT ? ring_bytes(B, VEC, V, T) : 0);
    static constexpr int next_stats = x + (NEXT ? ring_kept_bytes(S, VEC, V, T, B) : 0);
    static constexpr int y = next_stats + (NEXT ? ring_stats_bytes(T, B) : 0);
    static constexpr int post_stats = y + (BRANCH ? ring_kept_bytes(B, VEC, V, T, B) : 0);
    static constexpr int dout = post_stats + (BRANCH ? ring_stats_bytes(T, B) : 0);
    static constexpr int gate = dout + ring_bytes(S, VEC, V, T);
    static constexpr int end = gate + ring_kept_bytes(B, VEC, V, T, B);
};

// Lets a kernel have all of a block's shared memory on the current device; remembers the kernels that may.
cudaError_t allow_shared_memory(const void* kernel);

template <typename S> cudaError_t ring_forward(const kanb200_block_args& a, const RingPlan& p, cudaStream_t st);
template <typename S>
cudaError_t ring_backward(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st);

}  // namespace kanb200

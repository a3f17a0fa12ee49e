// The norm and the gated residual connection, rows in registers: every thread owns V chunks of four columns for the whole
// launch, and its share of the next rows is already on its way into shared memory.
//
//   * A team of threads owns a row at a time: 4, 8 or 16 lanes, W warps, or the warps of a cluster of up to 8 blocks.
//     Teams take rows in turn; with a shared gate a team takes consecutive rows, so that a gate row is read, and its
//     gradient leaves, once per team (consecutive rows everywhere cost 5 to 10 % of the bandwidth: norm of 65536 x 1024
//     forward 99 us against 91).
//   * Memory -> registers goes through a ring of 2 to 4 rows in shared memory, filled by cp.async.  A thread copies
//     exactly what it reads back itself, so the ring needs no barrier: only its own cp.async group to have landed.  The
//     bytes in flight then do not depend on registers or on how many warps wait in a barrier.  (Statistics and scales in the
//     backward are one lane's copies for its team's lanes: a __syncwarp on either side of them.)
//   * Parameters stay on chip: in registers in the forward, in shared memory in the backward, where the registers hold the
//     sums over rows that are their gradients (one slab row per block leaves the kernel at its end).  Read from L1 for every
//     row they came from L2 whenever the ring took most of the SM's memory, a few hundred cycles at a time (gated forward of
//     16777 x 1000: 85 us, most of the stalls).
//   * Sums over a row: lanes by shuffles, warps through shared memory with a barrier of the team alone, blocks of a
//     cluster through each other's shared memory; every thread gets the same bits.
//   * Four warps per scheduler is what the registers of sums and parameters allow, so besides bandwidth the number of
//     instructions and their latencies count: what a row costs besides its elements (sums, barriers, addresses) is shared by
//     4 V elements; distances between a thread's elements are constants; float arithmetic works on pairs (one instruction for
//     two elements).
//
// What bounds them, by counters: the norm alone memory (DRAM 74 to 80 % of nominal, a copy reaches
// 85 %; issue slots 26 to 33 %); the float32 connection memory and latencies together (71 %, issue slots 52 to 54 %); with 8-bit
// codes instructions and latencies (issue slots 62 to 64 %, DRAM 37 to 65 %); rows whose width is not a multiple of four their
// element-wise copies and loads (DRAM 21 to 36 %).
//
// Measured, float32: norm of 65536 x 1024 forward 89 us (6.0 TB/s), backward 137 us (5.9 TB/s); connection of 16384 x 1024
// with a gate per row and both norms forward 54 us (6.2 TB/s), backward 93 us (5.8 TB/s); a copy runs at 6.55 TB/s.
#pragma once
#include <cooperative_groups.h>

#include "kan_block.cuh"
#include "kan_block_plan.h"

namespace kanb200 {

template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
// all but the newest stages - 1 groups have landed
__device__ __forceinline__ void copies_wait_oldest(int stages) {
    if (stages == 2) copies_wait<1>();
    else if (stages == 3) copies_wait<2>();
    else copies_wait<3>();
}

// Which columns a thread owns.  A warp covers V chunks of 4 LANES columns, one after the other.  A thread has four of each:
// runs of SIDE columns, 16 bytes of the branch's type (kFull, kVector: rows, strides and pointers allow four elements at
// once; float64: two runs, so that the lanes' accesses stay side by side) or single ones (kScalar: connection of
// 16384 x 1024 that way forward 70 us instead of 54, backward 130 instead of 93).  kFull: the team's columns are exactly the
// row's, so nothing is masked (against kVector: forward of 4096 x 4096 60 us instead of 77, 8-bit half-precision pass of
// 16384 x 2048 211 instead of 222; no difference at 16384 x 1024).  Distances between a thread's elements are constants, so a
// row costs one address per tensor.
template <int LANES_, int V_, int MODE_, int SIDE_> struct Columns {
    static constexpr int LANES = LANES_, V = V_, MODE = MODE_, SIDE = SIDE_;
    int col, width;
    static __device__ __forceinline__ constexpr int apart(int j, int e) {
        return j * 4 * LANES + e / SIDE * SIDE * LANES + e % SIDE;
    }
    __device__ __forceinline__ int at(int j, int e) const { return col + apart(j, e); }
    __device__ __forceinline__ bool ok(int j, int e) const { return MODE == kFull || at(j, e / SIDE * SIDE) < width; }
};

// BYTES consecutive bytes as one access
template <int BYTES> __device__ __forceinline__ void move(void* dst, const void* src) {
    using T = std::conditional_t<BYTES == 16, float4, std::conditional_t<BYTES == 8, float2, std::conditional_t<
                  BYTES == 4, uint32_t, std::conditional_t<BYTES == 2, uint16_t, uint8_t>>>>;
    *static_cast<T*>(dst) = *static_cast<const T*>(src);
}

// ---- rows <-> registers -----------------------------------------------------------------------------------------------
// A thread's elements of one tensor on their way from a row in memory to registers, run by run.  Runs of less than 4 bytes
// have no ring slot: they are loaded where they are used.  T is the block's most threads: a slot's runs are arrays over T
// threads, so that all distances in a stage are constants too.  Places of columns beyond the row hold 0 (clear_ring) and are
// never written.  `row` points to the thread's own first element.
template <typename E, typename C, int T> struct Feed {
    static constexpr int kRun = C::SIDE * (int)sizeof(E), kRuns = 4 / C::SIDE;
    static constexpr bool kRing = kRun >= 4;

    static __device__ __forceinline__ void issue(uint32_t stage, const E* row, const C& c) {
        if constexpr (kRing) {
            const uint32_t dst = stage + threadIdx.x * kRun;
#pragma unroll
            for (int j = 0; j < C::V; ++j)
#pragma unroll
                for (int r = 0; r < kRuns; ++r)
                    if (c.ok(j, r * C::SIDE)) copy_async<kRun>(dst + (j * kRuns + r) * T * kRun, row + C::apart(j, r * C::SIDE));
        }
    }
    static __device__ __forceinline__ Quad<E> take(const char* stage, const E* row, const C& c, int j) {
        const char* src = stage + threadIdx.x * kRun;
        Quad<E> q;
#pragma unroll
        for (int r = 0; r < kRuns; ++r) {
            E* to = q.v + r * C::SIDE;
            if constexpr (kRing) {
                move<kRun>(to, src + (j * kRuns + r) * T * kRun);
            } else {
#pragma unroll
                for (int e = 0; e < C::SIDE; ++e) to[e] = E{};
                if (c.ok(j, r * C::SIDE)) move<kRun>(to, row + C::apart(j, r * C::SIDE));
            }
        }
        return q;
    }
};

// `row`: the thread's own first element, here and below
template <typename T, typename C> __device__ __forceinline__ void put(T* row, const C& c, int j, const Quad<T>& q) {
#pragma unroll
    for (int r = 0; r < 4; r += C::SIDE)
        if (c.ok(j, r)) move<C::SIDE * (int)sizeof(T)>(row + C::apart(j, r), q.v + r);
}
template <typename B, typename C> __device__ __forceinline__ void put(B* row, const C& c, int j, const Four<B>& x) {
    put(row, c, j, Quad<B>{{x.v[0], x.v[1], x.v[2], x.v[3]}});
}
// Four values of a parameter (or a shared gate row); 0 beyond the row.
template <typename B, typename C> __device__ __forceinline__ Four<B> get(const B* row, const C& c, int j) {
    Quad<B> q{};
#pragma unroll
    for (int r = 0; r < 4; r += C::SIDE)
        if (c.ok(j, r)) move<C::SIDE * (int)sizeof(B)>(q.v + r, row + C::apart(j, r));
    return widen4<B>(q);
}
// ... or `absent` where there is no such parameter, 0 beyond the row as well: what a mean-subtracting norm's backward leaves
// in the columns beyond the row (its mean) has to stay out of the sums behind it.
template <typename B, typename C> __device__ __forceinline__ Four<B> get_or(const void* p, const C& c, int j, B absent) {
    Four<B> ones = four<B>(absent);
    if constexpr (C::MODE != kFull) {
        Quad<B> q;
#pragma unroll
        for (int r = 0; r < 4; ++r) q.v[r] = c.ok(j, r / C::SIDE * C::SIDE) ? absent : B(0);
        ones = widen4<B>(q);
    }
    return p ? get(static_cast<const B*>(p) + c.col, c, j) : ones;
}
// x - mean for the row's own columns; 0 beyond them, where x is 0
template <typename B, typename C> __device__ __forceinline__ Four<B> centre(const C& c, int j, const Four<B>& x, B mean) {
    Four<B> m = four<B>(-mean);
    if constexpr (C::MODE != kFull)
#pragma unroll
        for (int r = 0; r < 4; r += C::SIDE) {
            const B own = c.ok(j, r) ? -mean : B(0);
#pragma unroll
            for (int e = 0; e < C::SIDE; ++e) m.v[r + e] = own;
        }
    return x + m;
}
// A parameter's values in shared memory: 16-byte pieces, arrays over the threads of a team.  `at`: the thread's first piece.
template <typename B> __device__ __forceinline__ void to_shelf(char* at, int threads, int j, const Four<B>& x) {
    constexpr int kPieces = 4 * sizeof(B) / 16;
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
        move<16>(at + (j * kPieces + p) * threads * 16, reinterpret_cast<const char*>(x.v) + 16 * p);
}
template <typename B> __device__ __forceinline__ Four<B> from_shelf(const char* at, int threads, int j) {
    constexpr int kPieces = 4 * sizeof(B) / 16;
    Quad<B> q;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) move<16>(reinterpret_cast<char*>(q.v) + 16 * p, at + (j * kPieces + p) * threads * 16);
    return widen4<B>(q);
}
__device__ __forceinline__ void clear_ring(char* ring, int bytes) {
    for (int at = threadIdx.x * 16; at < bytes; at += blockDim.x * 16)
        *reinterpret_cast<float4*>(ring + at) = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
}

// 1 / sqrt: the float approximation (2 ulp) and a Newton step, instead of a correctly rounded root and division.  0 for
// infinity (squares that overflow), where the step would give NaN.
__device__ __forceinline__ float rsqrt_newton(float v) {
    const float r = rsqrtf(v);
    return r == 0.0f ? 0.0f : r * fmaf(-0.5f * v * r, r, 1.5f);
}
__device__ __forceinline__ double rsqrt_newton(double v) { return 1.0 / sqrt(v); }

// ---- the team and its sums ------------------------------------------------------------------------------------------
struct TeamScratch {                       // per block, in shared memory
    static constexpr int kMaxSums = 2, kMaxCluster = 8;
    double warp[2][16][kMaxSums];          // by warp of the block; float teams use half of it
    double block[2][kMaxSums][kMaxCluster];
};

static_assert(sizeof(TeamScratch) == 768, "kSharedBytes");

template <typename B, int LANES, bool CLUSTERED> struct Team {
    TeamScratch* scratch;
    int warps, team, warp, lane;           // warps of this block in a row's team; team and warp within the team
    int group;                             // of 128 columns, the warp's first
    int cluster, rank;
    int phase = 0;

    template <int K> __device__ __forceinline__ void sum(B (&v)[K]) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
        if (LANES < 32 || (warps == 1 && (!CLUSTERED || cluster == 1))) return;
        // alternating buffers: a warp can only be one sum ahead of the others, so one barrier per sum is enough
        phase ^= 1;
        B* mine = reinterpret_cast<B*>(scratch->warp[phase]) + team * warps * K;
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) mine[warp * K + k] = v[k];
        asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(warps * 32) : "memory");
        // a lane takes one warp's sums (the low bits of its number say whose), and the lanes add them up in pairs
        const int low = warps > 8 ? 15 : warps > 4 ? 7 : warps > 2 ? 3 : 1, whose = lane & low;
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = whose < warps ? mine[whose * K + k] : B(0);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
            if (o <= low)
#pragma unroll
                for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
        if (CLUSTERED && cluster > 1) {
            namespace cg = cooperative_groups;
            cg::cluster_group all = cg::this_cluster();
            if (warp == 0 && lane < cluster) {
                TeamScratch* there = all.map_shared_rank(scratch, lane);
#pragma unroll
                for (int k = 0; k < K; ++k) *reinterpret_cast<B*>(&there->block[phase][k][rank]) = v[k];
            }
            all.sync();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                B s = B(0);
                for (int r = 0; r < cluster; ++r) s += *reinterpret_cast<const B*>(&scratch->block[phase][k][r]);
                v[k] = s;
            }
        }
    }
};

// start of a row: rows and strides are below 2^31 here, so one wide multiplication
template <typename T> __device__ __forceinline__ T* row_at(T* base, uint32_t row, int64_t stride) {
    return base + (uint64_t)row * (uint32_t)stride;
}

// The team's place: its first column, and its first row.
template <typename B, typename C, bool CLUSTERED>
__device__ __forceinline__ uint32_t set_up(const RingPlan& p, int width, TeamScratch* scratch, Team<B, C::LANES, CLUSTERED>& team,
                                           C& c) {
    constexpr int LANES = C::LANES, V = C::V;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    team.scratch = scratch;
    team.cluster = CLUSTERED ? p.cluster : 1;
    team.rank = CLUSTERED && p.cluster > 1 ? (int)(blockIdx.x % p.cluster) : 0;
    const uint32_t group = CLUSTERED && p.cluster > 1 ? blockIdx.x / p.cluster : blockIdx.x;
    uint32_t id;
    if (LANES == 32) {
        team.warps = p.warps;
        team.team = p.teams_per_block == 1 ? 0 : warp / p.warps;
        team.warp = warp - team.team * p.warps;
        team.lane = lane;
        c.col = (team.rank * p.warps + team.warp) * V * kPackGroup + C::SIDE * lane;
        id = group * p.teams_per_block + team.team;
    } else {
        team.warps = 1;
        team.team = 0;
        team.warp = 0;
        team.lane = lane & (LANES - 1);
        c.col = C::SIDE * team.lane;
        id = group * p.teams_per_block + threadIdx.x / LANES;
    }
    c.width = width;
    team.group = (c.col - C::SIDE * team.lane) / kPackGroup;
    if (CLUSTERED && p.cluster > 1) cooperative_groups::this_cluster().sync();      // every block's scratch exists
    return id;
}

__device__ __forceinline__ uint32_t word_of(const Quad<uint8_t>& q) { return *reinterpret_cast<const uint32_t*>(q.v); }

// Codes of a thread's elements and the scales of their groups.  A group is a warp's chunk, or with fewer lanes 32 / LANES
// chunks of the same threads.  Each lane forms the scale and its reciprocal of one group only.
template <typename B, typename C>
__device__ __forceinline__ void put_codes(int format, const Four<B> (&v)[C::V], const C& c, bool write, uint8_t* codes,
                                          B* scales, int lane, int first) {
    constexpr int LANES = C::LANES, V = C::V;
    constexpr int kTogether = 32 / LANES < V ? 32 / LANES : V, kGroups = V / kTogether;
    using Bits = typename AbsBits<B>::type;
    Bits mine = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        B largest = B(0);                                   // columns beyond the row hold 0
#pragma unroll
        for (int j = i * kTogether; j < (i + 1) * kTogether; ++j) largest = max_abs(largest, v[j]);
        const Bits top = lanes_max<LANES>(AbsBits<B>::of(largest));
        if (kGroups == 1 || lane % kGroups == i) mine = top;
    }
    const B scale = pack_scale<B>(format, AbsBits<B>::back(mine)), inverse = pack_inverse<B>(scale);
    if (write && lane < kGroups && (first + lane) * kPackGroup < c.width) scales[first + lane] = scale;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const B inv = kGroups == 1 ? inverse : __shfl_sync(0xffffffffu, inverse, i, LANES);
        if (!write) continue;
#pragma unroll
        for (int j = i * kTogether; j < (i + 1) * kTogether; ++j) {
            const uint32_t word = encode4(format, v[j], inv);
            put(codes, c, j, Quad<uint8_t>{{(uint8_t)word, (uint8_t)(word >> 8), (uint8_t)(word >> 16), (uint8_t)(word >> 24)}});
        }
    }
}

// ---- forward ----------------------------------------------------------------------------------------------------------
template <typename S, int LANES, int V, int MODE, bool BRANCH, bool BIG>
__global__ void __launch_bounds__(ring_threads(BIG), ring_blocks(BIG, sizeof(S) == 8))
    ring_forward_kernel(const __grid_constant__ kanb200_block_args a, const __grid_constant__ RingPlan p) {
    using B = Br<S>;
    constexpr int T = ring_threads(BIG);
    using C = Columns<LANES, V, MODE, MODE == kScalar ? 1 : 16 / (int)sizeof(B)>;
    using FS = Feed<S, C, T>;
    using FB = Feed<B, C, T>;
    constexpr int at_y = ring_bytes((int)sizeof(S), MODE != kScalar, V, T),
                  at_gate = at_y + ring_bytes((int)sizeof(B), MODE != kScalar, V, T);
    extern __shared__ __align__(16) char ring[];
    __shared__ TeamScratch scratch;
    constexpr bool CLUSTERED = LANES == 32 && (BIG || sizeof(S) == 8);
    Team<B, LANES, CLUSTERED> team;
    C c;
    const uint32_t id = set_up(p, (int)a.width, &scratch, team, c);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring), rows = (uint32_t)a.rows;
    const bool row_gate = BRANCH && a.gate && !p.shared;
    const int D = (int)a.width, groups = (D + kPackGroup - 1) / kPackGroup;
    const B eps = B(a.eps), per = B(1) / B(D);

    const S* x = static_cast<const S*>(a.x) + c.col;
    const B *y = static_cast<const B*>(a.y) + c.col, *gate = static_cast<const B*>(a.gate) + c.col;
    // parameters in registers, or with many chunks behind a branch in memory
    constexpr bool kHeld = !BRANCH || V == 2;
    Four<B> held[5][kHeld ? V : 1];
#pragma unroll
    for (int j = 0; j < (kHeld ? V : 1); ++j) {
        held[0][j] = get_or(BRANCH ? a.scale : nullptr, c, j, B(1));
        held[1][j] = get_or(BRANCH ? a.post_weight : nullptr, c, j, B(1));
        held[2][j] = get_or(BRANCH ? a.post_bias : nullptr, c, j, B(0));
        held[3][j] = get_or(a.next_weight, c, j, B(1));
        held[4][j] = get_or(a.next_bias, c, j, B(0));
    }
    const auto parameter = [&](int which, const void* from, int j, B absent) {
        if constexpr (kHeld) return held[which][j];
        else return get_or(from, c, j, absent);
    };

    const uint32_t first = p.shared ? id * p.rows_per_team : id, next = p.shared ? 1u : (uint32_t)p.teams,
                   last = p.shared ? min(first + p.rows_per_team, rows) : rows;
    const auto issue = [&](uint32_t row, int stage) {
        if (row < last) {
            const uint32_t at = ring_at + stage * p.stage_bytes;
            FS::issue(at, row_at(x, row, a.x_stride), c);
            if (BRANCH) FB::issue(at + at_y, row_at(y, row, a.y_stride), c);
            if (row_gate) FB::issue(at + at_gate, row_at(gate, row, a.gate_stride), c);
        }
        copies_commit();
    };
    // the row's mean and 1 / deviation; two passes over registers, so that the variance has no cancellation
    const auto moments = [&](int kind, const Four<B> (&v)[V], B& mean, B& rstd) {
        mean = B(0);
        Four<B> acc = four<B>(B(0));
        B s[1];
        if (kind == kNormLayer) {
#pragma unroll
            for (int j = 0; j < V; ++j) acc = acc + v[j];           // columns beyond the row hold 0
            s[0] = total(acc);
            team.template sum<1>(s);
            mean = s[0] * per;
            acc = four<B>(B(0));
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const Four<B> d = centre<B>(c, j, v[j], mean);
                acc = fma4(d, d, acc);
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) acc = fma4(v[j], v[j], acc);
        }
        s[0] = total(acc);
        team.template sum<1>(s);
        rstd = rsqrt_newton(fma(s[0], per, eps));
    };
    const auto put_stats = [&](void* stats, uint32_t row, B mean, B rstd) {
        if (c.col == 0) {
            B* at = static_cast<B*>(stats) + 2 * (uint64_t)row;
            at[0] = mean;
            at[1] = rstd;
        }
    };

    uint32_t span_end = first, span = 0;                    // of a shared gate: where its next row starts
    if (p.shared) {
        span = first / (uint32_t)a.gate_rows;
        span_end = first;
    }
    if (MODE != kFull) clear_ring(ring, p.stages * p.stage_bytes);
    uint32_t ahead = first;
    for (int s = 0; s + 1 < p.stages; ++s, ahead += next) issue(ahead, s);
    int stage = 0;
    Four<B> t[V];                                           // act(gate) of a shared gate
    // every team makes the same number of steps: teams that share a warp meet in its shuffles
    for (uint32_t step = 0, row = first; step < p.rows_per_team; ++step, row += next, ahead += next) {
        issue(ahead, stage == 0 ? p.stages - 1 : stage - 1);
        copies_wait_oldest(p.stages);
        const bool live = row < last;
        if (LANES == 32 && !live) break;                    // a whole team, alone in its warps
        const char* at = ring + stage * p.stage_bytes;
        const uint64_t dense = (uint64_t)row * (uint32_t)D + (uint32_t)c.col;      // of dense tensors
        Four<B> o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = four<B>(B(0));
        if (BRANCH) {
            Four<B> v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = live ? widen4<B>(FB::take(at + at_y, row_at(y, row, a.y_stride), c, j)) : four<B>(B(0));
            if (a.y_codes)
                put_codes<B>(a.checkpoint, v, c, live, static_cast<uint8_t*>(a.y_codes) + dense,
                             row_at(static_cast<B*>(a.y_scales), row, groups), team.lane, team.group);
            if (a.post_norm != kNormNone) {
                B mean, rstd;
                moments(a.post_norm, v, mean, rstd);
                if (a.post_stats && live) put_stats(a.post_stats, row, mean, rstd);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = centre<B>(c, j, v[j], mean) * four<B>(rstd);
            }
            if (p.shared && row >= span_end && live) {
                span = row / (uint32_t)a.gate_rows;
                span_end = (span + 1) * (uint32_t)a.gate_rows;
#pragma unroll
                for (int j = 0; j < V; ++j) t[j] = gate4<B>(a.gate_act, get(row_at(gate, span, a.gate_stride), c, j));
            }
            // out = x + scale act(gate) z; what v becomes is the branch's summand
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[j] = fma4(v[j], parameter(1, a.post_weight, j, B(1)), parameter(2, a.post_bias, j, B(0))) *
                       parameter(0, a.scale, j, B(1));
                if (p.shared) v[j] = v[j] * t[j];
            }
            if (row_gate) {
                Four<B> g[V];
#pragma unroll
                for (int j = 0; j < V; ++j)
                    g[j] = live ? widen4<B>(FB::take(at + at_gate, row_at(gate, row, a.gate_stride), c, j)) : four<B>(B(0));
                if (a.gate_codes)
                    put_codes<B>(a.checkpoint, g, c, live, static_cast<uint8_t*>(a.gate_codes) + dense,
                                 row_at(static_cast<B*>(a.gate_scales), row, groups), team.lane, team.group);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = v[j] * gate4<B>(a.gate_act, g[j]);
            }
            if (live)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const Quad<S> q = narrow4<S>(widen4<S>(FS::take(at, row_at(x, row, a.x_stride), c, j)) + v[j]);
                    o[j] = widen4<S>(q);                              // 0 beyond the row, as all its terms are
                    put(static_cast<S*>(a.out) + dense, c, j, q);
                }
        } else if (live) {
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = widen4<S>(FS::take(at, row_at(x, row, a.x_stride), c, j));
        }
        if (a.x_codes)
            put_codes<B>(a.checkpoint, o, c, live, static_cast<uint8_t*>(a.x_codes) + dense,
                         row_at(static_cast<B*>(a.x_scales), row, groups), team.lane, team.group);
        if (!BRANCH || a.next_norm != kNormNone) {
            B mean, rstd;
            moments(a.next_norm, o, mean, rstd);
            if (a.next_stats && live) put_stats(a.next_stats, row, mean, rstd);
            if (live)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    o[j] = fma4(centre<B>(c, j, o[j], mean) * four<B>(rstd), parameter(3, a.next_weight, j, B(1)),
                                parameter(4, a.next_bias, j, B(0)));
                    put(static_cast<B*>(a.h) + dense, c, j, o[j]);
                }
        }
        stage = stage + 1 == p.stages ? 0 : stage + 1;
    }
    copies_wait<0>();
}

// ---- backward -----------------------------------------------------------------------------------------------------------
template <typename S, int LANES, int V, int MODE, bool BRANCH, bool NEXT, bool BIG>
__global__ void __launch_bounds__(ring_threads(BIG), ring_blocks(BIG, sizeof(S) == 8))
    ring_backward_kernel(const __grid_constant__ kanb200_block_args a, const __grid_constant__ RingPlan p,
                         const __grid_constant__ BackwardSlabs slabs) {
    using B = Br<S>;
    constexpr int T = ring_threads(BIG);
    using C = Columns<LANES, V, MODE, MODE == kScalar ? 1 : 16 / (int)sizeof(B)>;
    using FS = Feed<S, C, T>;
    using FB = Feed<B, C, T>;
    using FQ = Feed<uint8_t, C, T>;
    using At = BackwardStage<NEXT, BRANCH, V, T, MODE != kScalar, (int)sizeof(S), (int)sizeof(B)>;
    extern __shared__ __align__(16) char ring[];
    __shared__ TeamScratch scratch;
    constexpr bool CLUSTERED = LANES == 32 && (BIG || sizeof(S) == 8);
    Team<B, LANES, CLUSTERED> team;
    C c;
    const uint32_t id = set_up(p, (int)a.width, &scratch, team, c);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring), rows = (uint32_t)a.rows;
    const int D = (int)a.width, groups = (D + kPackGroup - 1) / kPackGroup;
    const bool row_gate = BRANCH && (a.gate || a.gate_codes) && !p.shared;
    const B per = B(1) / B(D);
    const Four<B> zero = four<B>(B(0));

    const S *x = static_cast<const S*>(a.x) + c.col, *dout = static_cast<const S*>(a.dout) + c.col;
    const B *y = static_cast<const B*>(a.y) + c.col, *gate = static_cast<const B*>(a.gate) + c.col,
            *dh = static_cast<const B*>(a.dh) + c.col, *pb = static_cast<const B*>(a.post_bias) + c.col;
    // parameters: teams of a block share them
    const int per_team = blockDim.x / p.teams_per_block, in_team = threadIdx.x % per_team;
    const int array = per_team * 4 * V * (int)sizeof(B);
    char *const nw = ring + p.stages * p.stage_bytes + in_team * 16, *const pw = nw + (NEXT ? array : 0), *const scale = pw + array;
    if ((int)threadIdx.x < per_team)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (NEXT) to_shelf(nw, per_team, j, get_or(a.next_weight, c, j, B(1)));
            if (BRANCH) to_shelf(pw, per_team, j, get_or(a.post_weight, c, j, B(1)));
            if (BRANCH) to_shelf(scale, per_team, j, get_or(a.scale, c, j, B(1)));
        }
    __syncthreads();
    // sums over rows: of g a yhat and of g a behind a branch (its three parameters' gradients are multiples of those, see the
    // end), of dh xhat and dh at a norm, of dgate
    Four<B> sum_gay[V], sum_ga[V], sum_nw[V], sum_nb[V], sum_gate[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum_gay[j] = sum_ga[j] = sum_nw[j] = sum_nb[j] = sum_gate[j] = zero;

    // What a warp's lanes read in common (statistics, scales) one lane copies: a copy of one address by 32 lanes to 32 places
    // takes 32 passes of the shared memory.  The lanes meet in a __syncwarp before they read it.
    constexpr int kTogether = 32 / LANES < V ? 32 / LANES : V, kGroups = V / kTogether;
    const int clique = threadIdx.x / LANES;
    // a tensor that may be there as codes: codes and their groups' scales, or the values themselves
    const auto issue_kept = [&](uint32_t at, const void* codes, const void* scales, auto* values, int64_t stride, uint32_t row) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(values)>>;
        if (codes) {
            FQ::issue(at, static_cast<const uint8_t*>(codes) + (uint64_t)row * (uint32_t)D + (uint32_t)c.col, c);
            if (team.lane < kGroups && team.group + team.lane < groups)
                copy_async<sizeof(B)>(at + 4 * V * T + (clique * V + team.lane) * (uint32_t)sizeof(B),
                                      static_cast<const B*>(scales) + (uint64_t)row * (uint32_t)groups + team.group + team.lane);
        } else {
            Feed<E, C, T>::issue(at, row_at(values, row, stride), c);
        }
    };
    const auto take_kept = [&](const char* at, const void* codes, auto* values, int64_t stride, uint32_t row, int j) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(values)>>;
        if (codes) {
            const Quad<uint8_t> q = FQ::take(at, static_cast<const uint8_t*>(codes) + (uint64_t)row * (uint32_t)D + (uint32_t)c.col, c, j);
            const B s = reinterpret_cast<const B*>(at + 4 * V * T)[clique * V + j / kTogether];
            return decode4<B>(a.checkpoint, word_of(q), s);
        }
        return widen4<E>(Feed<E, C, T>::take(at, row_at(values, row, stride), c, j));
    };
    const auto issue_stats = [&](uint32_t at, const void* stats, uint32_t row) {
        if (team.lane == 0)
            copy_async<2 * sizeof(B)>(at + clique * 2 * (uint32_t)sizeof(B), static_cast<const B*>(stats) + 2 * (uint64_t)row);
    };
    const uint32_t first = p.shared ? id * p.rows_per_team : id, next = p.shared ? 1u : (uint32_t)p.teams,
                   last = p.shared ? min(first + p.rows_per_team, rows) : rows;
    const auto issue = [&](uint32_t row, int stage) {
        if (row < last) {
            const uint32_t at = ring_at + stage * p.stage_bytes;
            if (a.dout) FS::issue(at + At::dout, row_at(dout, row, a.dout_stride), c);
            if (NEXT) {
                FB::issue(at + At::dh, row_at(dh, row, a.dh_stride), c);
                issue_kept(at + At::x, a.x_codes, a.x_scales, x, a.x_stride, row);
                issue_stats(at + At::next_stats, a.next_stats, row);
            }
            if (BRANCH) {
                issue_kept(at + At::y, a.y_codes, a.y_scales, y, a.y_stride, row);
                if (row_gate) issue_kept(at + At::gate, a.gate_codes, a.gate_scales, gate, a.gate_stride, row);
                if (a.post_norm != kNormNone) issue_stats(at + At::post_stats, a.post_stats, row);
            }
        }
        copies_commit();
    };

    uint32_t span = 0, span_first = first, span_end = first;             // of a shared gate: the rows under its row
    if (p.shared) {
        span = first / (uint32_t)a.gate_rows;
        span_first = span * (uint32_t)a.gate_rows;
        span_end = span_first + (uint32_t)a.gate_rows;
    }
    if (MODE != kFull) clear_ring(ring, p.stages * p.stage_bytes);
    uint32_t ahead = first;
    for (int s = 0; s + 1 < p.stages; ++s, ahead += next) issue(ahead, s);
    int stage = 0;
    for (uint32_t step = 0, row = first; step < p.rows_per_team; ++step, row += next, ahead += next) {
        // The slot that is filled now is the one the step before has read, statistics and scales by all lanes but copied by one:
        // that lane waits for the others (a sum over the row may be the last thing that kept them together, or there was none).
        __syncwarp();
        issue(ahead, stage == 0 ? p.stages - 1 : stage - 1);
        copies_wait_oldest(p.stages);
        __syncwarp();                                       // ... and the others for its copies
        const bool live = row < last;
        if (LANES == 32 && !live) break;
        const char* at = ring + stage * p.stage_bytes;
        const uint64_t dense = (uint64_t)row * (uint32_t)D + (uint32_t)c.col;      // of dense tensors
        Four<B> g[V];                                       // gradient of the norm's input, then of y
#pragma unroll
        for (int j = 0; j < V; ++j)
            g[j] = a.dout && live ? widen4<S>(FS::take(at + At::dout, row_at(dout, row, a.dout_stride), c, j)) : zero;
        if (NEXT) {
            Four<B> v[V], d[V], s0 = zero, s1 = zero;
            B rstd = B(0);
            if (live) {
                const B* stats = reinterpret_cast<const B*>(at + At::next_stats) + 2 * clique;
                const B mean = stats[0];
                rstd = stats[1];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    d[j] = widen4<B>(FB::take(at + At::dh, row_at(dh, row, a.dh_stride), c, j));
                    v[j] = take_kept(at + At::x, a.x_codes, x, a.x_stride, row, j);
                    v[j] = centre<B>(c, j, v[j], mean) * four<B>(rstd);          // the normalised row
                    sum_nw[j] = fma4(d[j], v[j], sum_nw[j]);
                    sum_nb[j] = sum_nb[j] + d[j];
                    d[j] = d[j] * from_shelf<B>(nw, per_team, j);
                    s0 = s0 + d[j];
                    s1 = fma4(d[j], v[j], s1);
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = d[j] = zero;
            }
            B s[2] = {total(s0), total(s1)};
            team.template sum<2>(s);
            const Four<B> flat = four<B>(a.next_norm == kNormLayer ? -s[0] * per : B(0)), along = four<B>(-s[1] * per);
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = fma4(four<B>(rstd), fma4(v[j], along, d[j] + flat), g[j]);
        }
        if (a.dx && live)
#pragma unroll
            for (int j = 0; j < V; ++j) put(static_cast<S*>(a.dx) + dense, c, j, narrow4<S>(g[j]));
        if (BRANCH) {
            Four<B> v[V], s0 = zero, s1 = zero;
            B rstd = B(1);
            if (live) {
                B mean = B(0);
                if (a.post_norm != kNormNone) {
                    const B* stats = reinterpret_cast<const B*>(at + At::post_stats) + 2 * clique;
                    mean = stats[0];
                    rstd = stats[1];
                }
                if (p.shared && row == span_end) {
                    ++span;
                    span_first = span_end;
                    span_end += (uint32_t)a.gate_rows;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[j] = take_kept(at + At::y, a.y_codes, y, a.y_stride, row, j);
                    if (a.post_norm != kNormNone) v[j] = centre<B>(c, j, v[j], mean) * four<B>(rstd);
                    const Four<B> w = from_shelf<B>(pw, per_team, j), sc = from_shelf<B>(scale, per_team, j);
                    Four<B> z = v[j] * w;
                    if (a.post_bias) z = z + get(pb, c, j);
                    if (p.shared || row_gate) {
                        Four<B> act, dact;
                        const Four<B> gv = p.shared ? get(row_at(gate, span, a.gate_stride), c, j)
                                                    : take_kept(at + At::gate, a.gate_codes, gate, a.gate_stride, row, j);
                        gate4_grad<B>(a.gate_act, gv, act, dact);
                        const Four<B> dg = g[j] * z * (dact * sc);
                        if (p.shared) sum_gate[j] = sum_gate[j] + dg;
                        else if (a.dgate) put(row_at(static_cast<B*>(a.dgate) + c.col, row, a.dgate_stride), c, j, dg);
                        g[j] = g[j] * act;
                    }
                    sum_gay[j] = fma4(g[j], v[j], sum_gay[j]);
                    sum_ga[j] = sum_ga[j] + g[j];
                    g[j] = g[j] * (sc * w);
                    s0 = s0 + g[j];
                    s1 = fma4(g[j], v[j], s1);
                }
            }
            if (a.dy) {
                if (a.post_norm != kNormNone) {
                    B s[2] = {total(s0), total(s1)};
                    team.template sum<2>(s);
                    const Four<B> flat = four<B>(a.post_norm == kNormLayer ? -s[0] * per : B(0)), along = four<B>(-s[1] * per);
                    if (live)
#pragma unroll
                        for (int j = 0; j < V; ++j) g[j] = four<B>(rstd) * fma4(v[j], along, g[j] + flat);
                }
                if (live)
#pragma unroll
                    for (int j = 0; j < V; ++j) put(row_at(static_cast<B*>(a.dy) + c.col, row, a.dy_stride), c, j, g[j]);
            }
            if (slabs.gate && live && (row + 1 == span_end || row + 1 == last)) {
                // a gate row whose rows are all this team's is finished here, otherwise its share goes to a slab
                B* to = first <= span_first && row + 1 == span_end
                            ? row_at(static_cast<B*>(a.dgate) + c.col, span, a.dgate_stride)
                            : static_cast<B*>(slabs.gate) + (uint64_t)(id + span) * (uint32_t)D + c.col;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    put(to, c, j, sum_gate[j]);
                    sum_gate[j] = zero;
                }
            }
        }
        stage = stage + 1 == p.stages ? 0 : stage + 1;
    }
    copies_wait<0>();

    // one slab row per block: the teams' sums, added in the order of the teams
    const uint32_t block = CLUSTERED && p.cluster > 1 ? blockIdx.x / p.cluster : blockIdx.x;
    Four<B>* shelf = reinterpret_cast<Four<B>*>(ring);
    const auto leave = [&](int which, Four<B> (&v)[V]) {
        if (!slabs.column[which]) return;
        B* row = static_cast<B*>(slabs.column[which]) + (uint64_t)block * (uint32_t)D + c.col;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (p.teams_per_block > 1) {
                __syncthreads();
                shelf[threadIdx.x] = v[j];
                __syncthreads();
                if ((int)threadIdx.x >= per_team) continue;
                for (int i = 1; i < p.teams_per_block; ++i) v[j] = v[j] + shelf[i * per_team + threadIdx.x];
            }
            put(row, c, j, v[j]);
        }
    };
    if (BRANCH) {
        // z = yhat w + b:  dscale = sum g a z = w sum g a yhat + b sum g a,  dw = scale sum g a yhat,  db = scale sum g a
        Four<B> share[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
            share[j] = fma4(sum_gay[j], get_or(a.post_weight, c, j, B(1)), sum_ga[j] * get_or(a.post_bias, c, j, B(0)));
        leave(kSumScale, share);
#pragma unroll
        for (int j = 0; j < V; ++j) share[j] = sum_gay[j] * get_or(a.scale, c, j, B(1));
        leave(kSumPostWeight, share);
#pragma unroll
        for (int j = 0; j < V; ++j) share[j] = sum_ga[j] * get_or(a.scale, c, j, B(1));
        leave(kSumPostBias, share);
    }
    if (NEXT) {
        leave(kSumNextWeight, sum_nw);
        leave(kSumNextBias, sum_nb);
    }
}

}  // namespace kanb200

// ---- launches: included by one source per stream type ---------------------------------------------------------------
namespace kanb200 {

template <typename... P>
cudaError_t ring_launch(const RingPlan& p, cudaStream_t st, void (*kernel)(P...), const P&... args) {
    const int bytes = p.stages * p.stage_bytes + p.parameter_bytes;
    if (bytes > 48 * 1024 - (int)sizeof(TeamScratch)) {
        const cudaError_t e = allow_shared_memory(reinterpret_cast<const void*>(kernel));
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)p.blocks);
    cfg.blockDim = dim3((unsigned)p.threads);
    cfg.dynamicSmemBytes = (size_t)bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    if (p.cluster > 1) {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)p.cluster;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename S, int LANES, int MODE, bool BIG>
cudaError_t ring_forward_as(const kanb200_block_args& a, const RingPlan& p, cudaStream_t st) {
    constexpr bool f64 = sizeof(S) == 8;
    constexpr int few = ring_chunks(false, f64), many = ring_chunks(true, f64);
    if (!a.y) return ring_launch(p, st, ring_forward_kernel<S, LANES, many, MODE, false, BIG>, a, p);
    if constexpr (LANES == 32)
        if (BIG || p.many) return ring_launch(p, st, ring_forward_kernel<S, LANES, many, MODE, true, BIG>, a, p);
    if constexpr (BIG) return cudaErrorInvalidValue;         // not reached
    else return ring_launch(p, st, ring_forward_kernel<S, LANES, few, MODE, true, false>, a, p);
}
template <typename S, int LANES, int MODE, bool BIG>
cudaError_t ring_backward_as(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st) {
    constexpr bool f64 = sizeof(S) == 8;
    if (!a.has_branch)
        return ring_launch(p, st, ring_backward_kernel<S, LANES, ring_chunks(true, f64), MODE, false, true, BIG>,
                           a, p, slabs);
    return a.dh ? ring_launch(p, st, ring_backward_kernel<S, LANES, ring_chunks(false, f64), MODE, true, true, BIG>,
                              a, p, slabs)
                : ring_launch(p, st, ring_backward_kernel<S, LANES, ring_chunks(false, f64), MODE, true, false, BIG>,
                              a, p, slabs);
}

// name<S, LANES, MODE, BIG>(...) for the plan's lanes and mode
#define KANB200_RING_MODE(name, lanes, big, ...)                                              \
    switch (p.mode) {                                                                         \
        case kFull: return name<S, lanes, kFull, big>(__VA_ARGS__);                           \
        case kVector: return name<S, lanes, kVector, big>(__VA_ARGS__);                       \
        default: return name<S, lanes, kScalar, big>(__VA_ARGS__);                            \
    }
#define KANB200_RING_DISPATCH(name, ...)                                                      \
    if constexpr (sizeof(S) < 8) {                                                            \
        if (p.big) KANB200_RING_MODE(name, 32, true, __VA_ARGS__)                             \
    }                                                                                         \
    switch (p.lanes) {                                                                        \
        case 32: KANB200_RING_MODE(name, 32, false, __VA_ARGS__)                              \
        case 16: KANB200_RING_MODE(name, 16, false, __VA_ARGS__)                              \
        case 8: KANB200_RING_MODE(name, 8, false, __VA_ARGS__)                                \
        default: KANB200_RING_MODE(name, 4, false, __VA_ARGS__)                               \
    }

template <typename S> cudaError_t ring_forward(const kanb200_block_args& a, const RingPlan& p, cudaStream_t st) {
    KANB200_RING_DISPATCH(ring_forward_as, a, p, st)
}
template <typename S>
cudaError_t ring_backward(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st) {
    KANB200_RING_DISPATCH(ring_backward_as, a, p, slabs, st)
}
#undef KANB200_RING_DISPATCH
#undef KANB200_RING_MODE

}  // namespace kanb200

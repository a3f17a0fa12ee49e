// The norm and the gated residual connection, rows in registers: every thread owns V chunks of four columns for the whole
// launch, and its share of the next rows is already on its way into shared memory.
//
//   * A team of threads owns a row at a time: 4, 8 or 16 lanes, W warps, or the warps of a cluster of up to 8 blocks.
//     Teams take rows (or, with a shared gate, runs of rows under one gate row) in turn.
//   * Memory -> registers goes through a ring of 2 to 8 rows in shared memory, filled by cp.async.  A thread copies
//     exactly what it reads back itself, so the ring needs no barrier: only its own cp.async group to have landed.  The
//     bytes in flight then do not depend on registers or on how many warps wait in a barrier.
//   * The sums over rows that are the parameters' gradients stay in registers; one slab row per block leaves the kernel at
//     its end.  Parameters are read again for every row, from L1.
//   * Sums over a row: lanes by shuffles, warps through shared memory with a barrier of the team alone, blocks of a
//     cluster through each other's shared memory; every thread gets the same bits.
//   * V: what a row costs besides its elements -- its sums, barriers, waits, addresses, about 100 instructions -- is
//     shared by 4 V elements.  With V = 1 the kernels were bound by issue slots (norm of 65536 x 1024: 232 instructions
//     per warp and row forward, 345 backward, 76 % of the issue slots taken at 58 % of the copy bandwidth).
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
    switch (stages) {
        case 2: copies_wait<1>(); break;
        case 3: copies_wait<2>(); break;
        case 4: copies_wait<3>(); break;
        case 6: copies_wait<5>(); break;
        default: copies_wait<7>(); break;        // 8
    }
}

// Which columns a thread owns.  A warp covers V chunks of 4 LANES columns, one after the other; a thread has four of each,
// side by side (VEC: rows, strides and pointers allow four elements at once) or LANES apart.  Distances between a thread's
// elements are constants, so a row costs one address per tensor.
template <int LANES, int V, bool VEC> struct Columns {
    int col, width;
    static __device__ __forceinline__ constexpr int apart(int j, int e) { return j * 4 * LANES + (VEC ? e : LANES * e); }
    __device__ __forceinline__ int at(int j, int e) const { return col + apart(j, e); }
    __device__ __forceinline__ bool ok(int j, int e) const { return at(j, VEC ? 0 : e) < width; }
};

template <typename T> struct alignas(4 * sizeof(T) > 16 ? 16 : 4 * sizeof(T)) Quad {
    T v[4];
};
template <typename T> __device__ __forceinline__ Quad<T> load_quad(const T* p) {
    Quad<T> q;
    if constexpr (sizeof(T) == 8) {
        reinterpret_cast<float4*>(&q)[0] = reinterpret_cast<const float4*>(p)[0];
        reinterpret_cast<float4*>(&q)[1] = reinterpret_cast<const float4*>(p)[1];
    } else {
        q = *reinterpret_cast<const Quad<T>*>(p);
    }
    return q;
}
template <typename T> __device__ __forceinline__ void store_quad(T* p, const Quad<T>& q) {
    if constexpr (sizeof(T) == 8) {
        reinterpret_cast<float4*>(p)[0] = reinterpret_cast<const float4*>(&q)[0];
        reinterpret_cast<float4*>(p)[1] = reinterpret_cast<const float4*>(&q)[1];
    } else {
        *reinterpret_cast<Quad<T>*>(p) = q;
    }
}

// A thread's elements of one tensor on their way from a row in memory to registers.  Types of less than 4 bytes that
// cannot be copied four at a time have no ring slot: they are loaded where they are used.  T is the block's most threads:
// a slot's pieces are arrays over T threads, so that all distances in a stage are constants too.  `row` and `slot` point to
// the thread's own first element and place.
template <typename E, int LANES, int V, bool VEC, int T> struct Feed {
    using Cols = Columns<LANES, V, VEC>;
    static constexpr bool kRing = VEC || sizeof(E) >= 4;
    static constexpr int kPiece = VEC ? (4 * sizeof(E) > 16 ? 16 : 4 * (int)sizeof(E)) : (int)sizeof(E);
    static constexpr int kPieces = 4 * (int)sizeof(E) / kPiece;             // per chunk
    static constexpr int kBytes = kRing ? 4 * (int)sizeof(E) * V * T : 0;   // of a stage

    static __device__ __forceinline__ void issue(uint32_t stage, const E* row, const Cols& c) {
        if constexpr (!kRing) return;
        const uint32_t dst = stage + threadIdx.x * kPiece;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if constexpr (VEC) {
                if (c.ok(j, 0))
#pragma unroll
                    for (int p = 0; p < kPieces; ++p)
                        copy_async<kPiece>(dst + (j * kPieces + p) * T * kPiece,
                                           reinterpret_cast<const char*>(row + Cols::apart(j, 0)) + p * kPiece);
            } else if constexpr (kRing) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c.ok(j, e)) copy_async<kPiece>(dst + (4 * j + e) * T * kPiece, row + Cols::apart(j, e));
            }
        }
    }
    static __device__ __forceinline__ void take(const char* stage, const E* row, const Cols& c, int j, E (&v)[4]) {
        const char* src = stage + threadIdx.x * kPiece;
        if constexpr (VEC) {
            Quad<E> q{};
            if (c.ok(j, 0)) {
                if constexpr (kPieces == 2) {
                    reinterpret_cast<float4*>(&q)[0] = *reinterpret_cast<const float4*>(src + (2 * j) * T * kPiece);
                    reinterpret_cast<float4*>(&q)[1] = *reinterpret_cast<const float4*>(src + (2 * j + 1) * T * kPiece);
                } else {
                    q = *reinterpret_cast<const Quad<E>*>(src + j * T * kPiece);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = q.v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = E{};
                if (!c.ok(j, e)) continue;
                if constexpr (kRing) v[e] = *reinterpret_cast<const E*>(src + (4 * j + e) * T * kPiece);
                else v[e] = row[Cols::apart(j, e)];
            }
        }
    }
};

// `row`: the thread's own first element, here and below
template <typename T, int LANES, int V, bool VEC>
__device__ __forceinline__ void put(T* row, const Columns<LANES, V, VEC>& c, int j, const T (&v)[4]) {
    if constexpr (VEC) {
        if (!c.ok(j, 0)) return;
        Quad<T> q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[e] = v[e];
        store_quad(row + c.apart(j, 0), q);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c.ok(j, e)) row[c.apart(j, e)] = v[e];
    }
}

// Four values of a parameter (or a shared gate row); 0 beyond the row.
template <typename T, int LANES, int V, bool VEC>
__device__ __forceinline__ void get(const T* row, const Columns<LANES, V, VEC>& c, int j, T (&v)[4]) {
    if constexpr (VEC) {
        Quad<T> q{};
        if (c.ok(j, 0)) q = load_quad(row + c.apart(j, 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = q.v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c.ok(j, e) ? row[c.apart(j, e)] : T(0);
    }
}

// v = (v - mean) * rstd for the row's own columns, 0 beyond them
template <typename B, int LANES, int V, bool VEC>
__device__ __forceinline__ void normalise(const Columns<LANES, V, VEC>& c, int j, B mean, B rstd, B (&v)[4]) {
    if constexpr (VEC) {                                   // beyond the row v is 0 and so are both moments taken
        const B m = c.ok(j, 0) ? mean : B(0), r = c.ok(j, 0) ? rstd : B(0);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (v[e] - m) * r;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c.ok(j, e) ? (v[e] - mean) * rstd : B(0);
    }
}

// 1 / sqrt: the float approximation (2 ulp) and a Newton step, instead of a correctly rounded root and division
__device__ __forceinline__ float rsqrt_newton(float v) {
    const float r = rsqrtf(v);
    return r * fmaf(-0.5f * v * r, r, 1.5f);
}
__device__ __forceinline__ double rsqrt_newton(double v) { return 1.0 / sqrt(v); }

// ---- the team and its sums ------------------------------------------------------------------------------------------
struct TeamScratch {                       // per block, in shared memory
    static constexpr int kMaxSums = 2, kMaxCluster = 8;
    double warp[2][16][kMaxSums];          // by warp of the block; float teams use half of it
    double block[2][kMaxSums][kMaxCluster];
};

template <typename B, int LANES, bool BIG> struct Team {
    TeamScratch* scratch;
    int warps, team, warp, lane;           // warps of this block in a row's team; team and warp within the team
    int cluster, rank;
    int phase = 0;

    template <int K> __device__ __forceinline__ void sum(B (&v)[K]) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
        if (LANES < 32 || (warps == 1 && (!BIG || cluster == 1))) return;
        // alternating buffers: a warp can only be one sum ahead of the others, so one barrier per sum is enough
        phase ^= 1;
        B* mine = reinterpret_cast<B*>(scratch->warp[phase]) + team * warps * K;
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) mine[warp * K + k] = v[k];
        asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(warps * 32) : "memory");
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = mine[k];
        for (int w = 1; w < warps; ++w)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += mine[w * K + k];
        if (BIG && cluster > 1) {
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

// Rows of one team: item after item, `chunk` rows each.  Every team of a warp makes the same number of steps; a step
// beyond an item's or the matrix's end is not active.
struct RowCursor {
    uint32_t item, row, last;
    int pos;
    __device__ __forceinline__ void enter(const RingPlan& p) {
        pos = 0;
        row = item;
        last = item + 1;
        if (p.shared) {
            const uint32_t span = item / (uint32_t)p.per_span;
            row = span * (uint32_t)p.span + (item - span * (uint32_t)p.per_span) * (uint32_t)p.chunk;
            last = min(row + (uint32_t)p.chunk, (span + 1) * (uint32_t)p.span);
        }
        if (item >= (uint32_t)p.items) last = row = 0;
    }
    __device__ __forceinline__ bool active() const { return row < last; }
    __device__ __forceinline__ void next(const RingPlan& p) {
        ++row;
        if (++pos >= p.chunk) {
            item += (uint32_t)p.teams;
            enter(p);
        }
    }
};
// start of a row: rows and strides are below 2^31 here, so one wide multiplication
template <typename T> __device__ __forceinline__ T* row_at(T* base, uint32_t row, int64_t stride) {
    return base + (uint64_t)row * (uint32_t)stride;
}

template <int LANES, int V, bool VEC, bool BIG, typename B>
__device__ __forceinline__ void set_up(const RingPlan& p, int width, TeamScratch* scratch, Team<B, LANES, BIG>& team,
                                       Columns<LANES, V, VEC>& c, uint32_t& team_id, uint32_t& first_of_warp) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    team.scratch = scratch;
    team.cluster = BIG ? p.cluster : 1;
    team.rank = BIG && p.cluster > 1 ? (int)(blockIdx.x % p.cluster) : 0;
    const uint32_t group = BIG && p.cluster > 1 ? blockIdx.x / p.cluster : blockIdx.x;
    if (LANES == 32) {
        team.warps = p.warps;
        team.team = p.teams_per_block == 1 ? 0 : warp / p.warps;
        team.warp = warp - team.team * p.warps;
        team.lane = lane;
        c.col = (team.rank * p.warps + team.warp) * V * kPackGroup + (VEC ? 4 * lane : lane);
        team_id = group * p.teams_per_block + team.team;
        first_of_warp = team_id;
    } else {
        team.warps = 1;
        team.team = 0;
        team.warp = 0;
        team.lane = lane & (LANES - 1);
        c.col = VEC ? 4 * team.lane : team.lane;
        team_id = group * p.teams_per_block + threadIdx.x / LANES;
        first_of_warp = group * p.teams_per_block + warp * (32 / LANES);
    }
    c.width = width;
    if (BIG && p.cluster > 1) cooperative_groups::this_cluster().sync();      // every block's scratch exists
}

// Codes of a thread's elements and, from one lane each, the scales of their groups.  A group is a warp's chunk, or with
// fewer lanes 32 / LANES chunks of the same threads.
template <typename B, int LANES, int V, bool VEC>
__device__ __forceinline__ void put_codes(int format, const B (&v)[V][4], const Columns<LANES, V, VEC>& c, bool write,
                                          uint8_t* codes, B* scales, int lane) {
    constexpr int kTogether = 32 / LANES < V ? 32 / LANES : V;
#pragma unroll
    for (int j0 = 0; j0 < V; j0 += kTogether) {
        typename AbsBits<B>::type top = 0;
#pragma unroll
        for (int j = j0; j < j0 + kTogether; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, AbsBits<B>::of(c.ok(j, e) ? v[j][e] : B(0)));
        const B scale = pack_scale<B>(format, AbsBits<B>::back(lanes_max<LANES>(top))), inv = pack_inverse<B>(scale);
        if (!write) continue;
#pragma unroll
        for (int j = j0; j < j0 + kTogether; ++j) {
            uint8_t q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = (uint8_t)to_code(format, v[j][e], inv);
            put<uint8_t, LANES, V, VEC>(codes, c, j, q);
        }
        if (lane == 0 && c.at(j0, 0) < c.width) scales[c.at(j0, 0) / kPackGroup] = scale;
    }
}

#define KANB200_EACH(j, e)                  \
    _Pragma("unroll") for (int j = 0; j < V; ++j) _Pragma("unroll") for (int e = 0; e < 4; ++e)

// ---- forward ----------------------------------------------------------------------------------------------------------
template <typename S, int LANES, int V, bool VEC, bool BRANCH, bool BIG>
__global__ void __launch_bounds__(ring_threads(BIG), ring_blocks(false, BRANCH, BIG, sizeof(S) == 8))
    ring_forward_kernel(const __grid_constant__ kanb200_block_args a, const __grid_constant__ RingPlan p) {
    using B = Br<S>;
    constexpr int T = ring_threads(BIG);
    using FS = Feed<S, LANES, V, VEC, T>;
    using FB = Feed<B, LANES, V, VEC, T>;
    constexpr int at_y = FS::kBytes, at_gate = at_y + FB::kBytes;
    extern __shared__ __align__(16) char ring[];
    __shared__ TeamScratch scratch;
    Team<B, LANES, BIG> team;
    Columns<LANES, V, VEC> c;
    uint32_t team_id, first_of_warp;
    set_up<LANES, V, VEC, BIG, B>(p, (int)a.width, &scratch, team, c, team_id, first_of_warp);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const bool row_gate = BRANCH && a.gate && !p.shared;
    const int D = (int)a.width, groups = (D + kPackGroup - 1) / kPackGroup;
    const B eps = B(a.eps), per = B(1) / B(D);

    const S* x = static_cast<const S*>(a.x) + c.col;
    const B *y = static_cast<const B*>(a.y) + c.col, *gate = static_cast<const B*>(a.gate) + c.col,
            *scale = static_cast<const B*>(a.scale) + c.col, *pw = static_cast<const B*>(a.post_weight) + c.col,
            *pb = static_cast<const B*>(a.post_bias) + c.col, *nw = static_cast<const B*>(a.next_weight) + c.col,
            *nb = static_cast<const B*>(a.next_bias) + c.col;

    const auto issue = [&](const RowCursor& r, int stage) {
        if (r.active()) {
            const uint32_t at = ring_at + stage * p.stage_bytes;
            FS::issue(at, row_at(x, r.row, a.x_stride), c);
            if (BRANCH) FB::issue(at + at_y, row_at(y, r.row, a.y_stride), c);
            if (row_gate) FB::issue(at + at_gate, row_at(gate, r.row, a.gate_stride), c);
        }
        copies_commit();
    };
    // the row's mean and 1 / deviation; two passes over registers, so that the variance has no cancellation
    const auto moments = [&](int kind, const B (&v)[V][4], B& mean, B& rstd) {
        mean = B(0);
        B s[1] = {B(0)};
        if (kind == kNormLayer) {
            KANB200_EACH(j, e) s[0] += v[j][e];             // columns beyond the row hold 0
            team.template sum<1>(s);
            mean = s[0] * per;
            s[0] = B(0);
        }
        KANB200_EACH(j, e) {
            const B d = c.ok(j, e) ? v[j][e] - mean : B(0);
            s[0] += d * d;
        }
        team.template sum<1>(s);
        rstd = rsqrt_newton(s[0] * per + eps);
    };
    const auto put_stats = [&](void* stats, uint32_t row, B mean, B rstd) {
        if (c.col == 0) {
            B* at = static_cast<B*>(stats) + 2 * (uint64_t)row;
            at[0] = mean;
            at[1] = rstd;
        }
    };

    RowCursor now, ahead;
    now.item = team_id;
    now.enter(p);
    ahead = now;
    for (int s = 0; s + 1 < p.stages; ++s) {
        issue(ahead, s);
        ahead.next(p);
    }
    int stage = 0;
    B t[V][4];                                              // scale act(gate) of a shared gate
    for (uint32_t lead = first_of_warp; lead < (uint32_t)p.items;) {
        issue(ahead, stage == 0 ? p.stages - 1 : stage - 1);
        ahead.next(p);
        copies_wait_oldest(p.stages);
        const bool live = now.active();
        const char* at = ring + stage * p.stage_bytes;
        const uint32_t row = now.row;
        const uint64_t dense = (uint64_t)row * (uint32_t)D + (uint32_t)c.col;      // of dense tensors
        B o[V][4] = {};
        if (BRANCH) {
            B v[V][4] = {};
            if (live)
#pragma unroll
                for (int j = 0; j < V; ++j) FB::take(at + at_y, row_at(y, row, a.y_stride), c, j, v[j]);
            if (a.y_codes)
                put_codes<B, LANES, V, VEC>(a.checkpoint, v, c, live, static_cast<uint8_t*>(a.y_codes) + dense,
                                            row_at(static_cast<B*>(a.y_scales), row, groups), team.lane);
            B mean = B(0), rstd = B(1);
            if (a.post_norm != kNormNone) {
                moments(a.post_norm, v, mean, rstd);
                if (a.post_stats && live) put_stats(a.post_stats, row, mean, rstd);
            }
            if (p.shared && now.pos == 0 && live) {
                const B* shared = row_at(gate, row / (uint32_t)a.gate_rows, a.gate_stride);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    get<B, LANES, V, VEC>(shared, c, j, t[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[j][e] = gate_value<B>(a.gate_act, t[j][e]);
                }
            }
            // out = x + scale act(gate) z; what v becomes is the branch's summand
#pragma unroll
            for (int j = 0; j < V; ++j) {
                B w[4];
                normalise<B>(c, j, mean, rstd, v[j]);
                if (a.post_weight) {
                    get<B, LANES, V, VEC>(pw, c, j, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] *= w[e];
                }
                if (a.post_bias) {
                    get<B, LANES, V, VEC>(pb, c, j, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] += w[e];
                }
                if (p.shared)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] *= t[j][e];
                if (a.scale) {
                    get<B, LANES, V, VEC>(scale, c, j, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] *= w[e];
                }
            }
            if (row_gate) {
                B g[V][4] = {};
                if (live)
#pragma unroll
                    for (int j = 0; j < V; ++j) FB::take(at + at_gate, row_at(gate, row, a.gate_stride), c, j, g[j]);
                if (a.gate_codes)
                    put_codes<B, LANES, V, VEC>(a.checkpoint, g, c, live, static_cast<uint8_t*>(a.gate_codes) + dense,
                                                row_at(static_cast<B*>(a.gate_scales), row, groups), team.lane);
                KANB200_EACH(j, e) v[j][e] *= gate_value<B>(a.gate_act, g[j][e]);
            }
            if (live)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    S xv[4];
                    FS::take(at, row_at(x, row, a.x_stride), c, j, xv);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        xv[e] = narrow<S>(widen(xv[e]) + v[j][e]);
                        o[j][e] = c.ok(j, e) ? widen(xv[e]) : B(0);
                    }
                    put<S, LANES, V, VEC>(static_cast<S*>(a.out) + dense, c, j, xv);
                }
        } else if (live) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                S xv[4];
                FS::take(at, row_at(x, row, a.x_stride), c, j, xv);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] = widen(xv[e]);
            }
        }
        if (a.x_codes)
            put_codes<B, LANES, V, VEC>(a.checkpoint, o, c, live, static_cast<uint8_t*>(a.x_codes) + dense,
                                        row_at(static_cast<B*>(a.x_scales), row, groups), team.lane);
        if (!BRANCH || a.next_norm != kNormNone) {
            B mean, rstd;
            moments(a.next_norm, o, mean, rstd);
            if (a.next_stats && live) put_stats(a.next_stats, row, mean, rstd);
            if (live)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    B w[4];
                    normalise<B>(c, j, mean, rstd, o[j]);
                    if (a.next_weight) {
                        get<B, LANES, V, VEC>(nw, c, j, w);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][e] *= w[e];
                    }
                    if (a.next_bias) {
                        get<B, LANES, V, VEC>(nb, c, j, w);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][e] += w[e];
                    }
                    put<B, LANES, V, VEC>(static_cast<B*>(a.h) + dense, c, j, o[j]);
                }
        }
        now.next(p);
        if (now.pos == 0) lead += (uint32_t)p.teams;
        stage = stage + 1 == p.stages ? 0 : stage + 1;
    }
    copies_wait<0>();
}

// ---- backward -----------------------------------------------------------------------------------------------------------
template <typename S, int LANES, int V, bool VEC, bool BRANCH, bool NEXT, bool BIG>
__global__ void __launch_bounds__(ring_threads(BIG), ring_blocks(true, BRANCH, BIG, sizeof(S) == 8))
    ring_backward_kernel(const __grid_constant__ kanb200_block_args a, const __grid_constant__ RingPlan p,
                         const __grid_constant__ BackwardSlabs slabs) {
    using B = Br<S>;
    constexpr int T = ring_threads(BIG);
    using FS = Feed<S, LANES, V, VEC, T>;
    using FB = Feed<B, LANES, V, VEC, T>;
    using FQ = Feed<uint8_t, LANES, V, VEC, T>;
    using At = BackwardStage<NEXT, BRANCH, V, T, VEC, (int)sizeof(S), (int)sizeof(B)>;
    extern __shared__ __align__(16) char ring[];
    __shared__ TeamScratch scratch;
    Team<B, LANES, BIG> team;
    Columns<LANES, V, VEC> c;
    uint32_t team_id, first_of_warp;
    set_up<LANES, V, VEC, BIG, B>(p, (int)a.width, &scratch, team, c, team_id, first_of_warp);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const int D = (int)a.width, groups = (D + kPackGroup - 1) / kPackGroup;
    const bool row_gate = BRANCH && (a.gate || a.gate_codes) && !p.shared;
    const B per = B(1) / B(D);

    const S *x = static_cast<const S*>(a.x) + c.col, *dout = static_cast<const S*>(a.dout) + c.col;
    const B *y = static_cast<const B*>(a.y) + c.col, *gate = static_cast<const B*>(a.gate) + c.col,
            *dh = static_cast<const B*>(a.dh) + c.col, *scale = static_cast<const B*>(a.scale) + c.col,
            *pw = static_cast<const B*>(a.post_weight) + c.col, *pb = static_cast<const B*>(a.post_bias) + c.col,
            *nw = static_cast<const B*>(a.next_weight) + c.col;
    B sum_scale[V][4] = {}, sum_pw[V][4] = {}, sum_pb[V][4] = {}, sum_nw[V][4] = {}, sum_nb[V][4] = {}, sum_gate[V][4] = {};

    // a tensor that may be there as codes: codes and their groups' scales, or the values themselves
    const auto issue_kept = [&](uint32_t at, const void* codes, const void* scales, auto* values, int64_t stride, uint32_t row) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(values)>>;
        if (codes) {
            FQ::issue(at, static_cast<const uint8_t*>(codes) + (uint64_t)row * (uint32_t)D + (uint32_t)c.col, c);
            const B* from = static_cast<const B*>(scales) + (uint64_t)row * (uint32_t)groups + c.col / kPackGroup;
            const uint32_t dst = at + 4 * V * T + threadIdx.x * (uint32_t)sizeof(B);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c.at(j, 0) < D) copy_async<sizeof(B)>(dst + j * T * (uint32_t)sizeof(B), from + j * 4 * LANES / kPackGroup);
        } else {
            Feed<E, LANES, V, VEC, T>::issue(at, row_at(values, row, stride), c);
        }
    };
    const auto take_kept = [&](const char* at, const void* codes, auto* values, int64_t stride, uint32_t row, int j, B (&v)[4]) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(values)>>;
        if (codes) {
            uint8_t q[4];
            FQ::take(at, static_cast<const uint8_t*>(codes) + (uint64_t)row * (uint32_t)D + (uint32_t)c.col, c, j, q);
            const B s = c.at(j, 0) < D ? *reinterpret_cast<const B*>(at + 4 * V * T + (j * T + threadIdx.x) * sizeof(B)) : B(0);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = from_code<B>(a.checkpoint, q[e], s);
        } else {
            E raw[4];
            Feed<E, LANES, V, VEC, T>::take(at, row_at(values, row, stride), c, j, raw);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = widen(raw[e]);
        }
    };
    const auto issue = [&](const RowCursor& r, int stage) {
        if (r.active()) {
            const uint32_t at = ring_at + stage * p.stage_bytes;
            if (a.dout) FS::issue(at + At::dout, row_at(dout, r.row, a.dout_stride), c);
            if (NEXT) {
                FB::issue(at + At::dh, row_at(dh, r.row, a.dh_stride), c);
                issue_kept(at + At::x, a.x_codes, a.x_scales, x, a.x_stride, r.row);
                copy_async<2 * sizeof(B)>(at + At::next_stats + threadIdx.x * 2 * (uint32_t)sizeof(B),
                                          static_cast<const B*>(a.next_stats) + 2 * (uint64_t)r.row);
            }
            if (BRANCH) {
                issue_kept(at + At::y, a.y_codes, a.y_scales, y, a.y_stride, r.row);
                if (row_gate) issue_kept(at + At::gate, a.gate_codes, a.gate_scales, gate, a.gate_stride, r.row);
                if (a.post_norm != kNormNone)
                    copy_async<2 * sizeof(B)>(at + At::post_stats + threadIdx.x * 2 * (uint32_t)sizeof(B),
                                              static_cast<const B*>(a.post_stats) + 2 * (uint64_t)r.row);
            }
        }
        copies_commit();
    };

    RowCursor now, ahead;
    now.item = team_id;
    now.enter(p);
    ahead = now;
    for (int s = 0; s + 1 < p.stages; ++s) {
        issue(ahead, s);
        ahead.next(p);
    }
    int stage = 0;
    for (uint32_t lead = first_of_warp; lead < (uint32_t)p.items;) {
        issue(ahead, stage == 0 ? p.stages - 1 : stage - 1);
        ahead.next(p);
        copies_wait_oldest(p.stages);
        const bool live = now.active();
        const char* at = ring + stage * p.stage_bytes;
        const uint32_t row = now.row;
        const uint64_t dense = (uint64_t)row * (uint32_t)D + (uint32_t)c.col;      // of dense tensors
        B g[V][4] = {};                                     // gradient of the norm's input, then of y
        if (a.dout && live)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                S raw[4];
                FS::take(at + At::dout, row_at(dout, row, a.dout_stride), c, j, raw);
#pragma unroll
                for (int e = 0; e < 4; ++e) g[j][e] = widen(raw[e]);
            }
        if (NEXT) {
            B v[V][4] = {}, d[V][4] = {}, mean = B(0), rstd = B(0), s[2] = {B(0), B(0)};
            if (live) {
                const B* stats = reinterpret_cast<const B*>(at + At::next_stats + threadIdx.x * 2 * sizeof(B));
                mean = stats[0];
                rstd = stats[1];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    FB::take(at + At::dh, row_at(dh, row, a.dh_stride), c, j, d[j]);
                    take_kept(at + At::x, a.x_codes, x, a.x_stride, row, j, v[j]);
                    normalise<B>(c, j, mean, rstd, v[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sum_nw[j][e] += d[j][e] * v[j][e];
                        sum_nb[j][e] += d[j][e];
                    }
                    if (a.next_weight) {
                        B w[4];
                        get<B, LANES, V, VEC>(nw, c, j, w);
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[j][e] *= w[e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[0] += d[j][e];
                        s[1] += d[j][e] * v[j][e];
                    }
                }
            }
            team.template sum<2>(s);
            const B flat = a.next_norm == kNormLayer ? s[0] * per : B(0), along = s[1] * per;
            KANB200_EACH(j, e) g[j][e] += rstd * (d[j][e] - flat - v[j][e] * along);
        }
        if (a.dx && live)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                S o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = narrow<S>(g[j][e]);
                put<S, LANES, V, VEC>(static_cast<S*>(a.dx) + dense, c, j, o);
            }
        if (BRANCH) {
            B v[V][4] = {}, mean = B(0), rstd = B(1), s[2] = {B(0), B(0)};
            if (live) {
                if (a.post_norm != kNormNone) {
                    const B* stats = reinterpret_cast<const B*>(at + At::post_stats + threadIdx.x * 2 * sizeof(B));
                    mean = stats[0];
                    rstd = stats[1];
                }
                const B* shared = p.shared ? row_at(gate, row / (uint32_t)a.gate_rows, a.gate_stride) : nullptr;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    B w[4], act[4], dact[4], z[4];
                    take_kept(at + At::y, a.y_codes, y, a.y_stride, row, j, v[j]);
                    normalise<B>(c, j, mean, rstd, v[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        z[e] = v[j][e];
                        act[e] = B(1);
                        dact[e] = B(0);
                    }
                    if (a.post_weight) {
                        get<B, LANES, V, VEC>(pw, c, j, w);
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[e] *= w[e];
                    }
                    if (a.post_bias) {
                        B b[4];
                        get<B, LANES, V, VEC>(pb, c, j, b);
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[e] += b[e];
                    }
                    if (p.shared || row_gate) {
                        B gv[4];
                        if (p.shared) get<B, LANES, V, VEC>(shared, c, j, gv);
                        else take_kept(at + At::gate, a.gate_codes, gate, a.gate_stride, row, j, gv);
#pragma unroll
                        for (int e = 0; e < 4; ++e) gate_value_grad<B>(a.gate_act, gv[e], act[e], dact[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum_scale[j][e] += g[j][e] * act[e] * z[e];
                    if (a.scale) {
                        B sc[4];
                        get<B, LANES, V, VEC>(scale, c, j, sc);
#pragma unroll
                        for (int e = 0; e < 4; ++e) g[j][e] *= sc[e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        z[e] *= g[j][e] * dact[e];                          // this row's share of dgate
                        g[j][e] *= act[e];
                        sum_pw[j][e] += g[j][e] * v[j][e];
                        sum_pb[j][e] += g[j][e];
                    }
                    if (p.shared) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum_gate[j][e] += z[e];
                    } else if (a.dgate) {
                        put<B, LANES, V, VEC>(row_at(static_cast<B*>(a.dgate) + c.col, row, a.dgate_stride), c, j, z);
                    }
                    if (a.post_weight)
#pragma unroll
                        for (int e = 0; e < 4; ++e) g[j][e] *= w[e];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[0] += g[j][e];
                        s[1] += g[j][e] * v[j][e];
                    }
                }
            }
            if (a.dy) {
                if (a.post_norm != kNormNone) {
                    team.template sum<2>(s);
                    const B flat = a.post_norm == kNormLayer ? s[0] * per : B(0), along = s[1] * per;
                    KANB200_EACH(j, e) g[j][e] = rstd * (g[j][e] - flat - v[j][e] * along);
                }
                if (live)
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        put<B, LANES, V, VEC>(row_at(static_cast<B*>(a.dy) + c.col, row, a.dy_stride), c, j, g[j]);
            }
            if (slabs.gate && now.pos + 1 == p.chunk) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (now.item < (uint32_t)p.items)
                        put<B, LANES, V, VEC>(static_cast<B*>(slabs.gate) + (uint64_t)now.item * (uint32_t)D + c.col, c, j, sum_gate[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum_gate[j][e] = B(0);
                }
            }
        }
        now.next(p);
        if (now.pos == 0) lead += (uint32_t)p.teams;
        stage = stage + 1 == p.stages ? 0 : stage + 1;
    }
    copies_wait<0>();

    // one slab row per block: the teams' sums, added in the order of the teams
    const uint32_t block = BIG && p.cluster > 1 ? blockIdx.x / p.cluster : blockIdx.x;
    Quad<B>* shelf = reinterpret_cast<Quad<B>*>(ring);
    const int per_team = blockDim.x / p.teams_per_block;
    const auto leave = [&](int which, B (&v)[V][4]) {
        if (!slabs.column[which]) return;
        B* row = static_cast<B*>(slabs.column[which]) + (uint64_t)block * (uint32_t)D + c.col;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (p.teams_per_block > 1) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 4; ++e) shelf[threadIdx.x].v[e] = v[j][e];
                __syncthreads();
                if ((int)threadIdx.x >= per_team) continue;
                for (int i = 1; i < p.teams_per_block; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] += shelf[i * per_team + threadIdx.x].v[e];
            }
            put<B, LANES, V, VEC>(row, c, j, v[j]);
        }
    };
    if (BRANCH) {
        leave(kSumScale, sum_scale);
        leave(kSumPostWeight, sum_pw);
        leave(kSumPostBias, sum_pb);
    }
    if (NEXT) {
        leave(kSumNextWeight, sum_nw);
        leave(kSumNextBias, sum_nb);
    }
}
#undef KANB200_EACH

}  // namespace kanb200

// ---- launches: included by one source per stream type ---------------------------------------------------------------
namespace kanb200 {

template <typename... P>
cudaError_t ring_launch(const RingPlan& p, cudaStream_t st, void (*kernel)(P...), const P&... args) {
    const int bytes = p.stages * p.stage_bytes;
    cudaError_t e = cudaSuccess;
    if (bytes > 48 * 1024 - (int)sizeof(TeamScratch))
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
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

template <typename S, int LANES, bool VEC, bool BIG>
cudaError_t ring_forward_as(const kanb200_block_args& a, const RingPlan& p, cudaStream_t st) {
    constexpr bool f64 = sizeof(S) == 8;
    return a.y ? ring_launch(p, st, ring_forward_kernel<S, LANES, ring_chunks(false, true, f64), VEC, true, BIG>, a, p)
               : ring_launch(p, st, ring_forward_kernel<S, LANES, ring_chunks(false, false, f64), VEC, false, BIG>, a, p);
}
template <typename S, int LANES, bool VEC, bool BIG>
cudaError_t ring_backward_as(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st) {
    constexpr bool f64 = sizeof(S) == 8;
    constexpr int alone = ring_chunks(true, false, f64), branch = ring_chunks(true, true, f64);
    if (!a.has_branch) return ring_launch(p, st, ring_backward_kernel<S, LANES, alone, VEC, false, true, BIG>, a, p, slabs);
    return a.dh ? ring_launch(p, st, ring_backward_kernel<S, LANES, branch, VEC, true, true, BIG>, a, p, slabs)
                : ring_launch(p, st, ring_backward_kernel<S, LANES, branch, VEC, true, false, BIG>, a, p, slabs);
}

#define KANB200_RING_DISPATCH(name, ...)                                                                    \
    if (p.big) return p.vec ? name<S, 32, true, true>(__VA_ARGS__) : name<S, 32, false, true>(__VA_ARGS__);       \
    if (p.lanes == 32) return p.vec ? name<S, 32, true, false>(__VA_ARGS__) : name<S, 32, false, false>(__VA_ARGS__); \
    if (p.lanes == 16) return p.vec ? name<S, 16, true, false>(__VA_ARGS__) : name<S, 16, false, false>(__VA_ARGS__); \
    if (p.lanes == 8) return p.vec ? name<S, 8, true, false>(__VA_ARGS__) : name<S, 8, false, false>(__VA_ARGS__);    \
    return p.vec ? name<S, 4, true, false>(__VA_ARGS__) : name<S, 4, false, false>(__VA_ARGS__)

template <typename S> cudaError_t ring_forward(const kanb200_block_args& a, const RingPlan& p, cudaStream_t st) {
    KANB200_RING_DISPATCH(ring_forward_as, a, p, st);
}
template <typename S>
cudaError_t ring_backward(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st) {
    KANB200_RING_DISPATCH(ring_backward_as, a, p, slabs, st);
}
#undef KANB200_RING_DISPATCH

}  // namespace kanb200

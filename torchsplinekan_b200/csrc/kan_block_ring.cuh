// The norm and the gated residual connection for rows of up to 32768 columns (16384 in float64): every thread owns four
// columns for the whole launch, and its share of the next rows is already on its way into shared memory.
//
//   * A team of threads owns a row at a time: 8 or 16 lanes (up to 32 / 64 columns), W warps (128 columns each), or the
//     warps of a cluster of up to 8 blocks.  A warp's 128 columns are one group of a checkpoint, so its scale needs one
//     warp maximum.  Teams take rows (or, with a shared gate, runs of rows under one gate row) in turn.
//   * Memory -> registers goes through a ring of 2 to 8 rows in shared memory, filled by cp.async.  A thread copies
//     exactly what it reads back itself, so the ring needs no barrier: only its own cp.async group to have landed.  The
//     bytes in flight then do not depend on registers or on how many warps wait in a barrier.
//   * Parameters stay in registers, and so do the sums over rows that are their gradients; one slab row per block leaves
//     the kernel at its end.
//   * Sums over a row: lanes by shuffles, warps through shared memory with a barrier of the team alone, blocks of a
//     cluster through each other's shared memory; every thread gets the same bits.
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

// Which four columns a thread owns: col + e (VEC: rows, strides and pointers allow four elements at once) or
// col + LANES * e.  Either way the lanes of a warp cover the same 128 columns.
template <int LANES, bool VEC> struct Columns {
    int col, width;
    __device__ __forceinline__ int at(int e) const { return VEC ? col + e : col + LANES * e; }
    __device__ __forceinline__ bool ok(int e) const { return VEC ? col < width : at(e) < width; }
};

template <typename T> struct alignas(4 * sizeof(T) > 16 ? 16 : 4 * sizeof(T)) Quad {
    T v[4];
};

// A thread's four elements of one tensor on their way from a row in memory to registers.  Types of less than 4 bytes that
// cannot be copied four at a time have no ring slot: they are loaded where they are used.
template <typename T, int LANES, bool VEC> struct Feed {
    using Cols = Columns<LANES, VEC>;
    static constexpr bool kRing = VEC || sizeof(T) >= 4;
    static constexpr int kBytes = kRing ? 4 * (int)sizeof(T) : 0;       // per thread and stage
    static constexpr int kPiece = VEC ? (4 * sizeof(T) > 16 ? 16 : 4 * (int)sizeof(T)) : (int)sizeof(T);
    static constexpr int kPieces = kRing ? kBytes / kPiece : 0;

    // `slot`: this tensor's part of the stage; its pieces are arrays over the block's threads
    static __device__ __forceinline__ void issue(uint32_t slot, const T* row, const Cols& c) {
        const uint32_t dst = slot + threadIdx.x * kPiece, step = blockDim.x * kPiece;
        if constexpr (VEC) {
            if (c.ok(0))
#pragma unroll
                for (int p = 0; p < kPieces; ++p)
                    copy_async<kPiece>(dst + p * step, reinterpret_cast<const char*>(row + c.col) + p * kPiece);
        } else if constexpr (kRing) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c.ok(e)) copy_async<kPiece>(dst + e * step, row + c.at(e));
        }
    }
    static __device__ __forceinline__ void take(const char* slot, const T* row, const Cols& c, T (&v)[4]) {
        if constexpr (VEC) {
            Quad<T> q{};
            if (c.ok(0)) {
                const char* src = slot + threadIdx.x * kPiece;
                if constexpr (kPieces == 2) {
                    reinterpret_cast<float4*>(&q)[0] = *reinterpret_cast<const float4*>(src);
                    reinterpret_cast<float4*>(&q)[1] = *reinterpret_cast<const float4*>(src + blockDim.x * kPiece);
                } else {
                    q = *reinterpret_cast<const Quad<T>*>(src);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = q.v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = T{};
                if (!c.ok(e)) continue;
                if constexpr (kRing) v[e] = *reinterpret_cast<const T*>(slot + (e * blockDim.x + threadIdx.x) * kPiece);
                else v[e] = row[c.at(e)];
            }
        }
    }
};

template <typename T, int LANES, bool VEC>
__device__ __forceinline__ void put(T* row, const Columns<LANES, VEC>& c, const T (&v)[4]) {
    if constexpr (VEC) {
        if (!c.ok(0)) return;
        Quad<T> q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[e] = v[e];
        if constexpr (sizeof(T) == 8) {
            reinterpret_cast<float4*>(row + c.col)[0] = reinterpret_cast<const float4*>(&q)[0];
            reinterpret_cast<float4*>(row + c.col)[1] = reinterpret_cast<const float4*>(&q)[1];
        } else {
            *reinterpret_cast<Quad<T>*>(row + c.col) = q;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c.ok(e)) row[c.at(e)] = v[e];
    }
}

template <typename T, int LANES, bool VEC>
__device__ __forceinline__ void get_or(const void* p, const Columns<LANES, VEC>& c, T absent, T (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c.ok(e) ? (p ? static_cast<const T*>(p)[c.at(e)] : absent) : T(0);
}

// ---- the team and its sums ------------------------------------------------------------------------------------------
struct TeamScratch {                       // per block, in shared memory
    static constexpr int kMaxSums = 2, kMaxCluster = 8;
    double warp[2][kMaxSums][32];          // by warp of the block; float teams use half of each slot
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
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (lane == k) *reinterpret_cast<B*>(&scratch->warp[phase][k][team * warps + warp]) = v[k];
        asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(warps * 32) : "memory");
#pragma unroll
        for (int k = 0; k < K; ++k)
            v[k] = lane < warps ? *reinterpret_cast<const B*>(&scratch->warp[phase][k][team * warps + lane]) : B(0);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
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
    int64_t item, row, last;
    int pos;
    __device__ __forceinline__ void enter(const RingPlan& p) {
        if (item >= p.items) {
            row = 0;
            last = 0;
        } else if (p.shared) {
            const int64_t span = item / p.per_span, first = span * p.span + (item - span * p.per_span) * p.chunk;
            row = first;
            last = min(first + p.chunk, (span + 1) * p.span);
        } else {
            row = item;
            last = item + 1;
        }
        pos = 0;
    }
    __device__ __forceinline__ bool active() const { return row < last; }
    __device__ __forceinline__ void next(const RingPlan& p) {
        if (++pos < p.chunk) {
            ++row;
        } else {
            item += p.teams;
            enter(p);
        }
    }
};

template <int LANES, bool VEC, bool BIG, typename B>
__device__ __forceinline__ void set_up(const RingPlan& p, int width, TeamScratch* scratch, Team<B, LANES, BIG>& team,
                                       Columns<LANES, VEC>& c, int64_t& team_id, int64_t& first_of_warp) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    team.scratch = scratch;
    team.cluster = BIG ? p.cluster : 1;
    team.rank = BIG && p.cluster > 1 ? (int)(blockIdx.x % p.cluster) : 0;
    const int64_t group = BIG && p.cluster > 1 ? blockIdx.x / p.cluster : blockIdx.x;
    if (LANES == 32) {
        team.warps = p.warps;
        team.team = p.teams_per_block == 1 ? 0 : warp / p.warps;
        team.warp = warp - team.team * p.warps;
        team.lane = lane;
        const int first = (team.rank * p.warps + team.warp) * kPackGroup;
        c.col = first + (VEC ? 4 * lane : lane);
        team_id = group * p.teams_per_block + team.team;
        first_of_warp = team_id;
    } else {
        team.warps = 1;
        team.team = 0;
        team.warp = 0;
        team.lane = lane & (LANES - 1);
        c.col = VEC ? 4 * team.lane : team.lane;
        team_id = group * p.teams_per_block + (threadIdx.x / LANES);
        first_of_warp = group * p.teams_per_block + warp * (32 / LANES);
    }
    c.width = width;
    if (BIG && p.cluster > 1) cooperative_groups::this_cluster().sync();      // every block's scratch exists
}

// Codes of a thread's four elements and, from one lane, the scale of their group.
template <typename B, int LANES, bool VEC>
__device__ __forceinline__ void put_codes(int format, const B (&v)[4], const Columns<LANES, VEC>& c, bool write,
                                          uint8_t* codes, B* scales, int lane) {
    typename AbsBits<B>::type top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, AbsBits<B>::of(c.ok(e) ? v[e] : B(0)));
    const B scale = pack_scale<B>(format, AbsBits<B>::back(lanes_max<LANES>(top))), inv = pack_inverse<B>(scale);
    if (!write) return;
    uint8_t q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = (uint8_t)to_code(format, v[e], inv);
    put<uint8_t, LANES, VEC>(codes, c, q);
    if (lane == 0 && c.col < c.width) scales[c.col / kPackGroup] = scale;
}

// ---- forward ----------------------------------------------------------------------------------------------------------
template <typename S, int LANES, bool VEC, bool BRANCH, bool BIG>
__global__ void __launch_bounds__(ring_max_threads<S>(BIG), BIG ? 1 : sizeof(S) == 8 ? 2 : 4) ring_forward_kernel(const kanb200_block_args a, const RingPlan p) {
    using B = Br<S>;
    using FS = Feed<S, LANES, VEC>;
    using FB = Feed<B, LANES, VEC>;
    extern __shared__ __align__(16) char ring[];
    __shared__ TeamScratch scratch;
    Team<B, LANES, BIG> team;
    Columns<LANES, VEC> c;
    int64_t team_id, first_of_warp;
    set_up<LANES, VEC, BIG, B>(p, (int)a.width, &scratch, team, c, team_id, first_of_warp);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const int T = blockDim.x;
    const int at_y = FS::kBytes * T, at_gate = at_y + FB::kBytes * T;
    const bool row_gate = BRANCH && a.gate && !p.shared;
    const int64_t D = a.width, groups = (D + kPackGroup - 1) / kPackGroup;

    const S* x = static_cast<const S*>(a.x);
    const B* y = static_cast<const B*>(a.y);
    const B* gate = static_cast<const B*>(a.gate);
    B scale[4], pw[4], pb[4], nw[4], nb[4], t[4];
    if (BRANCH) {
        get_or<B>(a.scale, c, B(1), scale);
        get_or<B>(a.post_weight, c, B(1), pw);
        get_or<B>(a.post_bias, c, B(0), pb);
    }
    get_or<B>(a.next_weight, c, B(1), nw);
    get_or<B>(a.next_bias, c, B(0), nb);
    const B eps = B(a.eps);

    auto issue = [&](const RowCursor& r, int stage) {
        if (r.active()) {
            const uint32_t at = ring_at + stage * p.stage_bytes;
            FS::issue(at, x + r.row * a.x_stride, c);
            if (BRANCH) FB::issue(at + at_y, y + r.row * a.y_stride, c);
            if (row_gate) FB::issue(at + at_gate, gate + r.row * a.gate_stride, c);
        }
        copies_commit();
    };
    auto moments = [&](int kind, const B (&v)[4], B& mean, B& rstd) {
        mean = B(0);
        if (kind == kNormLayer) {
            B s[1] = {v[0] + v[1] + v[2] + v[3]};           // columns beyond the row hold 0
            team.template sum<1>(s);
            mean = s[0] / B(D);
        }
        B s[1] = {B(0)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const B d = c.ok(e) ? v[e] - mean : B(0);
            s[0] += d * d;
        }
        team.template sum<1>(s);
        rstd = inv_sqrt(s[0] / B(D) + eps);
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
    for (int64_t lead = first_of_warp; lead < p.items;) {
        const int into = stage == 0 ? p.stages - 1 : stage - 1;
        issue(ahead, into);
        ahead.next(p);
        copies_wait_oldest(p.stages);
        const bool live = now.active();
        const char* at = ring + stage * p.stage_bytes;
        const int64_t row = now.row;
        if (BRANCH && p.shared && now.pos == 0 && live) {
            B g[4];
            get_or<B>(gate + row / a.gate_rows * a.gate_stride, c, B(0), g);
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = gate_value<B>(a.gate_act, g[e]) * scale[e];
        }
        B o[4];
        {
            S raw[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[e] = S{};
            if (live) FS::take(at, x + row * a.x_stride, c, raw);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = widen(raw[e]);
        }
        if (BRANCH) {
            B v[4] = {B(0), B(0), B(0), B(0)};
            if (live) FB::take(at + at_y, y + row * a.y_stride, c, v);
            if (row_gate) {
                B g[4] = {B(0), B(0), B(0), B(0)};
                if (live) FB::take(at + at_gate, gate + row * a.gate_stride, c, g);
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = gate_value<B>(a.gate_act, g[e]) * scale[e];
                if (a.gate_codes)
                    put_codes<B, LANES, VEC>(a.checkpoint, g, c, live, static_cast<uint8_t*>(a.gate_codes) + row * D,
                                             static_cast<B*>(a.gate_scales) + row * groups, team.lane);
            } else if (!a.gate) {
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = scale[e];
            }
            if (a.y_codes)
                put_codes<B, LANES, VEC>(a.checkpoint, v, c, live, static_cast<uint8_t*>(a.y_codes) + row * D,
                                         static_cast<B*>(a.y_scales) + row * groups, team.lane);
            B mean = B(0), rstd = B(1);
            if (a.post_norm != kNormNone) {
                moments(a.post_norm, v, mean, rstd);
                if (a.post_stats && live && c.col == 0) {
                    static_cast<B*>(a.post_stats)[2 * row] = mean;
                    static_cast<B*>(a.post_stats)[2 * row + 1] = rstd;
                }
            }
            S out[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const B z = (v[e] - mean) * rstd * pw[e] + pb[e];
                out[e] = narrow<S>(o[e] + t[e] * z);
                o[e] = c.ok(e) ? widen(out[e]) : B(0);
            }
            if (live) put<S, LANES, VEC>(static_cast<S*>(a.out) + row * D, c, out);
        }
        if (a.x_codes)
            put_codes<B, LANES, VEC>(a.checkpoint, o, c, live, static_cast<uint8_t*>(a.x_codes) + row * D,
                                     static_cast<B*>(a.x_scales) + row * groups, team.lane);
        if (a.next_norm != kNormNone) {
            B mean, rstd;
            moments(a.next_norm, o, mean, rstd);
            if (a.next_stats && live && c.col == 0) {
                static_cast<B*>(a.next_stats)[2 * row] = mean;
                static_cast<B*>(a.next_stats)[2 * row + 1] = rstd;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (o[e] - mean) * rstd * nw[e] + nb[e];
            if (live) put<B, LANES, VEC>(static_cast<B*>(a.h) + row * D, c, o);
        }
        now.next(p);
        if (now.pos == 0) lead += p.teams;
        stage = stage + 1 == p.stages ? 0 : stage + 1;
    }
    copies_wait<0>();
}

// ---- backward -----------------------------------------------------------------------------------------------------------
template <typename S, int LANES, bool VEC, bool BRANCH, bool NEXT, bool BIG>
__global__ void __launch_bounds__(ring_max_threads<S>(BIG), BIG ? 1 : 2)
    ring_backward_kernel(const kanb200_block_args a, const RingPlan p, const BackwardSlabs slabs) {
    using B = Br<S>;
    using FS = Feed<S, LANES, VEC>;
    using FB = Feed<B, LANES, VEC>;
    using FQ = Feed<uint8_t, LANES, VEC>;
    extern __shared__ __align__(16) char ring[];
    __shared__ TeamScratch scratch;
    Team<B, LANES, BIG> team;
    Columns<LANES, VEC> c;
    int64_t team_id, first_of_warp;
    set_up<LANES, VEC, BIG, B>(p, (int)a.width, &scratch, team, c, team_id, first_of_warp);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const int64_t D = a.width, groups = (D + kPackGroup - 1) / kPackGroup;
    const bool row_gate = BRANCH && (a.gate || a.gate_codes) && !p.shared;

    B scale[4], pw[4], pb[4], nw[4];
    B sum_scale[4] = {}, sum_pw[4] = {}, sum_pb[4] = {}, sum_nw[4] = {}, sum_nb[4] = {}, sum_gate[4] = {};
    B act[4], dact[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        act[e] = B(1);
        dact[e] = B(0);
    }
    if (BRANCH) {
        get_or<B>(a.scale, c, B(1), scale);
        get_or<B>(a.post_weight, c, B(1), pw);
        get_or<B>(a.post_bias, c, B(0), pb);
    }
    if (NEXT) get_or<B>(a.next_weight, c, B(1), nw);

    // a tensor that may be there as codes: codes and the group's scale, or the values themselves
    auto issue_kept = [&](uint32_t at, const void* codes, const void* scales, auto* values, int64_t stride, int64_t row) {
        using T = std::remove_cv_t<std::remove_pointer_t<decltype(values)>>;
        if (codes) {
            FQ::issue(at, static_cast<const uint8_t*>(codes) + row * D, c);
            if (c.col < c.width)
                copy_async<sizeof(B)>(at + blockDim.x * 4 + threadIdx.x * (uint32_t)sizeof(B),
                                      static_cast<const B*>(scales) + row * groups + c.col / kPackGroup);
        } else {
            Feed<T, LANES, VEC>::issue(at, values + row * stride, c);
        }
    };
    auto take_kept = [&](const char* at, const void* codes, auto* values, int64_t stride, int64_t row, B (&v)[4]) {
        using T = std::remove_cv_t<std::remove_pointer_t<decltype(values)>>;
        if (codes) {
            uint8_t q[4];
            FQ::take(at, static_cast<const uint8_t*>(codes) + row * D, c, q);
            const B s = *reinterpret_cast<const B*>(at + blockDim.x * 4 + threadIdx.x * sizeof(B));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = c.ok(e) ? from_code<B>(a.checkpoint, q[e], s) : B(0);
        } else {
            T raw[4];
            Feed<T, LANES, VEC>::take(at, values + row * stride, c, raw);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = widen(raw[e]);
        }
    };
    const S *x = static_cast<const S*>(a.x), *dout = static_cast<const S*>(a.dout);
    const B *y = static_cast<const B*>(a.y), *gate = static_cast<const B*>(a.gate), *dh = static_cast<const B*>(a.dh);

    auto issue = [&](const RowCursor& r, int stage) {
        if (r.active()) {
            const uint32_t at = ring_at + stage * p.stage_bytes;
            if (dout) FS::issue(at + p.at_dout, dout + r.row * a.dout_stride, c);
            if (NEXT) {
                FB::issue(at + p.at_dh, dh + r.row * a.dh_stride, c);
                issue_kept(at + p.at_x, a.x_codes, a.x_scales, x, a.x_stride, r.row);
                copy_async<2 * sizeof(B)>(at + p.at_next_stats + threadIdx.x * 2 * (uint32_t)sizeof(B),
                                          static_cast<const B*>(a.next_stats) + 2 * r.row);
            }
            if (BRANCH) {
                issue_kept(at + p.at_y, a.y_codes, a.y_scales, y, a.y_stride, r.row);
                if (row_gate) issue_kept(at + p.at_gate, a.gate_codes, a.gate_scales, gate, a.gate_stride, r.row);
                if (a.post_norm != kNormNone)
                    copy_async<2 * sizeof(B)>(at + p.at_post_stats + threadIdx.x * 2 * (uint32_t)sizeof(B),
                                              static_cast<const B*>(a.post_stats) + 2 * r.row);
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
    for (int64_t lead = first_of_warp; lead < p.items;) {
        const int into = stage == 0 ? p.stages - 1 : stage - 1;
        issue(ahead, into);
        ahead.next(p);
        copies_wait_oldest(p.stages);
        const bool live = now.active();
        const char* at = ring + stage * p.stage_bytes;
        const int64_t row = now.row;
        B g[4] = {B(0), B(0), B(0), B(0)};
        if (dout && live) {
            S raw[4];
            FS::take(at + p.at_dout, dout + row * a.dout_stride, c, raw);
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = widen(raw[e]);
        }
        if (NEXT) {
            B v[4] = {}, d[4] = {}, st[2] = {};
            if (live) {
                FB::take(at + p.at_dh, dh + row * a.dh_stride, c, d);
                take_kept(at + p.at_x, a.x_codes, x, a.x_stride, row, v);
                const B* stats = reinterpret_cast<const B*>(at + p.at_next_stats + threadIdx.x * 2 * sizeof(B));
                st[0] = stats[0];
                st[1] = stats[1];
            }
            B s[2] = {B(0), B(0)};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = c.ok(e) ? (v[e] - st[0]) * st[1] : B(0);            // the normalised row
                sum_nw[e] += d[e] * v[e];
                sum_nb[e] += d[e];
                d[e] *= nw[e];
                s[0] += d[e];
                s[1] += d[e] * v[e];
            }
            team.template sum<2>(s);
            const B flat = a.next_norm == kNormLayer ? s[0] / B(D) : B(0), along = s[1] / B(D);
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] += st[1] * (d[e] - flat - v[e] * along);
            if (a.dx && live) {
                S o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = narrow<S>(g[e]);
                put<S, LANES, VEC>(static_cast<S*>(a.dx) + row * D, c, o);
            }
        }
        if (BRANCH) {
            if (!NEXT && a.dx && live) {
                S o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = narrow<S>(g[e]);
                put<S, LANES, VEC>(static_cast<S*>(a.dx) + row * D, c, o);
            }
            if (p.shared && live && now.pos == 0) {
                B v[4];
                get_or<B>(gate + row / a.gate_rows * a.gate_stride, c, B(0), v);
#pragma unroll
                for (int e = 0; e < 4; ++e) gate_value_grad<B>(a.gate_act, v[e], act[e], dact[e]);
            }
            B v[4] = {}, dg[4];
            B mean = B(0), rstd = B(1);
            if (live) {
                take_kept(at + p.at_y, a.y_codes, y, a.y_stride, row, v);
                if (a.post_norm != kNormNone) {
                    const B* stats = reinterpret_cast<const B*>(at + p.at_post_stats + threadIdx.x * 2 * sizeof(B));
                    mean = stats[0];
                    rstd = stats[1];
                }
                if (row_gate) {
                    B w[4];
                    take_kept(at + p.at_gate, a.gate_codes, gate, a.gate_stride, row, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) gate_value_grad<B>(a.gate_act, w[e], act[e], dact[e]);
                }
            }
            B s[2] = {B(0), B(0)};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = c.ok(e) ? (v[e] - mean) * rstd : B(0);
                const B z = v[e] * pw[e] + pb[e], ga = g[e] * act[e], gs = g[e] * scale[e];
                sum_scale[e] += ga * z;
                dg[e] = gs * dact[e] * z;
                const B dz = ga * scale[e];
                sum_pw[e] += dz * v[e];
                sum_pb[e] += dz;
                g[e] = dz * pw[e];
                s[0] += g[e];
                s[1] += g[e] * v[e];
            }
            if (p.shared) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sum_gate[e] += dg[e];
            } else if (a.dgate && live) {
                put<B, LANES, VEC>(static_cast<B*>(a.dgate) + row * a.dgate_stride, c, dg);
            }
            if (a.dy) {
                if (a.post_norm != kNormNone) {
                    team.template sum<2>(s);
                    const B flat = a.post_norm == kNormLayer ? s[0] / B(D) : B(0), along = s[1] / B(D);
#pragma unroll
                    for (int e = 0; e < 4; ++e) g[e] = rstd * (g[e] - flat - v[e] * along);
                }
                if (live) put<B, LANES, VEC>(static_cast<B*>(a.dy) + row * a.dy_stride, c, g);
            }
            if (slabs.gate && now.pos + 1 == p.chunk) {
                if (now.item < p.items) put<B, LANES, VEC>(static_cast<B*>(slabs.gate) + now.item * D, c, sum_gate);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum_gate[e] = B(0);
            }
        }
        now.next(p);
        if (now.pos == 0) lead += p.teams;
        stage = stage + 1 == p.stages ? 0 : stage + 1;
    }
    copies_wait<0>();

    // one slab row per block: the teams' sums, added in the order of the teams
    const int64_t block = BIG && p.cluster > 1 ? blockIdx.x / p.cluster : blockIdx.x;
    Quad<B>* shelf = reinterpret_cast<Quad<B>*>(ring);
    const int per_team = blockDim.x / p.teams_per_block;
    auto leave = [&](int which, B (&v)[4]) {
        if (!slabs.column[which]) return;
        B* row = static_cast<B*>(slabs.column[which]) + block * D;
        if (p.teams_per_block > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 4; ++e) shelf[threadIdx.x].v[e] = v[e];
            __syncthreads();
            if ((int)threadIdx.x >= per_team) return;
            for (int i = 1; i < p.teams_per_block; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += shelf[i * per_team + threadIdx.x].v[e];
        }
        put<B, LANES, VEC>(row, c, v);
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
    return a.y ? ring_launch(p, st, ring_forward_kernel<S, LANES, VEC, true, BIG>, a, p)
               : ring_launch(p, st, ring_forward_kernel<S, LANES, VEC, false, BIG>, a, p);
}
template <typename S, int LANES, bool VEC, bool BIG>
cudaError_t ring_backward_as(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st) {
    if (!a.has_branch) return ring_launch(p, st, ring_backward_kernel<S, LANES, VEC, false, true, BIG>, a, p, slabs);
    return a.dh ? ring_launch(p, st, ring_backward_kernel<S, LANES, VEC, true, true, BIG>, a, p, slabs)
                : ring_launch(p, st, ring_backward_kernel<S, LANES, VEC, true, false, BIG>, a, p, slabs);
}

#define KANB200_RING_DISPATCH(name, ...)                                                                    \
    if (p.big) return p.vec ? name<S, 32, true, true>(__VA_ARGS__) : name<S, 32, false, true>(__VA_ARGS__);       \
    if (p.lanes == 32) return p.vec ? name<S, 32, true, false>(__VA_ARGS__) : name<S, 32, false, false>(__VA_ARGS__); \
    if (p.lanes == 16) return p.vec ? name<S, 16, true, false>(__VA_ARGS__) : name<S, 16, false, false>(__VA_ARGS__); \
    return p.vec ? name<S, 8, true, false>(__VA_ARGS__) : name<S, 8, false, false>(__VA_ARGS__)

template <typename S> cudaError_t ring_forward(const kanb200_block_args& a, const RingPlan& p, cudaStream_t st) {
    KANB200_RING_DISPATCH(ring_forward_as, a, p, st);
}
template <typename S>
cudaError_t ring_backward(const kanb200_block_args& a, const RingPlan& p, const BackwardSlabs& slabs, cudaStream_t st) {
    KANB200_RING_DISPATCH(ring_backward_as, a, p, slabs, st);
}
#undef KANB200_RING_DISPATCH

}  // namespace kanb200

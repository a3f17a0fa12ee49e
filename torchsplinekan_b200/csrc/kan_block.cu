// The norm in front of a KAN layer and the gated residual connection behind it, forward and backward.
//
//   forward   [out = x + scale act(gate) post(y)],  h = next(out or x)
//   backward  g = dout + next'(dh),  dx = g,  dz = g scale act(gate),  dy = post'(dz),
//             dgate = g scale act'(gate) z,  and the sums over rows of the five parameters
//   norm'(d)  = r (v - mean(v) - xhat mean(v xhat)),  v = d w        (mean(v) for LAYER only)
//
// One pass over memory is the floor (5 floats per element forward and 8 backward with everything on); bandwidth bounds the
// large calls and latency the small ones.  Rows that fit a team's registers take the kernels of kan_block_ring.cuh; this
// file holds the plan of a call, the kernels for wider rows (a block per row, passes over the row in the caches) and the
// sum of the backward's slabs.
#include "kan_block.cuh"
#include "kan_block_plan.h"

#include <algorithm>
#include <mutex>
#include <new>
#include <set>
#include <utility>

namespace kanb200 {
namespace {

constexpr int kLoopThreads = 256;

template <typename B, int K> __device__ __forceinline__ void warp_sum(B (&v)[K]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}

// Sums of K values over the block, the same bits in every thread (fixed order over the warps).
template <typename B, int K> __device__ __forceinline__ void block_sum(B (&v)[K], B* buf) {
    warp_sum<B, K>(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    __syncthreads();                                        // buf may still be read from the sum before
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) buf[k * 32 + warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        B s = B(0);
        for (int w = 0; w < nw; ++w) s += buf[k * 32 + w];
        v[k] = s;
    }
}

// Calls body(c) for the columns of this thread: a warp owns blocks of 128 columns (the groups of a checkpoint).
template <typename F> __device__ __forceinline__ void for_columns(int64_t width, F body) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    for (int64_t b = warp; b * kPackGroup < width; b += nw)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t c = b * kPackGroup + e * 32 + lane;
            if (c < width) body(c);
        }
}

// Codes and scales of one row; value(c) gives its elements.
template <typename B, typename F>
__device__ __forceinline__ void pack_row(int format, uint8_t* codes, B* scales, int64_t width, F value) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    for (int64_t b = warp; b * kPackGroup < width; b += nw) {
        B v[4];
        typename AbsBits<B>::type top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t c = b * kPackGroup + e * 32 + lane;
            v[e] = c < width ? value(c) : B(0);
            top = max(top, AbsBits<B>::of(v[e]));
        }
        const B scale = pack_scale<B>(format, AbsBits<B>::back(lanes_max<32>(top))), inv = pack_inverse<B>(scale);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t c = b * kPackGroup + e * 32 + lane;
            if (c < width) codes[c] = (uint8_t)to_code(format, v[e], inv);
        }
        if (lane == 0) scales[b] = scale;
    }
}

template <typename B> struct Moments {
    B mean, rstd;
};

// m and r of a row whose elements are value(c): two passes, so that the variance has no cancellation.
template <typename B, typename F>
__device__ __forceinline__ Moments<B> row_moments(int kind, int64_t width, B eps, B* buf, F value) {
    B m = B(0);
    if (kind == kNormLayer) {
        B s[1] = {B(0)};
        for_columns(width, [&](int64_t c) { s[0] += value(c); });
        block_sum<B, 1>(s, buf);
        m = s[0] / B(width);
    }
    B s[1] = {B(0)};
    for_columns(width, [&](int64_t c) {
        const B d = value(c) - m;
        s[0] += d * d;
    });
    block_sum<B, 1>(s, buf);
    return {m, inv_sqrt(s[0] / B(width) + eps)};
}

// ---- rows of any width: a block per row, passes over the row in the caches ------------------------------------------
template <typename S> __global__ void __launch_bounds__(kLoopThreads) loop_forward_kernel(const kanb200_block_args a) {
    using B = Br<S>;
    __shared__ B buf[32];
    const int64_t D = a.width, groups = (D + kPackGroup - 1) / kPackGroup;
    const B eps = B(a.eps);
    const B *scale = static_cast<const B*>(a.scale), *pw = static_cast<const B*>(a.post_weight),
            *pb = static_cast<const B*>(a.post_bias), *nw = static_cast<const B*>(a.next_weight),
            *nb = static_cast<const B*>(a.next_bias);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const S* x = static_cast<const S*>(a.x) + row * a.x_stride;
        if (a.y) {
            const B* y = static_cast<const B*>(a.y) + row * a.y_stride;
            const B* gate = a.gate ? static_cast<const B*>(a.gate) + row / a.gate_rows * a.gate_stride : nullptr;
            S* out = static_cast<S*>(a.out) + row * D;
            Moments<B> p{B(0), B(1)};
            if (a.post_norm != kNormNone) {
                p = row_moments<B>(a.post_norm, D, eps, buf, [&](int64_t c) { return y[c]; });
                if (a.post_stats && threadIdx.x == 0) {
                    static_cast<B*>(a.post_stats)[2 * row] = p.mean;
                    static_cast<B*>(a.post_stats)[2 * row + 1] = p.rstd;
                }
            }
            for_columns(D, [&](int64_t c) {
                B z = (y[c] - p.mean) * p.rstd;
                if (pw) z *= pw[c];
                if (pb) z += pb[c];
                B t = gate ? gate_value<B>(a.gate_act, gate[c]) : B(1);
                if (scale) t *= scale[c];
                out[c] = narrow<S>(widen(x[c]) + t * z);
            });
            if (a.y_codes)
                pack_row<B>(a.checkpoint, static_cast<uint8_t*>(a.y_codes) + row * D,
                            static_cast<B*>(a.y_scales) + row * groups, D, [&](int64_t c) { return y[c]; });
            if (a.gate_codes)
                pack_row<B>(a.checkpoint, static_cast<uint8_t*>(a.gate_codes) + row * D,
                            static_cast<B*>(a.gate_scales) + row * groups, D, [&](int64_t c) { return gate[c]; });
            x = out;                                        // each thread reads back only what it wrote
        }
        if (a.next_norm != kNormNone) {
            const Moments<B> n = row_moments<B>(a.next_norm, D, eps, buf, [&](int64_t c) { return widen(x[c]); });
            if (a.next_stats && threadIdx.x == 0) {
                static_cast<B*>(a.next_stats)[2 * row] = n.mean;
                static_cast<B*>(a.next_stats)[2 * row + 1] = n.rstd;
            }
            B* h = static_cast<B*>(a.h) + row * D;
            for_columns(D, [&](int64_t c) {
                B v = (widen(x[c]) - n.mean) * n.rstd;
                if (nw) v *= nw[c];
                if (nb) v += nb[c];
                h[c] = v;
            });
        }
        if (a.x_codes)
            pack_row<B>(a.checkpoint, static_cast<uint8_t*>(a.x_codes) + row * D,
                        static_cast<B*>(a.x_scales) + row * groups, D, [&](int64_t c) { return widen(x[c]); });
    }
}

template <typename S>
__global__ void __launch_bounds__(kLoopThreads) loop_backward_kernel(const kanb200_block_args a, const RowSplit sp,
                                                                    const BackwardSlabs slabs) {
    using B = Br<S>;
    __shared__ B buf[64];
    const int64_t D = a.width, groups = (D + kPackGroup - 1) / kPackGroup;
    const B *scale = static_cast<const B*>(a.scale), *pw = static_cast<const B*>(a.post_weight),
            *pb = static_cast<const B*>(a.post_bias), *nw = static_cast<const B*>(a.next_weight);
    B* sum[kColumnSums];
#pragma unroll
    for (int k = 0; k < kColumnSums; ++k)
        sum[k] = slabs.column[k] ? static_cast<B*>(slabs.column[k]) + (int64_t)blockIdx.x * D : nullptr;
    for_columns(D, [&](int64_t c) {
#pragma unroll
        for (int k = 0; k < kColumnSums; ++k)
            if (sum[k]) sum[k][c] = B(0);
    });
    const int64_t first = (int64_t)blockIdx.x * sp.rows_per_team;
    const int64_t last = min(first + (int64_t)sp.rows_per_team, a.rows);
    for (int64_t row = first; row < last; ++row) {
        const int64_t span = sp.shared ? row / a.gate_rows : 0, span_first = span * a.gate_rows;
        B* gate_sum = nullptr;                       // where the row's share of a shared gate's gradient adds up
        if (slabs.gate)
            gate_sum = first <= span_first && span_first + a.gate_rows <= last
                           ? static_cast<B*>(a.dgate) + span * a.dgate_stride
                           : static_cast<B*>(slabs.gate) + (blockIdx.x + span) * D;
        const bool opens = row == first || row == span_first;
        const S* dout = a.dout ? static_cast<const S*>(a.dout) + row * a.dout_stride : nullptr;
        const B* dh = a.dh ? static_cast<const B*>(a.dh) + row * a.dh_stride : nullptr;
        B n_mean = B(0), n_rstd = B(0), n_flat = B(0), n_along = B(0);
        auto nhat = [&](int64_t c) {
            const B v = a.x_codes ? from_code<B>(a.checkpoint, static_cast<const uint8_t*>(a.x_codes)[row * D + c],
                                                 static_cast<const B*>(a.x_scales)[row * groups + c / kPackGroup])
                                  : widen(static_cast<const S*>(a.x)[row * a.x_stride + c]);
            return (v - n_mean) * n_rstd;
        };
        if (dh) {
            n_mean = static_cast<const B*>(a.next_stats)[2 * row];
            n_rstd = static_cast<const B*>(a.next_stats)[2 * row + 1];
            B s[2] = {B(0), B(0)};
            for_columns(D, [&](int64_t c) {
                const B v = nw ? dh[c] * nw[c] : dh[c], xh = nhat(c);
                s[0] += v;
                s[1] += v * xh;
                if (sum[kSumNextWeight]) sum[kSumNextWeight][c] += dh[c] * xh;
                if (sum[kSumNextBias]) sum[kSumNextBias][c] += dh[c];
            });
            block_sum<B, 2>(s, buf);
            n_flat = a.next_norm == kNormLayer ? s[0] / B(D) : B(0);
            n_along = s[1] / B(D);
        }
        auto grad = [&](int64_t c) {
            B g = dout ? widen(dout[c]) : B(0);
            if (dh) g += n_rstd * ((nw ? dh[c] * nw[c] : dh[c]) - n_flat - nhat(c) * n_along);
            return g;
        };
        if (a.dx) for_columns(D, [&](int64_t c) { static_cast<S*>(a.dx)[row * D + c] = narrow<S>(grad(c)); });
        if (!a.has_branch) continue;
        B p_mean = B(0), p_rstd = B(1);
        if (a.post_norm != kNormNone) {
            p_mean = static_cast<const B*>(a.post_stats)[2 * row];
            p_rstd = static_cast<const B*>(a.post_stats)[2 * row + 1];
        }
        auto yhat = [&](int64_t c) {
            const B v = a.y_codes ? from_code<B>(a.checkpoint, static_cast<const uint8_t*>(a.y_codes)[row * D + c],
                                                 static_cast<const B*>(a.y_scales)[row * groups + c / kPackGroup])
                                  : static_cast<const B*>(a.y)[row * a.y_stride + c];
            return (v - p_mean) * p_rstd;
        };
        auto gate = [&](int64_t c, B& act, B& dact) {
            act = B(1);
            dact = B(0);
            if (a.gate_codes)
                gate_value_grad<B>(a.gate_act,
                                   from_code<B>(a.checkpoint, static_cast<const uint8_t*>(a.gate_codes)[row * D + c],
                                                static_cast<const B*>(a.gate_scales)[row * groups + c / kPackGroup]),
                                   act, dact);
            else if (a.gate)
                gate_value_grad<B>(a.gate_act,
                                   static_cast<const B*>(a.gate)[row / a.gate_rows * a.gate_stride + c], act, dact);
        };
        B s[2] = {B(0), B(0)};
        for_columns(D, [&](int64_t c) {
            const B g = grad(c), yh = yhat(c);
            B z = pw ? yh * pw[c] : yh, act, dact;
            if (pb) z += pb[c];
            gate(c, act, dact);
            const B gs = scale ? g * scale[c] : g, dz = gs * act;
            if (sum[kSumScale]) sum[kSumScale][c] += g * act * z;
            if (a.dgate && !sp.shared) static_cast<B*>(a.dgate)[row * a.dgate_stride + c] = gs * dact * z;
            if (gate_sum) gate_sum[c] = (opens ? B(0) : gate_sum[c]) + gs * dact * z;
            if (sum[kSumPostWeight]) sum[kSumPostWeight][c] += dz * yh;
            if (sum[kSumPostBias]) sum[kSumPostBias][c] += dz;
            const B u = pw ? dz * pw[c] : dz;
            s[0] += u;
            s[1] += u * yh;
        });
        if (!a.dy) continue;
        B p_flat = B(0), p_along = B(0);
        if (a.post_norm != kNormNone) {
            block_sum<B, 2>(s, buf);
            p_flat = a.post_norm == kNormLayer ? s[0] / B(D) : B(0);
            p_along = s[1] / B(D);
        }
        for_columns(D, [&](int64_t c) {
            B act, dact;
            gate(c, act, dact);
            B u = grad(c) * act;
            if (scale) u *= scale[c];
            if (pw) u *= pw[c];
            static_cast<B*>(a.dy)[row * a.dy_stride + c] =
                a.post_norm != kNormNone ? p_rstd * (u - p_flat - yhat(c) * p_along) : u;
        });
    }
}

// Adds slab rows in a fixed order, 16 interleaved partial sums and then those: the same bits on every run.  A block sums 32
// columns of one result: a parameter's gradient (all slab rows), or a shared gate row's (those of the teams among which
// its rows were divided; one that a single team has is already in place).
struct SlabSums {
    const void* slab[kColumnSums];
    void* dst[kColumnSums];
    int parameters;
    int64_t slab_rows;
    const void* gate_slab;
    void* dgate;
    int64_t dgate_stride, gate_rows, spans, rows_per_team;
};
constexpr int kSumWarps = 16;
template <typename B> __global__ void __launch_bounds__(kSumWarps * 32) sum_slabs_kernel(const SlabSums s, int width) {
    __shared__ B buf[kSumWarps][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const auto reduce = [&](const B* slab, int n, B* dst) {
        B sum = B(0);
        if (c < width) {
            int i = warp;
            const B* at = slab + (int64_t)i * width + c;
            const int64_t next = (int64_t)kSumWarps * width;
            for (; i + 3 * kSumWarps < n; i += 4 * kSumWarps, at += 4 * next) {      // four loads under way
                const B p = at[0], q = at[next], r = at[2 * next], t = at[3 * next];
                sum += (p + q) + (r + t);
            }
            for (; i < n; i += kSumWarps, at += next) sum += *at;
        }
        __syncthreads();
        buf[warp][lane] = sum;
        __syncthreads();
        if (warp == 0 && c < width) {
#pragma unroll
            for (int w = 1; w < kSumWarps; ++w) sum += buf[w][lane];
            dst[c] = sum;
        }
    };
    if ((int)blockIdx.y < s.parameters) {
        reduce(static_cast<const B*>(s.slab[blockIdx.y]), (int)s.slab_rows, static_cast<B*>(s.dst[blockIdx.y]));
        return;
    }
    for (int64_t g = blockIdx.y - s.parameters; g < s.spans; g += gridDim.y - s.parameters) {
        const int64_t from = g * s.gate_rows / s.rows_per_team, to = ((g + 1) * s.gate_rows - 1) / s.rows_per_team;
        if (from != to)
            reduce(static_cast<const B*>(s.gate_slab) + (from + g) * width, (int)(to - from + 1),
                   static_cast<B*>(s.dgate) + g * s.dgate_stride);
    }
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

size_t branch_bytes(int dtype) { return dtype == KANB200_F64 ? 8 : 4; }

RowSplit split_rows(const kanb200_block_args& a, int64_t most_teams) {
    RowSplit s;
    s.shared = a.gate && a.gate_rows > 1;
    s.rows_per_team = (uint32_t)div_up(a.rows, most_teams);
    s.teams = div_up(a.rows, s.rows_per_team);
    return s;
}

constexpr int kLoopBlocks = kSms * 4;

// ---- the ring kernels' plan ---------------------------------------------------------------------------------------------
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Four elements at once everywhere: width and strides multiples of four, pointers aligned to four elements.
bool four_at_once(const kanb200_block_args& a) {
    const size_t s = 4 * (a.dtype == KANB200_F64 ? 4 : a.dtype == KANB200_F32 ? 4 : 2), b = 16;
    for (int64_t n : {a.width, a.x_stride, a.y ? a.y_stride : 0, a.gate ? a.gate_stride : 0, a.dout ? a.dout_stride : 0,
                      a.dh ? a.dh_stride : 0, a.dy ? a.dy_stride : 0, a.dgate ? a.dgate_stride : 0})
        if (n % 4) return false;
    for (const void* p : {a.x, (const void*)a.out, a.dout, (const void*)a.dx})
        if (!aligned(p, s)) return false;
    for (const void* p : {a.y, a.gate, (const void*)a.h, a.dh, (const void*)a.dy, (const void*)a.dgate})
        if (!aligned(p, b)) return false;
    // a parameter may be a view into a flat buffer, anywhere an element may be
    for (const void* p : {a.scale, a.post_weight, a.post_bias, a.next_weight, a.next_bias})
        if (!aligned(p, b)) return false;
    for (const void* p : {a.x_codes, a.y_codes, a.gate_codes})
        if (!aligned(p, 4)) return false;
    return true;
}

// Warps for a row: `warps` in each of `cluster` blocks, of `chunks` chunks per thread.  At most 8 warps make a small block.
struct Team {
    int chunks, warps, cluster;
    bool many, big;
};
Team team_for(const kanb200_block_args& a, bool backward) {
    const bool branch = backward ? a.has_branch : a.y != nullptr, f64 = a.dtype == KANB200_F64;
    Team t{};
    t.many = !branch;
    const auto cover = [&] {
        t.chunks = ring_chunks(t.many, f64);
        t.warps = (int)div_up(a.width, kPackGroup * t.chunks);
    };
    cover();
    if (t.warps > 8 && !backward && !t.many && !f64) {
        t.many = true;
        cover();
    }
    t.big = t.warps > 8 && !f64;
    t.cluster = 1;
    const int all = t.warps, most = ring_threads(t.big) / 32;
    while (div_up(all, t.cluster) > most) t.cluster *= 2;
    t.warps = (int)div_up(all, t.cluster);
    return t;
}
// The ring kernels take rows of up to 8 blocks, and 32-bit row numbers and strides.
bool ring_fits(const kanb200_block_args& a, bool backward) {
    for (int64_t n : {a.rows, a.x_stride, a.y_stride, a.gate_stride, a.dout_stride, a.dh_stride, a.dy_stride, a.dgate_stride})
        if (n >= ((int64_t)1 << 31) - 4096) return false;
    return team_for(a, backward).cluster <= 8;
}

RingPlan plan_ring(const kanb200_block_args& a, bool backward) {
    RingPlan p{};
    const int B = (int)branch_bytes(a.dtype), S = a.dtype == KANB200_F64 ? 8 : a.dtype == KANB200_F32 ? 4 : 2;
    const bool branch = backward ? a.has_branch : a.y != nullptr;
    const Team team = team_for(a, backward);
    const int V = team.chunks;
    p.lanes = 4;
    while (p.lanes < 32 && p.lanes * 4 * V < a.width) p.lanes *= 2;
    p.cluster = team.cluster;
    p.warps = team.warps;
    p.big = team.big;
    p.many = team.many;
    p.teams_per_block = p.big || p.cluster > 1 ? 1 : p.lanes == 32 ? 8 / p.warps : 256 / p.lanes;
    p.threads = p.lanes == 32 ? 32 * p.warps * p.teams_per_block : 256;
    const int T = p.threads;
    const bool vec = four_at_once(a);
    p.mode = !vec ? kScalar : p.lanes * 4 * V * (p.lanes == 32 ? p.warps * p.cluster : 1) == a.width ? kFull : kVector;

    // a stage of the ring: BackwardStage, or x, y and a gate per row
    const int most = ring_threads(p.big);
    const bool row_gate = branch && (a.gate || a.gate_codes) && !(a.gate && a.gate_rows > 1);
    if (backward) {
        const auto take = [&](bool there, int bytes) { p.stage_bytes += there ? bytes : 0; };
        take(a.dh, ring_bytes(B, vec, V, most) + ring_kept_bytes(S, vec, V, most, B) + ring_stats_bytes(most, B));
        take(branch, ring_kept_bytes(B, vec, V, most, B) + ring_stats_bytes(most, B));
        take(a.dout || row_gate, ring_bytes(S, vec, V, most));
        take(row_gate, ring_kept_bytes(B, vec, V, most, B));
    } else {
        p.stage_bytes = ring_bytes(S, vec, V, most) + (branch ? ring_bytes(B, vec, V, most) : 0) +
                        (row_gate ? ring_bytes(B, vec, V, most) : 0);
    }
    p.stage_bytes = std::max(p.stage_bytes, 4 * B * most);      // the blocks' column sums meet in the ring at the end

    // the backward's copies of next_weight, post_weight and scale
    p.parameter_bytes = backward ? ((a.dh ? 1 : 0) + (branch ? 2 : 0)) * (p.threads / p.teams_per_block) * 4 * V * B : 0;

    // blocks to an SM by registers (the kernels' launch bounds) and shared memory, then up to four stages while there is room
    const int registers = 65536 / (ring_threads(p.big) * ring_blocks(p.big, B == 8));
    int per_sm = std::max(1, 65536 / (registers * T));
    const auto fits = [&](int stages) { return stages * p.stage_bytes + p.parameter_bytes <= 228 * 1024 / per_sm - 228 * 1024 + kSharedBytes; };
    while (per_sm > 1 && !fits(2)) --per_sm;
    // Stages: two, more only where two leave less than 40 KB (a norm alone: 32) on their way to an SM.  Deeper rings are slower
    // (forward / backward in us, two against four stages: 16384 x 1024 connection 54 / 94 against 61 / 99, 8192 x 2048 53 / 88
    // against 60 / 94), too little as well (10922 x 1536, 36 KB: forward 56 with two, 52 with three).  Parameters read from
    // memory need the rest for L1.
    const int enough = (branch ? 40 : 32) * 1024, moving = (int)((int64_t)p.stage_bytes * T / most) * per_sm;
    p.stages = 2;
    if (backward || !branch || !p.many)
        while (p.stages < 4 && (p.stages - 1) * moving < enough && fits(p.stages + 1)) ++p.stages;
    // A handful of rows: one block leaves the parameters' gradients in place, which saves the launch that adds slabs (6 rows per
    // team take about 8 us, as long as that launch and the two kernels' starts).
    const bool one_block = backward && a.rows <= (int64_t)6 * p.teams_per_block;
    static_cast<RowSplit&>(p) = split_rows(a, one_block ? p.teams_per_block : (int64_t)kSms * per_sm / p.cluster * p.teams_per_block);
    p.blocks = (int)div_up(p.teams, p.teams_per_block) * p.cluster;
    if (!p.shared) {                     // rows in turn: over every team that is launched
        p.teams = (int64_t)p.blocks / p.cluster * p.teams_per_block;
        p.rows_per_team = (uint32_t)div_up(a.rows, p.teams);
    }
    return p;
}

// ---- launches -----------------------------------------------------------------------------------------------------------
void column_outputs(const kanb200_block_args& a, void* (&out)[kColumnSums]) {
    out[kSumScale] = a.dscale;
    out[kSumPostWeight] = a.dpost_weight;
    out[kSumPostBias] = a.dpost_bias;
    out[kSumNextWeight] = a.dnext_weight;
    out[kSumNextBias] = a.dnext_bias;
}

struct BackwardPlan {
    bool use_ring;
    RingPlan ring;
    RowSplit split;
    int slab_rows;
    BackwardSlabs slabs;
    size_t bytes;
};

// Slabs of the column sums first, then those of a shared gate.  A single slab row is the result itself, where the kernel's
// 16-byte stores can reach that.
BackwardPlan plan_backward(const kanb200_block_args& a, void* ws) {
    BackwardPlan p{};
    p.use_ring = ring_fits(a, true);
    if (p.use_ring) {
        p.ring = plan_ring(a, true);
        p.split = p.ring;
        p.slab_rows = p.ring.blocks / p.ring.cluster;
    } else {
        p.split = split_rows(a, kLoopBlocks);
        p.slab_rows = (int)p.split.teams;
    }
    const size_t row = (size_t)a.width * branch_bytes(a.dtype);
    const auto take = [&](size_t bytes) {
        void* at = static_cast<char*>(ws) + p.bytes;
        p.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    void* outs[kColumnSums];
    column_outputs(a, outs);
    for (int k = 0; k < kColumnSums; ++k)
        p.slabs.column[k] = !outs[k] ? nullptr : p.slab_rows == 1 && aligned(outs[k], 16) ? outs[k] : take(row * p.slab_rows);
    if (a.dgate && p.split.shared) p.slabs.gate = take(row * (p.split.teams + a.rows / a.gate_rows));
    return p;
}

template <typename S> cudaError_t launch_forward(const kanb200_block_args& a, cudaStream_t st) {
    if (ring_fits(a, false)) return ring_forward<S>(a, plan_ring(a, false), st);
    const int blocks = (int)std::min<int64_t>(a.rows, kLoopBlocks * 2);
    loop_forward_kernel<S><<<blocks, kLoopThreads, 0, st>>>(a);
    return cudaGetLastError();
}

template <typename S>
cudaError_t launch_backward(const kanb200_block_args& a, const BackwardPlan& p, cudaStream_t st) {
    using B = Br<S>;
    cudaError_t e;
    if (p.use_ring) {
        e = ring_backward<S>(a, p.ring, p.slabs, st);
    } else {
        loop_backward_kernel<S><<<p.slab_rows, kLoopThreads, 0, st>>>(a, p.split, p.slabs);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
    void* outs[kColumnSums];
    column_outputs(a, outs);
    SlabSums sums{};
    for (int k = 0; k < kColumnSums; ++k)
        if (outs[k] && p.slabs.column[k] != outs[k]) {
            sums.slab[sums.parameters] = p.slabs.column[k];
            sums.dst[sums.parameters++] = outs[k];
        }
    sums.slab_rows = p.slab_rows;
    int64_t spans = 0;
    if (p.slabs.gate && a.rows > p.split.rows_per_team && p.split.rows_per_team % a.gate_rows != 0) {
        sums.gate_slab = p.slabs.gate;
        sums.dgate = a.dgate;
        sums.dgate_stride = a.dgate_stride;
        sums.gate_rows = a.gate_rows;
        sums.rows_per_team = p.split.rows_per_team;
        sums.spans = spans = a.rows / a.gate_rows;
    }
    if (sums.parameters + spans > 0) {
        const dim3 grid((unsigned)div_up(a.width, 32), (unsigned)(sums.parameters + std::min<int64_t>(spans, 4096)));
        sum_slabs_kernel<B><<<grid, kSumWarps * 32, 0, st>>>(sums, (int)a.width);
        e = cudaGetLastError();
    }
    return e;
}

}  // namespace

cudaError_t allow_shared_memory(const void* kernel) {
    static std::mutex mutex;
    static std::set<std::pair<const void*, int>> allowed;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mutex);
    if (allowed.count({kernel, device})) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedBytes);
    try {
        if (e == cudaSuccess) allowed.insert({kernel, device});
    } catch (const std::bad_alloc&) {                        // not remembered, set again by the next call
    }
    return e;
}

int block_columns_at_once(const kanb200_block_args& a, bool backward) {
    return a.rows > 0 && ring_fits(a, backward) && plan_ring(a, backward).mode != kScalar ? 4 : 1;
}

cudaError_t block_forward(const kanb200_block_args& a, cudaStream_t st) {
    switch (a.dtype) {
        case KANB200_F32: return launch_forward<float>(a, st);
        case KANB200_F64: return launch_forward<double>(a, st);
        case KANB200_F16: return launch_forward<__half>(a, st);
        default: return launch_forward<__nv_bfloat16>(a, st);
    }
}

size_t block_backward_workspace(const kanb200_block_args& a) {
    return a.rows < 1 ? 0 : plan_backward(a, nullptr).bytes;
}

cudaError_t block_backward(const kanb200_block_args& a, void* ws, size_t ws_bytes, cudaStream_t st) {
    const BackwardPlan p = plan_backward(a, ws);
    if (p.bytes > ws_bytes) return cudaErrorMemoryAllocation;
    switch (a.dtype) {
        case KANB200_F32: return launch_backward<float>(a, p, st);
        case KANB200_F64: return launch_backward<double>(a, p, st);
        case KANB200_F16: return launch_backward<__half>(a, p, st);
        default: return launch_backward<__nv_bfloat16>(a, p, st);
    }
}

}  // namespace kanb200

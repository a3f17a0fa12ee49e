// 8-bit checkpoints of activations: pack (codes and one scale per 128 columns of a row) and unpack.
//
// Bandwidth bounds both: 4 + 1.03 bytes per float32 element in either direction.  A warp takes kRun groups one after the
// other in the order of (row, group), so that every lane has kRun 16-byte loads under way and forms the scale and its
// reciprocal (a division) of one group only; narrow rows share a warp.  Measured, 65536 x 1024 float32: pack 53 us, unpack
// 50 us (6.4 and 6.7 TB/s; a copy runs at 6.55).
#include "kan_block.cuh"

#include <algorithm>

namespace kanb200 {
namespace {

constexpr int kThreads = 256, kRun = 4;
constexpr int64_t kRowsPerLaunch = (int64_t)1 << 30;        // row numbers are 32-bit in the kernels

// How a run's chunks lie in memory.  kFlat: dense rows of whole groups (or of the one chunk that LANES lanes cover), so the
// chunks follow one another and addresses are one addition.  kRows: row by row, four elements at once.  kSingle: element by
// element.
enum { kFlat, kRows, kSingle };

// A warp's run of kRun chunks.  LANES lanes share a row's group (fewer than 32: rows of up to 4 LANES columns, one group,
// 32 / LANES rows to a chunk).
template <int LANES, int MODE> struct Run {
    int64_t first;                     // kFlat: the run's first group
    int row, rows, group, groups, lane, width, left;

    __device__ __forceinline__ Run(int rows_, int width_) : rows(rows_), width(width_) {
        const int64_t warp = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
        lane = threadIdx.x & (LANES - 1);
        groups = LANES == 32 ? (width + kPackGroup - 1) / kPackGroup : 1;
        row = group = left = 0;
        first = warp * kRun * (32 / LANES) + (threadIdx.x & 31) / LANES;
        if (MODE == kFlat) {
            const int64_t after = (int64_t)rows * groups - first;
            left = (int)min(after, (int64_t)kRun * (32 / LANES));
        } else if (LANES == 32) {
            row = (int)(first >> 32 ? first / groups : (uint32_t)first / (uint32_t)groups);
            group = (int)(first - (int64_t)row * groups);
        } else {
            row = (int)first;
        }
    }
    __device__ __forceinline__ void next() {
        if (MODE == kFlat) return;
        if (LANES < 32) {
            row += 32 / LANES;
        } else if (++group == groups) {
            group = 0;
            ++row;
        }
    }
    // the run's i-th chunk
    __device__ __forceinline__ bool there(int i) const { return MODE == kFlat ? i * (32 / LANES) < left : row < rows; }
    __device__ __forceinline__ int column(int e) const { return group * kPackGroup + (MODE == kSingle ? lane + LANES * e : 4 * lane + e); }
    __device__ __forceinline__ bool ok(int i, int e) const {
        return there(i) && (MODE == kFlat || column(MODE == kSingle ? e : 0) < width);
    }
    template <typename T> __device__ __forceinline__ T* at(T* base, int64_t stride, int i) const {
        if (MODE == kFlat) return base + first * (4 * LANES) + 4 * lane + i * (32 / LANES) * (4 * LANES);
        return base + (int64_t)row * stride + column(0);
    }
    template <typename T> __device__ __forceinline__ T* scale_at(T* base, int i) const {
        if (MODE == kFlat) return base + first + i * (32 / LANES);
        return base + (int64_t)row * groups + group;
    }
};

template <typename S, int LANES, int MODE>
__global__ void __launch_bounds__(kThreads) pack_kernel(int format, const S* __restrict__ x, int64_t x_stride,
                                                       uint8_t* __restrict__ codes, Br<S>* __restrict__ scales,
                                                       int rows, int width) {
    using B = Br<S>;
    using Bits = typename AbsBits<B>::type;
    const Run<LANES, MODE> start(rows, width);
    Four<B> v[kRun];
    {
        Run<LANES, MODE> r = start;
#pragma unroll
        for (int i = 0; i < kRun; ++i, r.next()) {
            Quad<S> q{};
            const S* at = r.at(x, x_stride, i);
            if constexpr (MODE != kSingle) {
                if (r.ok(i, 0)) q = load_quad(at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r.ok(i, e)) q.v[e] = at[LANES * e];
            }
            v[i] = widen4<S>(q);
        }
    }
    Run<LANES, MODE> r = start;
    Bits mine = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const Bits top = lanes_max<LANES>(AbsBits<B>::of(max_abs(B(0), v[i])));
        if (r.lane % kRun == i) mine = top;
    }
    const B scale = pack_scale<B>(format, AbsBits<B>::back(mine)), inverse = pack_inverse<B>(scale);
#pragma unroll
    for (int i = 0; i < kRun; ++i, r.next()) {
        const B inv = __shfl_sync(0xffffffffu, inverse, i, LANES);
        if (r.lane == i && r.there(i)) *r.scale_at(scales, i) = scale;
        const uint32_t word = encode4(format, v[i], inv);
        uint8_t* at = r.at(codes, width, i);
        if constexpr (MODE != kSingle) {
            if (r.ok(i, 0)) *reinterpret_cast<uint32_t*>(at) = word;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r.ok(i, e)) at[LANES * e] = (uint8_t)(word >> 8 * e);
        }
    }
}

template <typename S, int LANES, int MODE>
__global__ void __launch_bounds__(kThreads) unpack_kernel(int format, const uint8_t* __restrict__ codes,
                                                         const Br<S>* __restrict__ scales, S* __restrict__ x, int rows,
                                                         int width) {
    using B = Br<S>;
    const Run<LANES, MODE> start(rows, width);
    uint32_t word[kRun];
    B scale[kRun];
    {
        Run<LANES, MODE> r = start;
#pragma unroll
        for (int i = 0; i < kRun; ++i, r.next()) {
            const uint8_t* at = r.at(codes, width, i);
            word[i] = 0;
            if constexpr (MODE != kSingle) {
                if (r.ok(i, 0)) word[i] = *reinterpret_cast<const uint32_t*>(at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r.ok(i, e)) word[i] |= (uint32_t)at[LANES * e] << 8 * e;
            }
            scale[i] = r.there(i) ? *r.scale_at(scales, i) : B(0);
        }
    }
    Run<LANES, MODE> r = start;
#pragma unroll
    for (int i = 0; i < kRun; ++i, r.next()) {
        const Quad<S> q = narrow4<S>(decode4<B>(format, word[i], scale[i]));
        S* at = r.at(x, width, i);
        if constexpr (MODE != kSingle) {
            if (r.ok(i, 0)) store_quad(at, q);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r.ok(i, e)) at[LANES * e] = q.v[e];
        }
    }
}

struct Shape {
    int lanes, mode;
    unsigned blocks;
};
// false: more blocks than a grid can have
bool shape_of(int64_t rows, int64_t width, bool dense, bool vec, Shape& s) {
    s.lanes = width <= 16 ? 4 : width <= 32 ? 8 : width <= 64 ? 16 : 32;
    s.mode = !vec || width % 4 ? kSingle : dense && (s.lanes == 32 ? width % kPackGroup == 0 : width == 4 * s.lanes) ? kFlat : kRows;
    const int64_t chunks = s.lanes == 32 ? rows * ((width + kPackGroup - 1) / kPackGroup) : (rows * s.lanes + 31) / 32;
    const int64_t blocks = (chunks + kRun * (kThreads / 32) - 1) / (kRun * (kThreads / 32));
    s.blocks = (unsigned)blocks;
    return blocks < ((int64_t)1 << 31);
}
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
template <typename S> constexpr size_t quad_alignment() { return 4 * sizeof(S) > 16 ? 16 : 4 * sizeof(S); }

// body(LANES, MODE) as constants, for a shape
template <typename F> void with_shape(const Shape& s, F body) {
    const auto lanes = [&](auto l) {
        if (s.mode == kFlat) body(l, std::integral_constant<int, kFlat>{});
        else if (s.mode == kRows) body(l, std::integral_constant<int, kRows>{});
        else body(l, std::integral_constant<int, kSingle>{});
    };
    switch (s.lanes) {
        case 4: return lanes(std::integral_constant<int, 4>{});
        case 8: return lanes(std::integral_constant<int, 8>{});
        case 16: return lanes(std::integral_constant<int, 16>{});
        default: return lanes(std::integral_constant<int, 32>{});
    }
}

template <typename S>
cudaError_t pack(int format, const void* x, int64_t x_stride, void* codes, void* scales, int64_t rows, int64_t width,
                 cudaStream_t st) {
    const int64_t groups = (width + kPackGroup - 1) / kPackGroup;
    const bool vec = x_stride % 4 == 0 && aligned(x, quad_alignment<S>()) && aligned(codes, 4);
    for (int64_t r = 0; r < rows; r += kRowsPerLaunch) {
        const int64_t n = std::min(rows - r, kRowsPerLaunch);
        Shape s;
        if (!shape_of(n, width, x_stride == width, vec, s)) return cudaErrorInvalidValue;
        with_shape(s, [&](auto lanes, auto mode) {
            pack_kernel<S, lanes, mode><<<s.blocks, kThreads, 0, st>>>(
                format, static_cast<const S*>(x) + r * x_stride, x_stride, static_cast<uint8_t*>(codes) + r * width,
                static_cast<Br<S>*>(scales) + r * groups, (int)n, (int)width);
        });
    }
    return cudaGetLastError();
}

template <typename S>
cudaError_t unpack(int format, const void* codes, const void* scales, void* x, int64_t rows, int64_t width,
                   cudaStream_t st) {
    const int64_t groups = (width + kPackGroup - 1) / kPackGroup;
    const bool vec = aligned(x, quad_alignment<S>()) && aligned(codes, 4);
    for (int64_t r = 0; r < rows; r += kRowsPerLaunch) {
        const int64_t n = std::min(rows - r, kRowsPerLaunch);
        Shape s;
        if (!shape_of(n, width, true, vec, s)) return cudaErrorInvalidValue;
        with_shape(s, [&](auto lanes, auto mode) {
            unpack_kernel<S, lanes, mode><<<s.blocks, kThreads, 0, st>>>(
                format, static_cast<const uint8_t*>(codes) + r * width, static_cast<const Br<S>*>(scales) + r * groups,
                static_cast<S*>(x) + r * width, (int)n, (int)width);
        });
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t pack_activation(int dtype, int format, const void* x, int64_t x_stride, void* codes, void* scales,
                            int64_t rows, int64_t width, cudaStream_t st) {
    switch (dtype) {
        case KANB200_F32: return pack<float>(format, x, x_stride, codes, scales, rows, width, st);
        case KANB200_F64: return pack<double>(format, x, x_stride, codes, scales, rows, width, st);
        case KANB200_F16: return pack<__half>(format, x, x_stride, codes, scales, rows, width, st);
        default: return pack<__nv_bfloat16>(format, x, x_stride, codes, scales, rows, width, st);
    }
}

cudaError_t unpack_activation(int dtype, int format, const void* codes, const void* scales, void* x, int64_t rows,
                              int64_t width, cudaStream_t st) {
    switch (dtype) {
        case KANB200_F32: return unpack<float>(format, codes, scales, x, rows, width, st);
        case KANB200_F64: return unpack<double>(format, codes, scales, x, rows, width, st);
        case KANB200_F16: return unpack<__half>(format, codes, scales, x, rows, width, st);
        default: return unpack<__nv_bfloat16>(format, codes, scales, x, rows, width, st);
    }
}

}  // namespace kanb200

// 8-bit checkpoints of activations: pack (codes and one scale per 128 columns of a row) and unpack.
//
// Bandwidth bounds both: 4 + 1.03 bytes per float32 element in either direction.  A warp takes kRun groups one after the
// other in the order of (row, group), so that every lane has kRun 16-byte loads under way and forms the scale and its
// reciprocal (a division) of one group only; narrow rows share a warp.
#include "kan_block.cuh"

#include <algorithm>

namespace kanb200 {
namespace {

constexpr int kThreads = 256, kRun = 4;

// Where a run of kRun chunks lies.  LANES lanes share a row's group (fewer than 32: rows of up to 4 LANES columns, one
// group, 32 / LANES rows to a chunk).
template <int LANES, bool VEC> struct Run {
    int64_t row, rows;
    int group, groups, lane, width;

    __device__ __forceinline__ Run(int64_t rows_, int width_) : rows(rows_), width(width_) {
        const int64_t warp = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
        lane = threadIdx.x & (LANES - 1);
        if (LANES == 32) {
            groups = (width + kPackGroup - 1) / kPackGroup;
            const int64_t first = warp * kRun;
            row = first >> 32 ? first / groups : (uint32_t)first / (uint32_t)groups;
            group = (int)(first - row * groups);
        } else {
            groups = 1;
            group = 0;
            row = warp * kRun * (32 / LANES) + (threadIdx.x & 31) / LANES;
        }
    }
    __device__ __forceinline__ void next() {
        if (LANES < 32) {
            row += 32 / LANES;
        } else if (++group == groups) {
            group = 0;
            ++row;
        }
    }
    __device__ __forceinline__ int column(int e) const { return group * kPackGroup + (VEC ? 4 * lane + e : lane + LANES * e); }
    __device__ __forceinline__ bool ok(int e) const { return row < rows && column(VEC ? 0 : e) < width; }
    __device__ __forceinline__ int64_t scale_at() const { return row * groups + group; }
};

template <typename S, int LANES, bool VEC>
__global__ void __launch_bounds__(kThreads, sizeof(S) == 8 ? 3 : 6) pack_kernel(int format, const S* __restrict__ x, int64_t x_stride,
                                                       uint8_t* __restrict__ codes, Br<S>* __restrict__ scales,
                                                       int64_t rows, int width) {
    using B = Br<S>;
    using Bits = typename AbsBits<B>::type;
    Four<B> v[kRun];
    const Run<LANES, VEC> start(rows, width);
    {
        Run<LANES, VEC> r = start;
#pragma unroll
        for (int i = 0; i < kRun; ++i, r.next()) {
            Quad<S> q{};
            if constexpr (VEC) {
                if (r.ok(0)) q = load_quad(x + r.row * x_stride + r.column(0));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r.ok(e)) q.v[e] = x[r.row * x_stride + r.column(e)];
            }
            v[i] = widen4<S>(q);
        }
    }
    Run<LANES, VEC> r = start;
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
        if (r.lane == i && r.row < rows) scales[r.scale_at()] = scale;
        const uint32_t word = encode4(format, v[i], inv);
        uint8_t* at = codes + r.row * width + r.column(0);
        if constexpr (VEC) {
            if (r.ok(0)) *reinterpret_cast<uint32_t*>(at) = word;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r.ok(e)) at[LANES * e] = (uint8_t)(word >> 8 * e);
        }
    }
}

template <typename S, int LANES, bool VEC>
__global__ void __launch_bounds__(kThreads) unpack_kernel(int format, const uint8_t* __restrict__ codes,
                                                         const Br<S>* __restrict__ scales, S* __restrict__ x,
                                                         int64_t rows, int width) {
    using B = Br<S>;
    uint32_t word[kRun];
    B scale[kRun];
    const Run<LANES, VEC> start(rows, width);
    {
        Run<LANES, VEC> r = start;
#pragma unroll
        for (int i = 0; i < kRun; ++i, r.next()) {
            const uint8_t* at = codes + r.row * width + r.column(0);
            word[i] = 0;
            if constexpr (VEC) {
                if (r.ok(0)) word[i] = *reinterpret_cast<const uint32_t*>(at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r.ok(e)) word[i] |= (uint32_t)at[LANES * e] << 8 * e;
            }
            scale[i] = r.row < rows ? scales[r.scale_at()] : B(0);
        }
    }
    Run<LANES, VEC> r = start;
#pragma unroll
    for (int i = 0; i < kRun; ++i, r.next()) {
        const Quad<S> q = narrow4<S>(decode4<B>(format, word[i], scale[i]));
        S* at = x + r.row * width + r.column(0);
        if constexpr (VEC) {
            if (r.ok(0)) store_quad(at, q);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r.ok(e)) at[LANES * e] = q.v[e];
        }
    }
}

struct Shape {
    int lanes;
    bool vec;
    unsigned blocks;
};
// false: more blocks than a grid can have
bool shape_of(int64_t rows, int64_t width, bool vec, Shape& s) {
    s.lanes = width <= 16 ? 4 : width <= 32 ? 8 : width <= 64 ? 16 : 32;
    s.vec = vec && width % 4 == 0;
    const int64_t chunks = s.lanes == 32 ? rows * ((width + kPackGroup - 1) / kPackGroup) : (rows * s.lanes + 31) / 32;
    const int64_t blocks = (chunks + kRun * (kThreads / 32) - 1) / (kRun * (kThreads / 32));
    s.blocks = (unsigned)blocks;
    return blocks < ((int64_t)1 << 31);
}
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
template <typename S> constexpr size_t quad_alignment() { return 4 * sizeof(S) > 16 ? 16 : 4 * sizeof(S); }

// body.template operator()<LANES, VEC>() for a shape
template <typename F> void with_shape(const Shape& s, F body) {
    const auto lanes = [&](auto l) {
        if (s.vec) body(l, std::true_type{});
        else body(l, std::false_type{});
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
    Shape s;
    if (!shape_of(rows, width, x_stride % 4 == 0 && aligned(x, quad_alignment<S>()) && aligned(codes, 4), s))
        return cudaErrorInvalidValue;
    with_shape(s, [&](auto lanes, auto vec) {
        pack_kernel<S, lanes, vec><<<s.blocks, kThreads, 0, st>>>(format, static_cast<const S*>(x), x_stride,
                                                                  static_cast<uint8_t*>(codes), static_cast<Br<S>*>(scales),
                                                                  rows, (int)width);
    });
    return cudaGetLastError();
}

template <typename S>
cudaError_t unpack(int format, const void* codes, const void* scales, void* x, int64_t rows, int64_t width,
                   cudaStream_t st) {
    Shape s;
    if (!shape_of(rows, width, aligned(x, quad_alignment<S>()) && aligned(codes, 4), s)) return cudaErrorInvalidValue;
    with_shape(s, [&](auto lanes, auto vec) {
        unpack_kernel<S, lanes, vec><<<s.blocks, kThreads, 0, st>>>(format, static_cast<const uint8_t*>(codes),
                                                                    static_cast<const Br<S>*>(scales), static_cast<S*>(x),
                                                                    rows, (int)width);
    });
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

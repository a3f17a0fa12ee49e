// 8-bit checkpoints of activations: pack (codes and one scale per 128 columns of a row) and unpack.
// Bandwidth bounds both: 4 + 1.03 bytes per float32 element in either direction.
#include "kan_block.cuh"

#include <algorithm>

namespace kanb200 {
namespace {

constexpr int kThreads = 256;

// A warp per group of 128 columns.
template <typename S>
__global__ void __launch_bounds__(kThreads) pack_kernel(int format, const S* __restrict__ x, int64_t x_stride,
                                                       uint8_t* __restrict__ codes, Br<S>* __restrict__ scales,
                                                       int64_t rows, int64_t width) {
    using B = Br<S>;
    const int lane = threadIdx.x & 31;
    const int64_t groups = (width + kPackGroup - 1) / kPackGroup, total = rows * groups;
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < total;
         i += (int64_t)gridDim.x * (kThreads / 32)) {
        const int64_t row = i / groups, first = (i - row * groups) * kPackGroup;
        B v[4];
        typename AbsBits<B>::type top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t c = first + e * 32 + lane;
            v[e] = c < width ? widen(x[row * x_stride + c]) : B(0);
            top = max(top, AbsBits<B>::of(v[e]));
        }
        const B scale = pack_scale<B>(format, AbsBits<B>::back(lanes_max<32>(top))), inv = pack_inverse<B>(scale);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t c = first + e * 32 + lane;
            if (c < width) codes[row * width + c] = (uint8_t)to_code(format, v[e], inv);
        }
        if (lane == 0) scales[i] = scale;
    }
}

template <typename S>
__global__ void __launch_bounds__(kThreads) unpack_kernel(int format, const uint8_t* __restrict__ codes,
                                                         const Br<S>* __restrict__ scales, S* __restrict__ x,
                                                         int64_t rows, int64_t width) {
    using B = Br<S>;
    const int lane = threadIdx.x & 31;
    const int64_t groups = (width + kPackGroup - 1) / kPackGroup, total = rows * groups;
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < total;
         i += (int64_t)gridDim.x * (kThreads / 32)) {
        const int64_t row = i / groups, first = (i - row * groups) * kPackGroup;
        const B scale = scales[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t c = first + e * 32 + lane;
            if (c < width) x[row * width + c] = narrow<S>(from_code<B>(format, codes[row * width + c], scale));
        }
    }
}

int grid_for(int64_t rows, int64_t width) {
    const int64_t warps = rows * ((width + kPackGroup - 1) / kPackGroup);
    return (int)std::min<int64_t>((warps + kThreads / 32 - 1) / (kThreads / 32), 148 * 64);
}

template <typename S>
cudaError_t pack(int format, const void* x, int64_t x_stride, void* codes, void* scales, int64_t rows, int64_t width,
                 cudaStream_t st) {
    pack_kernel<S><<<grid_for(rows, width), kThreads, 0, st>>>(format, static_cast<const S*>(x), x_stride,
                                                               static_cast<uint8_t*>(codes), static_cast<Br<S>*>(scales),
                                                               rows, width);
    return cudaGetLastError();
}

template <typename S>
cudaError_t unpack(int format, const void* codes, const void* scales, void* x, int64_t rows, int64_t width,
                   cudaStream_t st) {
    unpack_kernel<S><<<grid_for(rows, width), kThreads, 0, st>>>(format, static_cast<const uint8_t*>(codes),
                                                                 static_cast<const Br<S>*>(scales), static_cast<S*>(x),
                                                                 rows, width);
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

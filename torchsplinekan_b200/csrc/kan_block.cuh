// Building blocks of the kernels around a KAN layer (kan_block.cu, kan_pack.cu): element types, sums over the
// threads that share a row, gate activations, and the 8-bit codes of a checkpoint.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kan_block.h"
#include "kan_device.cuh"

namespace kanb200 {

// ---- element types ------------------------------------------------------------------------------------------------
// S: the stream (x, out and their gradients).  Br<S>: the side the layers compute on (y, gate, h, parameters and
// their gradients) and the type of all arithmetic: float64 next to a float64 stream, float32 otherwise.
template <typename S> struct BranchOf { using type = float; };
template <> struct BranchOf<double> { using type = double; };
template <typename S> using Br = typename BranchOf<S>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <typename S> __device__ __forceinline__ S narrow(Br<S> v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ double narrow<double>(double v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float exp2f_approx(float v) {
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float reciprocal_approx(float v) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// 1 / (1 + exp(-x)).  Float: 1 / (1 + 2^t), t = -x log2(e), with the hardware's 2^t (2 ulp) and reciprocal (1 ulp).
// Rounding t moves 2^t by up to |x| 2^-24 of it, so the relative error stays below (1.3 |x| + 6) 2^-24; the ends are 0 and
// 1, NaN stays NaN.  The library's exp and division take three times the instructions, and issue slots bound the gated
// kernels.
__device__ __forceinline__ float gate_sigmoid(float x) { return reciprocal_approx(1.0f + exp2f_approx(x * -1.44269504f)); }
__device__ __forceinline__ double gate_sigmoid(double x) { return sigmoid_t<double>(x); }

// ---- gate activations ---------------------------------------------------------------------------------------------
template <typename B> __device__ __forceinline__ B gate_value(int act, B g) {
    if (act == kActNone) return g;
    const B s = gate_sigmoid(g);
    return act == kActSigmoid ? s : g * s;
}
template <typename B> __device__ __forceinline__ void gate_value_grad(int act, B g, B& a, B& da) {
    if (act == kActNone) {
        a = g;
        da = B(1);
        return;
    }
    const B s = gate_sigmoid(g);
    if (act == kActSigmoid) {
        a = s;
        da = s * (B(1) - s);
    } else {
        a = g * s;
        da = s * (B(1) + g * (B(1) - s));
    }
}

__device__ __forceinline__ float inv_sqrt(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

// ---- 8-bit codes ----------------------------------------------------------------------------------------------------
// A group is kPackGroup consecutive columns of one row.  With A = max |x| over the group
//     scale = max(A * (1 / top), smallest normal),   code = round(x * (1 / scale)),   x~ = code * scale
// (top = 127 for int8, 448 for e4m3).  The lower bound on the scale keeps its reciprocal finite, so an all-zero or
// subnormal group needs no case of its own.  A NaN or infinity in the group makes the scale NaN or infinite; the codes
// are then 0 and every x~ of the group is 0 * scale = NaN: an overflow stays visible instead of being clipped.
// |x| as an unsigned integer orders like |x| with NaN on top, so one integer maximum finds A and keeps NaN.
template <typename B> struct AbsBits;
template <> struct AbsBits<float> {
    using type = uint32_t;
    static __device__ __forceinline__ uint32_t of(float v) { return __float_as_uint(v) & 0x7fffffffu; }
    static __device__ __forceinline__ float back(uint32_t b) { return __uint_as_float(b); }
};
template <> struct AbsBits<double> {
    using type = unsigned long long;
    static __device__ __forceinline__ unsigned long long of(double v) {
        return (unsigned long long)__double_as_longlong(v) & 0x7fffffffffffffffull;
    }
    static __device__ __forceinline__ double back(unsigned long long b) { return __longlong_as_double((long long)b); }
};
// maximum over the W lanes (a power of two, aligned) that share a group
template <int W> __device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    if constexpr (W == 32) {
        return __reduce_max_sync(0xffffffffu, v);
    } else {
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
}
template <int W> __device__ __forceinline__ unsigned long long lanes_max(unsigned long long v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
        v = u > v ? u : v;
    }
    return v;
}

__device__ __forceinline__ float smallest_normal(float) { return 1.17549435e-38f; }
__device__ __forceinline__ double smallest_normal(double) { return 2.2250738585072014e-308; }

template <typename B> __device__ __forceinline__ B pack_scale(int format, B amax) {
    const B by = format == kPackInt8 ? B(1.0 / 127.0) : B(1.0 / 448.0);
    const B s = amax * by;
    return s < smallest_normal(s) ? smallest_normal(s) : s;         // false for NaN: stays NaN
}
// 1 / scale, or 0 for a scale that is not finite (the codes are then 0)
template <typename B> __device__ __forceinline__ B pack_inverse(B scale) {
    return AbsBits<B>::of(scale) < AbsBits<B>::of(B(INFINITY)) ? B(1) / scale : B(0);
}
__device__ __forceinline__ uint32_t to_code(int format, float v, float inv) {
    // inv == 0: the group is not finite, v may be infinite or NaN
    const float q = inv == 0.0f ? 0.0f : v * inv;
    if (format == kPackInt8) return (uint32_t)min(127, max(-127, __float2int_rn(q))) & 0xffu;
    return __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t to_code(int format, double v, double inv) {
    const double q = inv == 0.0 ? 0.0 : v * inv;
    if (format == kPackInt8) return (uint32_t)min(127, max(-127, __double2int_rn(q))) & 0xffu;
    return __nv_cvt_double_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}
template <typename B> __device__ __forceinline__ B from_code(int format, uint32_t code, B scale) {
    if (format == kPackInt8) return B((int)(int8_t)code) * scale;
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3);
    return B(__half2float(__half(h))) * scale;                      // e4m3 fits float16 exactly
}

}  // namespace kanb200

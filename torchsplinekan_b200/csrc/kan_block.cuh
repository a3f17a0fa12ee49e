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
// 0 where the result is below the normal numbers
__device__ __forceinline__ float reciprocal_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// -x within [-88, 88], NaN stays NaN
__device__ __forceinline__ float negated_gate(float x) {
    float r;
    asm("min.NaN.xorsign.abs.f32 %0, %1, 0fc2b00000;" : "=f"(r) : "f"(x));
    return r;
}
// 1 / (1 + exp(-x)).  Float: exp(-x) = 2^t e^r with t the rounded -x log2(e) and r = -x - t ln 2 what its rounding leaves, so
// e^r = 1 + r.  In units of 2^-24, with the hardware's 2^t (4) and reciprocal (2), the product with 1 + r and the sum (1 each)
// the relative error stays below 8 (largest seen 4.7 for x from -87.3 to 40, and 65 with r left out).  The ends are 0 (below
// -87.4, where the value is no normal number) and 1, NaN stays NaN.  The library's exp and division reach 3.4, but take so many
// more instructions that the 8-bit gated training pass of 16384 x 2048 bfloat16 went from 211 us to 258.
constexpr float kLog2E = 1.44269504f, kLn2 = 0.693147182f, kLn2Rest = -1.90465432e-9f;      // ln 2 = kLn2 + kLn2Rest
__device__ __forceinline__ float gate_sigmoid(float x) {
    const float n = negated_gate(x), t = n * kLog2E, r = fmaf(t, -kLn2Rest, fmaf(t, -kLn2, n)), e = exp2f_approx(t);
    return reciprocal_approx(1.0f + fmaf(e, r, e));
}
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

// ---- four elements --------------------------------------------------------------------------------------------------
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

// Four values in the branch's type; float works on pairs (sm_100's two-element FMA pipe instructions).
template <typename B> struct alignas(16) Four {
    B v[4];
};
template <typename B> __device__ __forceinline__ Four<B> four(B s) { return {{s, s, s, s}}; }
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split_pair(unsigned long long p, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
#define KANB200_PAIRWISE(name, instruction)                                                                          \
    __device__ __forceinline__ Four<float> name(const Four<float>& x, const Four<float>& y) {                        \
        Four<float> r;                                                                                               \
        _Pragma("unroll") for (int e = 0; e < 4; e += 2) {                                                           \
            unsigned long long p;                                                                                    \
            asm(instruction " %0, %1, %2;" : "=l"(p) : "l"(pair_of(x.v[e], x.v[e + 1])), "l"(pair_of(y.v[e], y.v[e + 1]))); \
            split_pair(p, r.v[e], r.v[e + 1]);                                                                       \
        }                                                                                                            \
        return r;                                                                                                    \
    }
KANB200_PAIRWISE(operator+, "add.rn.f32x2")
KANB200_PAIRWISE(operator*, "mul.rn.f32x2")
#undef KANB200_PAIRWISE
// x y + z, rounded once
__device__ __forceinline__ Four<float> fma4(const Four<float>& x, const Four<float>& y, const Four<float>& z) {
    Four<float> r;
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
        unsigned long long p;
        asm("fma.rn.f32x2 %0, %1, %2, %3;"
            : "=l"(p)
            : "l"(pair_of(x.v[e], x.v[e + 1])), "l"(pair_of(y.v[e], y.v[e + 1])), "l"(pair_of(z.v[e], z.v[e + 1])));
        split_pair(p, r.v[e], r.v[e + 1]);
    }
    return r;
}
__device__ __forceinline__ Four<double> operator+(const Four<double>& x, const Four<double>& y) {
    return {{x.v[0] + y.v[0], x.v[1] + y.v[1], x.v[2] + y.v[2], x.v[3] + y.v[3]}};
}
__device__ __forceinline__ Four<double> operator*(const Four<double>& x, const Four<double>& y) {
    return {{x.v[0] * y.v[0], x.v[1] * y.v[1], x.v[2] * y.v[2], x.v[3] * y.v[3]}};
}
__device__ __forceinline__ Four<double> fma4(const Four<double>& x, const Four<double>& y, const Four<double>& z) {
    return {{fma(x.v[0], y.v[0], z.v[0]), fma(x.v[1], y.v[1], z.v[1]), fma(x.v[2], y.v[2], z.v[2]), fma(x.v[3], y.v[3], z.v[3])}};
}
// max(top, |x|), NaN if any is
__device__ __forceinline__ float max_abs(float top, const Four<float>& x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(fabsf(x.v[e])));
    return top;
}
__device__ __forceinline__ double max_abs(double top, const Four<double>& x) {
    unsigned long long t = AbsBits<double>::of(top);         // |x| as an integer orders like |x| with NaN on top
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned long long v = AbsBits<double>::of(x.v[e]);
        t = v > t ? v : t;
    }
    return AbsBits<double>::back(t);
}
template <typename B> __device__ __forceinline__ B total(const Four<B>& x) { return (x.v[0] + x.v[2]) + (x.v[1] + x.v[3]); }

template <typename S> __device__ __forceinline__ Four<Br<S>> widen4(const Quad<S>& q) {
    return {{widen(q.v[0]), widen(q.v[1]), widen(q.v[2]), widen(q.v[3])}};
}
template <typename S> __device__ __forceinline__ Quad<S> narrow4(const Four<Br<S>>& x) {
    Quad<S> q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = narrow<S>(x.v[e]);
    return q;
}
template <> __device__ __forceinline__ Quad<__nv_bfloat16> narrow4<__nv_bfloat16>(const Four<float>& x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.v[0], x.v[1]), b = __floats2bfloat162_rn(x.v[2], x.v[3]);
    return {{a.x, a.y, b.x, b.y}};
}
template <> __device__ __forceinline__ Quad<__half> narrow4<__half>(const Four<float>& x) {
    const __half2 a = __floats2half2_rn(x.v[0], x.v[1]), b = __floats2half2_rn(x.v[2], x.v[3]);
    return {{a.x, a.y, b.x, b.y}};
}

// gate_sigmoid of four
__device__ __forceinline__ Four<float> sigmoid4(const Four<float>& g) {
    Four<float> n, e;
#pragma unroll
    for (int k = 0; k < 4; ++k) n.v[k] = negated_gate(g.v[k]);
    const Four<float> t = n * four<float>(kLog2E);
    const Four<float> r = fma4(t, four<float>(-kLn2Rest), fma4(t, four<float>(-kLn2), n));
#pragma unroll
    for (int k = 0; k < 4; ++k) e.v[k] = exp2f_approx(t.v[k]);
    e = fma4(e, r, e) + four<float>(1.0f);
#pragma unroll
    for (int k = 0; k < 4; ++k) e.v[k] = reciprocal_approx(e.v[k]);
    return e;
}
__device__ __forceinline__ Four<double> sigmoid4(const Four<double>& g) {
    return {{gate_sigmoid(g.v[0]), gate_sigmoid(g.v[1]), gate_sigmoid(g.v[2]), gate_sigmoid(g.v[3])}};
}
template <typename B> __device__ __forceinline__ Four<B> gate4(int act, const Four<B>& g) {
    if (act == kActNone) return g;
    const Four<B> s = sigmoid4(g);
    return act == kActSigmoid ? s : g * s;
}
// activation and derivative: sigmoid s, s (1 - s);  silu g s, s + g s (1 - s)
template <typename B> __device__ __forceinline__ void gate4_grad(int act, const Four<B>& g, Four<B>& a, Four<B>& da) {
    a = g;
    da = four<B>(B(1));
    if (act == kActNone) return;
    const Four<B> s = sigmoid4(g), rest = fma4(s, four<B>(B(-1)), four<B>(B(1)));
    a = act == kActSigmoid ? s : g * s;
    da = act == kActSigmoid ? s * rest : fma4(a, rest, s);
}

// Codes of four elements as one word, lowest byte first.  int8 without conversions: the byte becomes the mantissa of
// 2^23 + 128 + code, and back by adding 1.5 * 2^23, which leaves the rounded integer in the low bits.
template <typename B> __device__ __forceinline__ Four<B> decode4(int format, uint32_t word, B scale);
template <> __device__ __forceinline__ Four<float> decode4<float>(int format, uint32_t word, float scale) {
    Four<float> r;
    if (format == kPackInt8) {
        const uint32_t w = word ^ 0x80808080u;
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[e] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + e));
        r = r + four<float>(-8388736.0f);
    } else {
        const __half2 a(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word & 0xffffu), __NV_E4M3));
        const __half2 b(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word >> 16), __NV_E4M3));
        const float2 fa = __half22float2(a), fb = __half22float2(b);
        r = {{fa.x, fa.y, fb.x, fb.y}};
    }
    return r * four<float>(scale);
}
template <> __device__ __forceinline__ Four<double> decode4<double>(int format, uint32_t word, double scale) {
    Four<double> r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[e] = from_code<double>(format, word >> 8 * e & 0xffu, scale);
    return r;
}
// |x / scale| is at most 127 (1 + 2^-21) by the choice of the scale, so rounding cannot leave the codes' range.  The product
// is rounded before it is rounded to a code (the definition; the pairwise instructions above would be merged into one
// multiply-add, which turns 63.49999952 into 63 where the float product is 63.5).
__device__ __forceinline__ uint32_t encode4(int format, const Four<float>& x, float inv) {
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = __fmul_rn(x.v[e], inv);
    uint32_t word;
    if (format == kPackInt8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = __fadd_rn(q[e], 12582912.0f);
        const uint32_t a = __byte_perm(__float_as_uint(q[0]), __float_as_uint(q[1]), 0x0040);
        const uint32_t b = __byte_perm(__float_as_uint(q[2]), __float_as_uint(q[3]), 0x0040);
        word = __byte_perm(a, b, 0x5410);
    } else {
        const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
        word = a | b << 16;
    }
    return inv == 0.0f ? 0u : word;                          // a group that is not finite
}
__device__ __forceinline__ uint32_t encode4(int format, const Four<double>& x, double inv) {
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) word |= to_code(format, x.v[e], inv) << 8 * e;
    return word;
}

}  // namespace kanb200

// linear16.cuh -- the activations of the 16-bit products (linear16.cu) and
// their slopes, in f32.
//
//   gelu(z) = z Phi(z) = max(z, 0) - |z| Q(|z|),  gelu'(z) = Phi(z) + z phi(z)
//   silu(z) = z s, s = 1 / (1 + e^-z),            silu'(z) = s (1 + z (1 - s))
//
// Q(a) = 1 - Phi(a) = e^(-a^2/2) R(a) with R(a) = erfcx(a / sqrt 2) / 2 smooth:
// a polynomial of degree 7 in t = 1 / (1 + 0.35 a), fitted to least relative
// error over 0 <= a <= 14.5 (3e-7; 6e-7 in f32).  So the tail keeps its relative
// accuracy, as erfc would, at about 17 instructions a value: an epilogue that calls
// erfcf and expf leaves the tensor core idle.  From a = 13.2 on e^(-a^2/2) is below
// 2^-126 and taken for 0, which is 5e-39 of gelu and 6e-38 of its slope.
// Against 16-bit results, half a step of which is 2^-9 or 2^-12, this is exact.
#pragma once

#include <cuda_runtime.h>

#include "chelis_cuda.h"

namespace chelis {
namespace linear16 {

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// max and min that keep a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Two f32 in a 64-bit register, the unit of Blackwell's packed arithmetic: an
// epilogue is bound by its instructions.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 both(float v) { return gemm8::pack2(v, v); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { return gemm8::fma2(a, b, c); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { return gemm8::mul2(a, b); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { return gemm8::add2(a, b); }

// What the packed gelu multiplies and adds.  Packed instructions take registers
// alone, and the compiler would rather make a constant again at each use, two
// instructions for two values: HOLD keeps it from knowing that they are constants,
// so an epilogue makes them once (67 to 64 million instructions of 16384 x 4096 x
// 1024 with gelu).
template <bool HOLD>
struct GeluConstants {
    f32x2 step, one, half_log2e, density, poly[8];
    __device__ __forceinline__ static f32x2 make(float v) {
        if constexpr (!HOLD) return both(v);
        f32x2 r;
        asm volatile("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
        return r;
    }
    __device__ __forceinline__ GeluConstants()
        : step(make(-0.35f)), one(make(1.0f)), half_log2e(make(-0.72134752044f)), density(make(0.39894228040f)),
          poly{make(-2.69914980890e-5f), make(0.140264645219f), make(0.133395001292f), make(0.155816540122f),
               make(-0.016725681722f),   make(0.240291759372f), make(-0.201901435852f), make(0.048886287957f)} {}
};
// R(a) of a = -na, 0 <= a <= 16; *gauss is e^(-a^2/2).
template <bool HOLD>
__device__ __forceinline__ f32x2 upper_tail(const GeluConstants<HOLD> &k, f32x2 na, f32x2 *gauss) {
    const float2 d = gemm8::unpack2(fma2(k.step, na, k.one));
    const f32x2 t = gemm8::pack2(rcp(d.x), rcp(d.y));
    const float2 s = gemm8::unpack2(mul2(mul2(na, k.half_log2e), na));
    const f32x2 e = gemm8::pack2(ex2(s.x), ex2(s.y));
    f32x2 r = k.poly[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) r = fma2(r, t, k.poly[i]);
    *gauss = e;
    return r;
}
// -|z|, no further than Q(16) = 0: an infinity times it would be NaN.
__device__ __forceinline__ f32x2 negative(float2 z) {
    return gemm8::pack2(max_nan(-fabsf(z.x), -16.0f), max_nan(-fabsf(z.y), -16.0f));
}
template <bool HOLD>
__device__ __forceinline__ f32x2 gelu_value(const GeluConstants<HOLD> &k, f32x2 v) {
    const float2 z = gemm8::unpack2(v);
    const f32x2 na = negative(z);
    f32x2 e;
    const f32x2 q = upper_tail(k, na, &e);
    return fma2(na, mul2(e, q), gemm8::pack2(fmaxf(z.x, 0.0f), fmaxf(z.y, 0.0f)));
}
// gelu'(-a) = Q(a) - a phi(a) = e^(-a^2/2) (R(a) - a / sqrt(2 pi)), and
// gelu'(a) = 1 - gelu'(-a).
template <bool HOLD>
__device__ __forceinline__ f32x2 gelu_slope(const GeluConstants<HOLD> &k, f32x2 v) {
    const float2 z = gemm8::unpack2(v);
    const f32x2 na = negative(z);
    f32x2 e;
    const f32x2 r = upper_tail(k, na, &e);
    const float2 h = gemm8::unpack2(mul2(e, fma2(na, k.density, r)));
    return gemm8::pack2(z.x < 0.0f ? h.x : 1.0f - h.x, z.y < 0.0f ? h.y : 1.0f - h.y);
}
// A quarter of 1 + e^-z, so that the reciprocal of one between 2^126 and 2^128 (z below
// -87.33) is no number that the hardware's takes for 0; s itself may be one.
__device__ __forceinline__ float sigmoid(float z) { return 0.25f * rcp(fmaf(ex2(z * -1.44269504089f), 0.25f, 0.25f)); }
__device__ __forceinline__ float silu_value(float z) {
    return max_nan(z, -128.0f) * sigmoid(z);  // s(-128) is 0 in f32
}
__device__ __forceinline__ float silu_slope(float z) {
    const float c = max_nan(min_nan(z, 128.0f), -128.0f), s = sigmoid(c);
    return s * fmaf(c, 1.0f - s, 1.0f);
}
// the library's relu: NaN and -0 stay, and its slope is 1 where 0 < z
__device__ __forceinline__ float relu_value(float z) { return z < 0.0f ? 0.0f : z; }

__device__ __forceinline__ float relu_slope_times(float g, float z) { return z > 0.0f ? g : 0.0f; }

template <bool HOLD>
__device__ __forceinline__ f32x2 value(const GeluConstants<HOLD> &k, f32x2 z, int32_t act) {
    const float2 f = gemm8::unpack2(z);
    switch (act) {
        case CHELIS_ACT_RELU: return gemm8::pack2(relu_value(f.x), relu_value(f.y));
        case CHELIS_ACT_GELU: return gelu_value(k, z);
        case CHELIS_ACT_SILU: return gemm8::pack2(silu_value(f.x), silu_value(f.y));
        default: return z;
    }
}
// g times the slope at z; where relu's slope is 0 the result is 0 whatever g is
template <bool HOLD>
__device__ __forceinline__ f32x2 slope_times(const GeluConstants<HOLD> &k, f32x2 g, f32x2 z, int32_t act) {
    const float2 a = gemm8::unpack2(g), f = gemm8::unpack2(z);
    switch (act) {
        case CHELIS_ACT_RELU: return gemm8::pack2(relu_slope_times(a.x, f.x), relu_slope_times(a.y, f.y));
        case CHELIS_ACT_GELU: return mul2(g, gelu_slope(k, z));
        case CHELIS_ACT_SILU: return mul2(g, gemm8::pack2(silu_slope(f.x), silu_slope(f.y)));
        default: return g;
    }
}
__device__ __forceinline__ float value(float z, int32_t act) {
    return gemm8::unpack2(value(GeluConstants<false>(), both(z), act)).x;
}
__device__ __forceinline__ float slope_times(float g, float z, int32_t act) {
    return gemm8::unpack2(slope_times(GeluConstants<false>(), both(g), both(z), act)).x;
}

}  // namespace linear16
}  // namespace chelis

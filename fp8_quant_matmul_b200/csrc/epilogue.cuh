// What a fused epilogue does with a finished sum: bias, activation, residual, the gate, all in fp32.
//   none   x                     silu       x / (1 + exp(-x))
//   relu   x < 0 ? 0 : x         gelu       x (1 + erf(x / sqrt 2)) / 2
//                                gelu_tanh  x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))) / 2 = x / (1 + exp(-2 sqrt(2/pi) (x + 0.044715 x^3)))
// An activation is a few instructions for each of a thread's 64 or 128 columns, issued by two warps per scheduler: what counts is their
// number.  4096 x 7168 x 512 with bias on pair tiles: 23 us without activation, relu 24, silu 37, gelu_tanh 38, gelu 44; a copy of silu without
// any exponential or reciprocal took 2 us less, and steps interleaved over two, four or eight pairs of values are no faster.  Two values
// share one reciprocal (1 / d0 = d1 / (d0 d1)).
// Errors (2^-22 of the exponential and of the reciprocal, the rounding of the argument): silu below 2^-17 of the result down to -40, gelu_tanh 2^-16 down to
// -7.4, less than 1 % of a bf16 step; below that they stay at -2e-16 and -2e-17 while the formulas go on to 0.  gelu: 7.5e-8 |x| of its formula and
// 2^-19 of erfc's share of the result.  An output in 8 bits has its scale from the largest elements, where the exponential is next to nothing.
// (In packed fp32 instructions the activations were no faster and the K loop of the pair kernel, which shares their registers, 17 %
// slower, whichever was chosen at run time.)
#pragma once
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <cstdint>
#include <type_traits>

namespace fp8bs {

// torch's maximum: NaN if either is (fmaxf drops it), so that a NaN in a group shows in its bytes and scale.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// The largest magnitude over a warp's lanes, NaN if one is.
__device__ __forceinline__ float warp_absmax_nan(float a)
{
    float d;
    asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(a));
    return d;
}
// Two fp32 -> two e4m3fn bytes (lo in bits 0-7, hi in bits 8-15), round to nearest even.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_ERF = 3, ACT_TANH = 4 };     // the numbers of FP8BS_ACT_*

struct Epilogue {
    const void* bias;               // [N], NULL: none
    const __nv_bfloat16* residual;  // [rows, N] with a pitch of ldr elements, NULL: none; may be C
    long long ldr;
    const float* up_scale;          // gated: b_scale of the second matrix (GemmParams::b_scale is the first one's)
    uint8_t* q_out;                 // gated with an output in 8 bits: [N][M] ...
    float* scale_out;               // ... and its inverse scales [N / 128][M]
    int bias_is_bf16;
    int act;
    float fp8_max;
};

// Two fp32 values in one 64-bit register, the operand form of fma.rn.f32x2 (low word = first value).
__device__ __forceinline__ unsigned long long pack_f32x2(float lo, float hi)
{
    return static_cast<unsigned long long>(__float_as_uint(lo)) | (static_cast<unsigned long long>(__float_as_uint(hi)) << 32);
}
__device__ __forceinline__ float f32x2_lo(unsigned long long v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float f32x2_hi(unsigned long long v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }

__device__ __forceinline__ float ex2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// x0 / (1 + 2^z0), x1 / (1 + 2^z1); z up to 60, so that the product of the denominators does not overflow.
__device__ __forceinline__ unsigned long long logistic_times_2(float x0, float x1, float z0, float z1)
{
    const float d0 = 1.0f + ex2_approx(z0), d1 = 1.0f + ex2_approx(z1), r = rcp_approx(d0 * d1);
    return pack_f32x2(x0 * (r * d1), x1 * (r * d0));
}
// silu.  Below -40 it stays at -40 / (1 + e^40) = -2e-16.  A NaN stays one, and out of the other value: its exponential is taken of something else.
__device__ __forceinline__ unsigned long long silu_2(unsigned long long x)
{
    const float x0 = max_nan(f32x2_lo(x), -40.0f), x1 = max_nan(f32x2_hi(x), -40.0f);
    constexpr float A = -1.4426950408889634f;
    return logistic_times_2(x0, x1, fminf(x0 * A, 60.0f), fminf(x1 * A, 60.0f));
}
// gelu_tanh: x / (1 + 2^(A x + B x^3)).  Below -7.4 it stays there, at -2e-17; above 40 the exponential is 0 (and x^3 could overflow).
__device__ __forceinline__ unsigned long long gelu_tanh_2(unsigned long long x)
{
    const float x0 = max_nan(f32x2_lo(x), -7.4f), x1 = max_nan(f32x2_hi(x), -7.4f);
    const float t0 = fminf(x0, 40.0f), t1 = fminf(x1, 40.0f);                       // NaN: 40
    constexpr float A = -1.4426950408889634f * 2.0f * 0.7978845608028654f, B = A * 0.044715f;
    return logistic_times_2(x0, x1, t0 * fmaf(t0 * t0, B, A), t1 * fmaf(t1 * t1, B, A));
}
// gelu: x (1 + erf(x / sqrt 2)) / 2 = max(x, 0) - |x| erfc(|x| / sqrt 2) / 2 with erfc(z) = (a1 t + .. + a5 t^5) exp(-z^2), t = 1 / (1 + p z): formula
// 7.1.26 of Abramowitz and Stegun, off by 1.5e-7 at most, that is 7.5e-8 |x| here, about what 1 + erf loses in fp32 as soon as erf is near -1.  Relative
// to the result the formula is off by 5e-5 at -3, 5e-4 at -4 (result -1.3e-4), 1.6e-3 at -5 and 3.6e-3 at -6 (-6e-9), where half a bf16 step is 2e-3 to
// 3.9e-3: below -3.5 the last bit of a bf16 result is not always the formula's.  (A sixth term and coefficients fitted for the tail give
// 3e-5 everywhere, but 48.4 -> 50.7 us on 4096 x 7168 x 512.  CUDA's erff in this place cost the K loop of the pair kernel 15 spilled registers.)
__device__ __forceinline__ unsigned long long gelu_2(unsigned long long x)
{
    const float x0 = f32x2_lo(x), x1 = f32x2_hi(x);
    const float u0 = fminf(fabsf(x0), 100.0f), u1 = fminf(fabsf(x1), 100.0f);       // the tail is 0 there; NaN becomes 100
    constexpr float P = 0.3275911f * 0.70710678118654752f, E = -0.5f * 1.4426950408889634f;
    const float p0 = fmaf(P, u0, 1.0f), p1 = fmaf(P, u1, 1.0f), r = rcp_approx(p0 * p1);
    auto tail = [](float t, float u) {                                              // -erfc / 2
        const float poly = fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.5f * 1.061405429f, 0.5f * 1.453152027f), -0.5f * 1.421413741f), 0.5f * 0.284496736f),
                                -0.5f * 0.254829592f);
        return poly * t * ex2_approx(u * u * E);
    };
    return pack_f32x2(fmaf(u0, tail(r * p1, u0), max_nan(x0, 0.0f)), fmaf(u1, tail(r * p0, u1), max_nan(x1, 0.0f)));
}
template <int ACT>
__device__ __forceinline__ unsigned long long activate_2(unsigned long long x)
{
    if constexpr (ACT == ACT_RELU) return pack_f32x2(max_nan(f32x2_lo(x), 0.0f), max_nan(f32x2_hi(x), 0.0f));       // a NaN stays one
    else if constexpr (ACT == ACT_SILU) return silu_2(x);
    else if constexpr (ACT == ACT_ERF) return gelu_2(x);
    else if constexpr (ACT == ACT_TANH) return gelu_tanh_2(x);
    else return x;
}
// f(integral constant of the activation): one branch per call of this, not per element.
template <class F>
__device__ __forceinline__ void with_activation(int which, F f)
{
    if (which == ACT_SILU) f(std::integral_constant<int, ACT_SILU>{});
    else if (which == ACT_TANH) f(std::integral_constant<int, ACT_TANH>{});
    else if (which == ACT_ERF) f(std::integral_constant<int, ACT_ERF>{});
    else if (which == ACT_RELU) f(std::integral_constant<int, ACT_RELU>{});
    else f(std::integral_constant<int, ACT_NONE>{});
}

// bias[n .. n + 3]
__device__ __forceinline__ float4 bias_4(const Epilogue& e, int n)
{
    if (e.bias_is_bf16) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(e.bias) + n));
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xffff0000u));
    }
    return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(e.bias) + n));
}
__device__ __forceinline__ float bias_1(const Epilogue& e, int n)
{
    return e.bias_is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(e.bias)[n]) : __ldg(static_cast<const float*>(e.bias) + n);
}

// The activation of R groups of four values.
template <int R>
__device__ __forceinline__ void activate_4(float4 (&v)[R], const Epilogue& e)
{
    with_activation(e.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const unsigned long long a = activate_2<decltype(act)::value>(pack_f32x2(v[i].x, v[i].y));
            const unsigned long long b = activate_2<decltype(act)::value>(pack_f32x2(v[i].z, v[i].w));
            v[i] = make_float4(f32x2_lo(a), f32x2_hi(a), f32x2_lo(b), f32x2_hi(b));
        }
    });
}
// gate = act(gate) * up
template <int R>
__device__ __forceinline__ void gate_4(float4 (&gate)[R], const float4 (&up)[R], const Epilogue& e)
{
    activate_4(gate, e);
#pragma unroll
    for (int i = 0; i < R; ++i) gate[i] = make_float4(gate[i].x * up[i].x, gate[i].y * up[i].y, gate[i].z * up[i].z, gate[i].w * up[i].w);
}

// The residual of columns n .. n + 3 of rows m, m + step, ..; those from `rows` on are left at 0.
template <int R>
__device__ __forceinline__ void residual_4(uint2 (&r)[R], const Epilogue& e, int m, int step, int rows, int n)
{
#pragma unroll
    for (int i = 0; i < R; ++i) {
        r[i] = make_uint2(0u, 0u);
        if (e.residual && m + i * step < rows) r[i] = *reinterpret_cast<const uint2*>(e.residual + (m + i * step) * e.ldr + n);
    }
}
// act(v + bias) + residual of columns n .. n + 3 of R rows.
template <int R>
__device__ __forceinline__ void finish_4(float4 (&v)[R], const uint2 (&r)[R], const Epilogue& e, int n)
{
    if (e.bias) {
        const float4 b = bias_4(e, n);
#pragma unroll
        for (int i = 0; i < R; ++i) v[i] = make_float4(v[i].x + b.x, v[i].y + b.y, v[i].z + b.z, v[i].w + b.w);
    }
    activate_4(v, e);
    if (e.residual) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            v[i] = make_float4(v[i].x + __uint_as_float(r[i].x << 16), v[i].y + __uint_as_float(r[i].x & 0xffff0000u),
                               v[i].z + __uint_as_float(r[i].y << 16), v[i].w + __uint_as_float(r[i].y & 0xffff0000u));
    }
}

// The factor that takes a group whose largest magnitude is amax to 8 bits, and the inverse scale to be stored (as in
// quantize.cuh: scale = fp8_max / max(amax, 1e-12)).  No product with the factor rounds to more than fp8_max: it is three roundings
// off at most, and eight are taken off where the largest product shows one.
__device__ __forceinline__ float scale_factor(float amax, float fp8_max, float& inverse)
{
    const float sc = __fmul_rn(__frcp_rn(max_nan(amax, 1e-12f)), fp8_max);
    inverse = __frcp_rn(sc);
    return __fmul_rn(amax, sc) > fp8_max ? __fmul_rn(sc, 1.0f - 0x1p-21f) : sc;
}

}  // namespace fp8bs

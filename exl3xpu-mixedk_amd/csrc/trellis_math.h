// trellis_math.h -- device functions shared by the kernels that multiply with
// trellis-coded weights: codebook values as fp16 pairs, the block-128 transform
// in registers, activations and their slopes, 16-bit loads and stores.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "viterbi_kernels.h"

namespace xtq {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
// Vectors at the alignment of their 16-bit elements: gfx950 takes global
// accesses of any width at any address.
typedef u4 u4_a2 __attribute__((aligned(2)));
typedef u2 u2_a2 __attribute__((aligned(2)));
typedef u2 u2_a1 __attribute__((aligned(1)));
typedef uint32_t u1_a2 __attribute__((aligned(2)));
typedef f4 f4_a4 __attribute__((aligned(4)));

// Element types of activations (the C-ABI's numbers).
enum ElemType { kBf16 = 0, kF16 = 1 };
enum Act { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

// Codebook values of two 16-bit states as a pair of halves; the EXL3 codes'
// values are fp16 numbers, so nothing is rounded here that the table has not
// rounded.  mul1: 1024 + byte sum < 2048 is the fp16 number with the bits
// 0x6400 + byte sum, and one fp16 fused multiply-add rounds once, as the table
// does.  v_mul_lo_u32 issues at the rate of v_sad_u8 and v_bfe_u32 on gfx950
// (33-37 T lane-operations/s measured), so a value costs 3.5 instructions.
template <int CODE>
__device__ __forceinline__ uint32_t code_pair(uint32_t s0, uint32_t s1) {
    if constexpr (CODE == kCodeMul1) {
        uint32_t t = __builtin_amdgcn_sad_u8(s0 * 0x83DCD12Du, 0u, 0x64006400u);
        t = __builtin_amdgcn_sad_hi_u8(s1 * 0x83DCD12Du, 0u, t);
        const _Float16 c1 = (_Float16)(1774.0f / 262144.0f), c2 = (_Float16)(-1329.0f / 128.0f);
        const h2 v = __builtin_elementwise_fma(__builtin_bit_cast(h2, t), (h2){c1, c1},
                                               (h2){c2, c2});
        return __builtin_bit_cast(uint32_t, v);
    } else {
        uint32_t a = CODE == kCode3Inst ? s0 * 89226354u + 64248484u : s0 * 0xCBAC1FEDu;
        uint32_t b = CODE == kCode3Inst ? s1 * 89226354u + 64248484u : s1 * 0xCBAC1FEDu;
        a = (a & 0x8FFF8FFFu) ^ 0x3B603B60u;
        b = (b & 0x8FFF8FFFu) ^ 0x3B603B60u;
        const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05040100u);   // low halves
        const uint32_t hi = __builtin_amdgcn_perm(b, a, 0x07060302u);   // high halves
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, lo) + __builtin_bit_cast(h2, hi));
    }
}

// fp32 value of a 16-bit activation.
template <int T>
__device__ __forceinline__ float from16(uint32_t bits) {
    if constexpr (T == kBf16) return __uint_as_float(bits << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Activation rounded to nearest even to 16 bits (the outputs' only rounding).
template <int T>
__device__ __forceinline__ uint32_t to16(float v) {
    if constexpr (T == kBf16) return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v);
    else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v);
}

__device__ __forceinline__ float half_bits(uint32_t bits) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Exponential and reciprocal of the vector unit: a few units of 2^-24, times the
// argument for the exponential, of results that are rounded to 16 bits.
__device__ __forceinline__ float fast_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ float fast_rcp(float v) { return __builtin_amdgcn_rcpf(v); }

// Normal distribution function, cdf(z) = erfc(-z / sqrt(2)) / 2, from
// erfc(x) = t exp(P(t) - x^2), t = 1 / (1 + x / 2), x >= 0, the form of W. H. Press
// et al., Numerical Recipes, section 6.2, with a P of its own: a Chebyshev fit of
// log(erfc(x) exp(x^2) / t) over x <= 20, whose relative error is 8e-8.  In fp32 the
// roundings of x and of the exponent add some x^2 2^-23 to it: 5e-7 for |z| <= 1,
// 2e-6 to 4, 7e-6 to 8, 2e-5 to 13, of results that are rounded to 2^-12 at best.
// (Small values keep their digits: the tail is not 1 - (1 - tail).)
__device__ __forceinline__ float normal_cdf(float z) {
    const float x = fabsf(z) * 0.70710678f, t = fast_rcp(__builtin_fmaf(0.5f, x, 1.0f));
    float p = 0.176894663f;
    p = __builtin_fmaf(p, t, -0.850723108f);
    p = __builtin_fmaf(p, t, 1.54551778f);
    p = __builtin_fmaf(p, t, -1.19725316f);
    p = __builtin_fmaf(p, t, 0.318832828f);
    p = __builtin_fmaf(p, t, -0.201707699f);
    p = __builtin_fmaf(p, t, 0.100208923f);
    p = __builtin_fmaf(p, t, 0.373702067f);
    p = __builtin_fmaf(p, t, 1.00003991f);
    p = __builtin_fmaf(p, t, -1.26551212f);
    const float h = 0.5f * t * fast_exp(__builtin_fmaf(-x, x, p));
    return z < 0.0f ? h : 1.0f - h;
}

// Activations in fp32 (act is uniform); relu keeps NaN.  silu's exponential
// overflows to infinity for z < -88, its reciprocal is 0 and the product -0.
template <int N>
__device__ __forceinline__ void activate(float* v, int act) {
    if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
    } else if (act == kActSilu) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= fast_rcp(1.0f + fast_exp(-v[i]));
    } else if (act == kActGelu) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= normal_cdf(v[i]);
    }
}

// Slope of the activation at z; at infinities the limits (z * exp(-z^2/2)
// and z * (1 - sigmoid) are products of infinity and zero there).
__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == kActRelu) return z > 0.0f ? 1.0f : (z == z ? 0.0f : z);
    if (act == kActSilu) {
        const float s = fast_rcp(1.0f + fast_exp(-z));
        const float t = fabsf(z) > 100.0f ? 0.0f : z * (1.0f - s);
        return s * (1.0f + t);
    }
    if (act == kActGelu) {
        const float d = fabsf(z) > 20.0f ? 0.0f : z * fast_exp(-0.5f * z * z);
        return __builtin_fmaf(0.39894228f, d, normal_cdf(z));
    }
    return 1.0f;
}

// Both at once: the activation, as activate gives it, and its slope, as act_slope does.
__device__ __forceinline__ void act_and_slope(float z, int act, float& value, float& slope) {
    if (act == kActSilu) {
        const float s = fast_rcp(1.0f + fast_exp(-z)), t = fabsf(z) > 100.0f ? 0.0f : z * (1.0f - s);
        value = z * s;
        slope = s * (1.0f + t);
    } else if (act == kActGelu) {
        const float c = normal_cdf(z), d = fabsf(z) > 20.0f ? 0.0f : z * fast_exp(-0.5f * z * z);
        value = z * c;
        slope = __builtin_fmaf(0.39894228f, d, c);
    } else {
        value = act == kActRelu && z < 0.0f ? 0.0f : z;
        slope = act_slope(z, act);
    }
}

// Data-parallel move inside a row of 16 lanes (4 of lane_xor is the mirror of 8
// lanes and the mirror of 4).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    const int b = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(b, b, CTRL, 0xf, 0xf, true));
}

// Largest value of the lanes that differ in bits 4 and 5.
__device__ __forceinline__ float rows_max(float v) {
    const uint32_t a = __float_as_uint(v);
    auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const uint32_t b = __float_as_uint(v);
    r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Value of the lane whose number differs in one bit, M = 1, 2, 4 or 8.
template <int M>
__device__ __forceinline__ float lane_xor(float v) {
    if constexpr (M == 1) return dpp<0xB1>(v);
    else if constexpr (M == 2) return dpp<0x4E>(v);
    else if constexpr (M == 4) return dpp<0x141>(dpp<0x1B>(v));
    else return dpp<0x128>(v);
}

// Largest value of the wave.
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, lane_xor<1>(v));
    v = fmaxf(v, lane_xor<2>(v));
    v = fmaxf(v, dpp<0x141>(v));        // the mirror of 8 lanes, of 16: any partner of the other half will do
    v = fmaxf(v, dpp<0x140>(v));
    return rows_max(v);
}

// One stage of the block-128 transform over lane bit 4 (M = 16) or 5 (M = 32),
// for two values a lane: v_permlane16_swap and v_permlane32_swap exchange one register's upper rows (half) with the other's
// lower, so one sum and one difference serve both lanes' values, and a second
// swap brings them home.
template <int M>
__device__ __forceinline__ void cross_pair(float& a, float& b) {
    auto swap = [](float& x, float& y) {
        const uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
        auto r = M == 32 ? __builtin_amdgcn_permlane32_swap(u, v, false, false)
                         : __builtin_amdgcn_permlane16_swap(u, v, false, false);
        x = __uint_as_float(r[0]);
        y = __uint_as_float(r[1]);
    };
    swap(a, b);
    const float s = a + b, d = a - b;
    a = s;
    b = d;
    swap(a, b);
}

// Block-128 transform (without its 1/sqrt(128)) of one row by a wave: lane l
// holds elements 2 l and 2 l + 1.
__device__ __forceinline__ void transform_row(float& a, float& b, int lane) {
    float s = a + b, d = a - b;
    auto stage = [&](auto m) {
        constexpr int M = decltype(m)::value;
        const float os = lane_xor<M>(s), od = lane_xor<M>(d);
        s = (lane & M) ? os - s : s + os;
        d = (lane & M) ? od - d : d + od;
    };
    stage(std::integral_constant<int, 1>());
    stage(std::integral_constant<int, 2>());
    stage(std::integral_constant<int, 4>());
    stage(std::integral_constant<int, 8>());
    cross_pair<16>(s, d);
    cross_pair<32>(s, d);
    a = s;
    b = d;
}

// Exponent s with v * 2^s in [2^top, 2^(top+1)) for finite v > 0; 0 for 0,
// infinities and NaN (their products then stay what they are).
__device__ __forceinline__ int shift_to(float v, int top) {
    if (!(v > 0.0f) || !(v <= 3.4028234663852886e38f)) return 0;
    return top + 1 - __builtin_amdgcn_frexp_expf(v);
}

}  // namespace xtq

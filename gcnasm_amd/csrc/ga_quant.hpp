// ga_quant.hpp -- what the kernels that quantise share: a lane's input elements,
// block maxima, the E8M0 scale rules, and the division by a scale of its own.
#pragma once

#include "ga_device.hpp"

namespace ga {

// EPL elements of a lane as they lie in memory: one 16-byte load (f32: 4,
// bf16: 8 elements) or one 8-byte load (bf16: 4). A kernel issues all its
// loads first, those of out-of-range lanes from element 0, and unpack() turns
// those into zeros: a load under a branch is waited for inside it, so several
// such loads of a lane ran one after the other (measured on MI355X together
// with the encoders' NaN rule out of the common path, prepare_mx_a_kernel:
// 8192x8192 bf16 MXFP8 43.7 -> 32.9 us, 2048x8192 MXFP4 14.3 -> 9.2).
template <int IN, int EPL>
struct Raw {
    static_assert(IN == GA_IN_BF16 || EPL == 4, "f32: 4 elements per 16-byte load");
    static constexpr int kDwords = IN == GA_IN_F32 ? 4 : EPL / 2;
    uint32_t w[kDwords];

    __device__ __forceinline__ void load(const void* x, size_t idx, bool ok)
    {
        const size_t i = ok ? idx : 0;
        if constexpr (kDwords == 4) {
            const v4i t = IN == GA_IN_F32 ? *(const v4i*)((const float*)x + i)
                                          : *(const v4i*)((const uint16_t*)x + i);
#pragma unroll
            for (int j = 0; j < 4; j++)
                w[j] = (uint32_t)t[j];
        } else {
            const uint2 t = *(const uint2*)((const uint16_t*)x + i);
            w[0] = t.x;
            w[1] = t.y;
        }
    }

    __device__ __forceinline__ void unpack(bool ok, float (&v)[EPL]) const
    {
#pragma unroll
        for (int j = 0; j < kDwords; j++) {
            const uint32_t u = ok ? w[j] : 0u;
            if constexpr (IN == GA_IN_F32) {
                v[j] = __uint_as_float(u);
            } else {
                v[2 * j] = __uint_as_float(u << 16);
                v[2 * j + 1] = __uint_as_float(u & 0xFFFF0000u);
            }
        }
    }
};

// Block maxima of |x| are taken on the bit patterns: for x >= 0 the IEEE bit
// order is the value order, and every NaN (quiet or signalling) maps to 0, so
// the maximum ignores NaNs exactly as the CPU reference's `a > amax` scan
// does (a float max would turn a signalling NaN into a NaN result).
__device__ __forceinline__ uint32_t abs_key(float x)
{
    const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
    return u > 0x7F800000u ? 0u : u;
}

template <int EPL>
__device__ __forceinline__ uint32_t amax_n(const float (&v)[EPL])
{
    uint32_t a = abs_key(v[0]);
#pragma unroll
    for (int j = 1; j < EPL; j++)
        a = max(a, abs_key(v[j]));
    return a;
}

// Maximum over aligned groups of W lanes (W = 4, 8, 16, 32). Inside a 16-lane
// row the exchange uses DPP (quad_perm xor 1 and xor 2, then the half- and
// full-row mirrors, which pair each 4- / 8-lane group with its neighbour once
// every lane of a group holds the group's max); across rows one swizzle.
template <int W>
__device__ __forceinline__ uint32_t group_max_dpp(uint32_t a)
{
    auto dpp = [](uint32_t v, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF,
                                                     false);
    };
    a = max(a, dpp(a, std::integral_constant<int, 0xB1>{})); // quad_perm(1,0,3,2)
    a = max(a, dpp(a, std::integral_constant<int, 0x4E>{})); // quad_perm(2,3,0,1)
    if constexpr (W >= 8)
        a = max(a, dpp(a, std::integral_constant<int, 0x141>{})); // row_half_mirror
    if constexpr (W >= 16)
        a = max(a, dpp(a, std::integral_constant<int, 0x140>{})); // row_mirror
    if constexpr (W >= 32)
        a = max(a, (uint32_t)__shfl_xor((int)a, 16, 64));
    return a;
}

// Maximum of the plain keys bits & 0x7FFFFFFF: one instruction per element
// instead of abs_key's three. A NaN's key is above +inf's, so a maximum above
// 0x7F800000 means the block holds a NaN; only then (rare) is the
// NaN-ignoring maximum taken.
template <int EPL>
__device__ __forceinline__ uint32_t amax_raw(const float (&v)[EPL])
{
    uint32_t a = __float_as_uint(v[0]) & 0x7FFFFFFFu;
#pragma unroll
    for (int j = 1; j < EPL; j++)
        a = max(a, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    return a;
}

// The NaN-ignoring maximum of |x| over aligned groups of W lanes. The
// recomputation is taken by the whole wave when any of its blocks holds a
// NaN (a ballot makes the branch uniform), so the lane exchanges always run
// with every lane active.
// nan says so (the same in every lane): the encoders' NaN rule is then needed.
template <int W, int EPL>
__device__ __forceinline__ uint32_t block_amax(const float (&v)[EPL], bool& nan)
{
    uint32_t a = group_max_dpp<W>(amax_raw<EPL>(v));
    nan = __builtin_amdgcn_ballot_w64(a > 0x7F800000u) != 0;
    if (nan)
        a = group_max_dpp<W>(amax_n<EPL>(v));
    return a;
}

// E8M0 exponent of an MX block whose element format (elem 0 E4M3, 1 E5M2, 2
// e2m1) has the largest value max = (1 + frac / 2^23) * 2^emax, from the bit
// pattern u of the block's maximum (no NaN). Rule 0: floor(log2(amax / max)),
// 1: ceil, 2: floor(log2 amax) - emax; within -127 .. 127, a zero block -127,
// an infinite one 127. Adding `add` carries into the exponent field where the
// rule rounds up; a zero or subnormal maximum comes out below -127 under every
// rule, so it needs no branch of its own.
struct MxScaleRule {
    uint32_t add;
    int sub;
    __device__ __forceinline__ MxScaleRule(int elem, int rule)
    {
        const uint32_t frac = elem == 2 ? 0x400000u : 0x600000u; // 6 = 1.5 * 2^2, else 1.75 * 2^n
        const int emax = elem == 2 ? 2 : (elem == 1 ? 15 : 8);
        add = rule == 0 ? 0x800000u - frac : (rule == 1 ? 0x7FFFFFu - frac : 0u);
        sub = 127 + emax + (rule == 0 ? 1 : 0);
    }
    __device__ __forceinline__ int exp(uint32_t u) const
    {
        const int e = (int)((u + add) >> 23) - sub;
        return u == 0x7F800000u ? 127 : max(e, -127);
    }
};

// The scale of a block of 128: amax / 448, 1 for zeros.
__device__ __forceinline__ float ds_scale(float amax) { return amax > 0.0f ? amax / 448.0f : 1.0f; }

// x / s for the elements that share one scale s, exact wherever the quotient
// decides an E4M3 code. For finite s >= 2^-64: the reciprocal r = 1/s
// (correctly rounded, once per scale), q0 = x*r, and two corrections
// q <- q + (x - q*s)*r, each residual and product one FMA. With r within
// half an ulp of 1/s and q within one ulp of x/s, the corrected quotient is
// x/s correctly rounded (Markstein's theorem; the first correction brings
// q0, within 1.5 ulp, inside one ulp). The residuals stay normal numbers for
// every x whose quotient is at least 2^-12 (|x| >= 2^-76), the range in which
// the fp32 quotient can change an E4M3 code; smaller quotients come out
// below 2^-11 with x's sign, and such values encode to the signed zero either
// way. The sign is taken from x, so -0 stays -0. tests/scale_div_check.c
// restates this arithmetic on the CPU and compares it with IEEE division
// (every bf16 x and random fp32 x under scales over the whole range; 1.4e9
// quotients without a mismatch). Other scales (subnormal, infinite) divide. Five
// VALU instructions per element instead of the IEEE division's ten; the choice is
// made once per scale.
struct ScaleDiv {
    float s, r;
    bool fast;
    __device__ __forceinline__ explicit ScaleDiv(float s_)
        : s(s_), r(1.0f / s_), fast(s_ >= 0x1p-64f && s_ <= 3.40282347e38f)
    {
    }
    template <int N>
    __device__ __forceinline__ void div(const float (&v)[N], float (&t)[N]) const
    {
        if (fast) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float q0 = v[j] * r;
                const float q1 = fmaf(fmaf(-q0, s, v[j]), r, q0);
                t[j] = copysignf(fmaf(fmaf(-q1, s, v[j]), r, q1), v[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++)
                t[j] = v[j] / s;
        }
    }
};

// EPL elements divided by their scale as E4M3 bytes at dst. NAN_RULE false: no
// quotient is a NaN, i.e. no element is one and the scale is neither infinite
// (inf/inf) nor zero (0/0); ScaleDiv::fast holds for no such scale.
template <bool NAN_RULE, int EPL, class D>
__device__ __forceinline__ void fp8_store_codes(const D& d, const float (&v)[EPL], uint8_t* dst)
{
    float t[EPL];
    d.div(v, t);
    uint32_t w[EPL / 4];
#pragma unroll
    for (int j = 0; j < EPL / 4; j++)
        w[j] = e4m3_encode4<NAN_RULE>(t[4 * j], t[4 * j + 1], t[4 * j + 2], t[4 * j + 3]);
    if constexpr (EPL == 8)
        *(uint2*)dst = make_uint2(w[0], w[1]);
    else
        *(uint32_t*)dst = w[0];
}

} // namespace ga

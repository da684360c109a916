// ga_mx4_cache.hpp -- the MXFP4 key/value cache: where a page keeps what, and how
// codes become matrix operands.
//
// A page of one kv head (P tokens, D elements): K codes [P][D/2], V codes
// [P/4][16][4][D/32], K scales [P][D/32], V scales [P/4][D/32][4].
//
// Why so: both products run on the 16x16x32 bf16 matrix instruction, whose
// operand gives lane 16*g + r eight consecutive summands of row r.
//   scores  S[t][q] = sum_d K[t][d] Q[q][d]: the order of d is free as long as
//           K and Q agree on it, so lane 16*g + r takes the D/4 elements d =
//           g*D/4 .. of token r: one load of D/8 bytes, 16 tokens' whole rows
//           together, under one scale (two for D = 256).
//   output  O[d][q] = sum_t V[t][d] P[t][q]: lane 16*g + r needs eight tokens
//           of one d. The order of t is free too, and taken as the scores leave
//           the first product: lane 16*g + q holds tokens 4g .. 4g+3 of each
//           16. Four tokens side by side give lane r the D/16 elements d = r*D/16 ..
//           of tokens 4g .. 4g+3 in one load of D/8 bytes, so the
//           probabilities never change lanes.
// Every token has bytes of its own, so tokens can be appended at the same time.
#pragma once

#include "ga_device.hpp"

namespace ga {

template <int D>
struct Mx4Page {
    static constexpr int kRow = D / 2;     // code bytes of a token's key or value
    static constexpr int kScales = D / 32; // scale bytes of them
    static constexpr int kLane = D / 8;    // code bytes a lane takes of 16 tokens

    int P;
    __host__ __device__ __forceinline__ explicit Mx4Page(int page_size) : P(page_size) {}
    __host__ __device__ __forceinline__ uint32_t bytes() const { return (uint32_t)P * (D + D / 16); }
    // token t of the page
    __device__ __forceinline__ uint32_t k_row(uint32_t t) const { return t * kRow; }
    // tokens 4 * quad .. + 3, elements i * D/16 ..: 4 tokens of D/32 bytes
    __device__ __forceinline__ uint32_t v_quad(uint32_t quad, uint32_t i) const
    {
        return (uint32_t)P * kRow + quad * (4 * kRow) + i * kLane;
    }
    __device__ __forceinline__ uint32_t k_scale(uint32_t t) const
    {
        return (uint32_t)P * D + t * kScales;
    }
    // tokens 4 * quad .. + 3 of 32-element block blk: 4 bytes
    __device__ __forceinline__ uint32_t v_scale(uint32_t quad, uint32_t blk) const
    {
        return (uint32_t)P * (D + kScales) + quad * (4 * kScales) + blk * 4;
    }
};

// Scale byte J of a dword as a float whose value is 2^(byte - 127): the exponent
// field is the byte. 0xFF is a NaN to the converter, as in the format.
template <int J>
__device__ __forceinline__ float e8m0_of(uint32_t w)
{
    constexpr int sh = 23 - 8 * J;
    return __uint_as_float((sh >= 0 ? w << (sh >= 0 ? sh : 0) : w >> (sh >= 0 ? 0 : -sh)) &
                           0x7F800000u);
}

// Two codes (byte B of w) times their scale as packed bf16: exact, a code has
// two significant bits.
template <int B>
__device__ __forceinline__ uint32_t fp4_pair_bf16(uint32_t w, float scale)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}

// Eight codes (a dword) under one scale as a matrix operand.
__device__ __forceinline__ v4i fp4_oct_bf16(uint32_t w, float scale)
{
    return (v4i){(int)fp4_pair_bf16<0>(w, scale), (int)fp4_pair_bf16<1>(w, scale),
                 (int)fp4_pair_bf16<2>(w, scale), (int)fp4_pair_bf16<3>(w, scale)};
}

// A code times 2^e, e = scale byte - 127 (byte 255: NaN), in fp32 without the
// converter's limits: values below the normal range are kept, those past it
// become infinite.
__device__ __forceinline__ float fp4_value(uint32_t code, uint32_t scale)
{
    const uint32_t m = code & 7u;
    // 0, .5, 1, 1.5, 2, 3, 4, 6 as halves: 0, 1, 2, 3, 4, 6, 8, 12
    const int h = m < 4 ? (int)m : (m & 1 ? 3 << (m / 2 - 1) : 2 << (m / 2 - 1));
    const float x = scale == 255u ? __uint_as_float(0x7FC00000u)
                                  : ldexpf((float)h, (int)scale - 128);
    return code & 8u ? -x : x;
}

} // namespace ga

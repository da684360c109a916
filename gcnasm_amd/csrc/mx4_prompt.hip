// mx4_prompt.hip -- attention of many rows (prompts and pieces of them) over the MXFP4
// key/value cache (the page's layout: ga_mx4_cache.hpp; the sums: ga_mx4_attention.hpp).
#include "ga_device.hpp"
#include "ga_mx4_attention.hpp"

namespace ga {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// D = A(32x16) * B(16x32) + C with bf16 operands: lane l = 32*h + r holds row r (column r of B),
// k [8h, 8h+8). Output: register i of lane l holds row 8*(i/4) + 4*h + i%4, column r.
__device__ __forceinline__ v16f mfma_bf16_32x32x16(v4i a, v4i b, v16f c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// Probabilities enter the second product in bf16, each off by up to 2^-8 of it. The output is
// divided by the sum of what entered, so that what their roundings have in common leaves no trace
// (512 equal scores below a larger one, values of 1.5: 1.492 divided by the sum of the unrounded
// ones, which stays the one that lse is taken of). What is left of an output element is at most
// 2^-8 of sum p |v - out|. Of random values it is, with the output's own rounding, 1.12, 1.21 and
// 1.25 times that rounding's root mean square (2048 tokens, D = 64, 128, 256), 1.3 for the D = 64
// pieces measured below and up to 1.4 where no row has a second term. Where a probability is more than kShare of its lane's sum so far a second bf16 term
// follows, 16 bits together: few tokens carry such a row. A second term for all of them would take
// the rest away and makes the second product twice as long: the two measured below 740 and
// 747 us where this took 596 and 648, and without the rounded ones' sum 576 and 610.
constexpr float kShare = 1.0f / 16;

// sum[i] + the four bf16 of a lane's two dwords, on the matrix cores: a lane's four are a column of
// their own, so a NaN stays in its row. v_dot2_f32_bf16, which the vector units take along with the
// rest of the softmax, made D = 64 take 678 us for this one's 648; a product of 16 columns would
// add up rows r and r + 16 in one, and 0 * NaN reach the other.
__device__ __forceinline__ v4f add_four(int a, int b, v4f sum)
{
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef int v2i __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(
        __builtin_bit_cast(v4s, (v2i){0x3F803F80, 0x3F803F80}),
        __builtin_bit_cast(v4s, (v2i){a, b}), sum, 0, 0, 0);
}

// A wave has 32 rows, a workgroup four waves; both products give a row to a lane pair (l, l + 32):
//   scores  S[token][row] = K Q^T, 32 tokens x 32 rows a product,
//   sums    O[d][row] += V^T P^T: the score registers 8u .. 8u+7 of a lane are the tokens
//           16u + 4h + {0..3, 8..11} of its row, and V's operands are laid out for just those, so
//           the probabilities go from product to product in their lanes.
// 64 tokens at a time are turned into bf16 operands in LDS once for all waves, beside
// the products of the 64 before: K as [d/8][token][8], V as [8 tokens][d/2 x parity][8 tokens],
// which a lane reads 16 bytes at a time, neighbours side by side.
//
// Bound by no unit alone: a wave's products and its softmax follow each other, and the two (D =
// 64: three) waves of a SIMD that the registers leave room for do not fill the gaps. At D = 128
// matrix instructions are under way for 47 % of the cycles and vector instructions for 52, at 2.15
// of 2.4 GHz; at D = 64 for 25 and 51 %, at 2.4 GHz. A prompt of 8192 tokens (32 heads over 8, D = 128,
// pages of 64) 580 to 606 us from card to card, 0.91 to 0.95 PFLOP/s, where a large
// bf16 product reaches 1.39; pieces of 500 to 1000 rows over up to 8191 tokens (64 heads over 8,
// D = 64, pages of 16) 650 us; 4096 tokens at D = 256 (16 heads over 4) 204 us. Capped scores take
// a tanhf each: 918 us for the first. Tried beside it, with the times of then: eight waves, whose barrier the products of all
// wait at (2048 tokens 82 us with four, 116 with eight); operands read as the compiler places
// them and not a few products ahead (677 us where that took 642); their turning between the products, a
// piece each (593, 616); D = 64 without the limit of registers that holds three waves a
// SIMD (806 us where that took 685).
template <int D>
struct PromptShape {
    static constexpr int kWaves = 4;
    static constexpr int kRows = 32 * kWaves;
    static constexpr int kChunks = D / 8;              // of a key
    static constexpr int kPer = kChunks / kWaves;      // a wave turns over, of 64 tokens
    static constexpr int kTiles = D / 32;              // output tiles of 32 elements
    static constexpr int kBytes = kTiles / 2;          // of a value's D/32 under one i
    static constexpr int kWords = D == 64 ? 2 : 4;     // a thread loads of a quad of tokens
};

// A thread's codes of the 64 tokens that its workgroup turns over next.
template <int D>
struct PromptCodes {
    using S = PromptShape<D>;
    uint32_t k[S::kPer], k_scale;
    uint32_t v[2][S::kWords], v_scale[2];
};

template <int D>
struct PromptLds {
    using S = PromptShape<D>;
    v4i k[2][S::kChunks][64];
    v4i v[2][8][S::kTiles][32];
    int left_out; // some tokens' values are past bf16
    static_assert(S::kWaves * (D / 64) * 16 * 64 * 4 <= 2 * (S::kChunks * 64 + 8 * S::kTiles * 32) * 16,
                  "add_left_out' share of k and v");
};

// Where this thread reads: token lane of the keys, quads `quad` and quad + 2 of the values.
template <int D>
struct PromptThread {
    using S = PromptShape<D>;
    int lane, wave, i, group, quad, part;
    __device__ __forceinline__ PromptThread(int lane_, int wave_)
    {
        lane = lane_;
        wave = wave_;
        i = lane & 15;
        const int half = wave / 2, q4 = lane >> 4;
        group = half * 4 + q4;                   // of 8 tokens
        quad = 8 * half + 4 * (q4 >> 1) + (q4 & 1);
        part = wave % 2;                         // which half of a token's bytes
    }

    struct Ids {
        int k, v;
    };
    // what is left of the ids once the codes are on their way, so that the next ids' loads can
    // take their registers
    struct Seen {
        uint64_t away; // tokens t0 + lane whose page is outside the cache
        bool v;        // the quads' page is inside
    };
    // BIG: pages of 64 tokens or more, so that all 64 are in one and addresses are a scalar
    // and what stays the same; else smaller pages, which start where the 64 do. t0 is a multiple
    // of 64. Past the end: of the last token.
    template <bool BIG>
    __device__ __forceinline__ Ids ids(const AttnParams& p, const int* table, int t0, int end) const
    {
        if (BIG)
            return {table[min(t0, end - 1) >> p.log2p], 0};
        return {table[min(t0 + lane, end - 1) >> p.log2p],
                table[min(t0 + 4 * quad, end - 1) >> p.log2p]};
    }
    // pages: the kv head's bytes of the first page
    template <bool BIG>
    __device__ __forceinline__ Seen load(const AttnParams& p, Mx4Page<D> lay, const uint8_t* pages,
                                         int t0, Ids id, PromptCodes<D>& c) const
    {
        const uint32_t mask = (1u << p.log2p) - 1u;
        const uint8_t *kp, *vp;  // the pages of the key and of the values
        uint32_t in = 0;         // where the 64 tokens start in the page
        uint32_t t = lane, at = quad; // the key and the quads from there
        Seen seen;
        if (BIG) {
            const int page = __builtin_amdgcn_readfirstlane(id.k);
            const bool ok = page >= 0 && page < p.num_pages;
            kp = vp = pages + (ok ? page : 0) * p.stride_page;
            in = (uint32_t)t0 & mask;
            seen = {ok ? 0 : ~0ull, ok};
        } else {
            const bool ok_k = id.k >= 0 && id.k < p.num_pages;
            const bool ok_v = id.v >= 0 && id.v < p.num_pages;
            kp = pages + (ok_k ? id.k : 0) * p.stride_page;
            vp = pages + (ok_v ? id.v : 0) * p.stride_page;
            t &= mask;
            at &= mask / 4;
            seen = {__builtin_amdgcn_ballot_w64(!ok_k), ok_v};
        }
        const uint8_t* src = kp + in * (D / 2) + (lay.k_row(t) + wave * (S::kPer * 4));
        if constexpr (S::kPer == 2) {
            const uint2 x = *(const uint2*)src;
            c.k[0] = x.x;
            c.k[1] = x.y;
        } else {
#pragma unroll
            for (int j = 0; j < S::kPer / 4; j++) {
                const v4i x = *(const v4i*)(src + 16 * j);
#pragma unroll
                for (int a = 0; a < 4; a++)
                    c.k[4 * j + a] = (uint32_t)x[a];
            }
        }
        const uint8_t* sc = kp + in * (D / 32) + (lay.k_scale(t) + wave * S::kPer / 4);
        if constexpr (S::kPer == 8)
            c.k_scale = *(const uint16_t*)sc;
        else
            c.k_scale = *sc;
        const uint8_t* vs = vp + in * (D / 2) + lay.v_quad(at, i);
        const uint8_t* vsc = vp + in * (D / 32) + lay.v_scale(at, i * (D / 16) / 32);
#pragma unroll
        for (int q = 0; q < 2; q++) { // quads quad and quad + 2 are of the same 16 tokens
            if constexpr (D == 64) {
                const uint2 x = *(const uint2*)(vs + 4 * D * q);
                c.v[q][0] = x.x;
                c.v[q][1] = x.y;
            } else if constexpr (D == 128) {
                const v4i x = *(const v4i*)(vs + 4 * D * q);
#pragma unroll
                for (int a = 0; a < 4; a++)
                    c.v[q][a] = (uint32_t)x[a];
            } else {
#pragma unroll
                for (int a = 0; a < 4; a++)
                    c.v[q][a] = *(const uint32_t*)(vs + 4 * D * q + 8 * a + 4 * part);
            }
            c.v_scale[q] = *(const uint32_t*)(vsc + D / 4 * q);
        }
        return seen;
    }
    // codes -> operands in LDS; t0, seen: as they were loaded
    __device__ __forceinline__ void turn(PromptLds<D>& lds, int buf, int t0, int end, Seen seen,
                                         PromptCodes<D>& c) const
    {
#pragma unroll
        for (int j = 0; j < S::kPer; j++)
            lds.k[buf][wave * S::kPer + j][lane] =
                fp4_oct_bf16(c.k[j], j >= 4 ? e8m0_of<1>(c.k_scale) : e8m0_of<0>(c.k_scale));
        if (t0 + 64 > end || seen.away) { // tokens that no row sees: scales that make finite values
            const int t = t0 + 4 * quad;
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const int left = seen.v ? min(max(end - t - 8 * q, 0), 4) : 0;
                c.v_scale[q] &= left == 4 ? ~0u : (1u << (8 * left)) - 1u;
            }
        }
        if (any_huge(c.v_scale[0]) | any_huge(c.v_scale[1])) {
            // values past bf16, or NaN: left to the end
            lds.left_out = 1;
#pragma unroll
            for (int q = 0; q < 2; q++)
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if ((c.v_scale[q] >> (8 * u) & 0xFFu) >= 253u) {
                        c.v_scale[q] &= ~(0xFFu << (8 * u));
                        c.v[q][D == 64 ? u / 2 : u] &= D == 64 ? 0xFFFFu << (16 - u % 2 * 16) : 0;
                    }
        }
        if (D == 256 || part == 0)
            turn_values<0>(lds, buf, c);
        else
            turn_values<D == 256 ? 0 : 1>(lds, buf, c);
    }
    // PART: which half of the bytes in the words
    template <int PART>
    __device__ __forceinline__ void turn_values(PromptLds<D>& lds, int buf,
                                                const PromptCodes<D>& c) const
    {
        static_for<S::kBytes>([&](auto byte) {
            constexpr int B = decltype(byte)::value;
            uint32_t y[2][4];
            static_for<4>([&](auto token) {
                constexpr int U = decltype(token)::value;
                constexpr int W = D == 64 ? U / 2 : U;
                constexpr int AT = D == 64 ? U % 2 * 2 + PART : (D == 128 ? 2 * PART + B : B);
                y[0][U] = fp4_pair_bf16<AT>(c.v[0][W], e8m0_of<U>(c.v_scale[0]));
                y[1][U] = fp4_pair_bf16<AT>(c.v[1][W], e8m0_of<U>(c.v_scale[1]));
            });
            v4i even, odd;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t a = y[j / 2][j % 2 * 2], b = y[j / 2][j % 2 * 2 + 1];
                even[j] = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
                odd[j] = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
            }
            const int tile = part * S::kBytes + B;
            lds.v[buf][group][tile][i] = even;
            lds.v[buf][group][tile][i + 16] = odd;
        });
    }
};

// Element d of output tile T, register r of lane half h: lane r' = 8*(r/4) + 4*h + r%4 of the tile
// is d = (r' % 16) * D/16 + 2T + r'/16.
template <int D>
__device__ __forceinline__ int out_element(int tile, int reg, int h)
{
    const int r = 8 * (reg / 4) + 4 * h + reg % 4;
    return r % 16 * (D / 16) + 2 * tile + r / 16;
}

// The tokens that turn() left out, added in fp32 by each row that sees them, times `share` for the
// sum that the output is divided by: score and values
// straight from the codes, in the order of the tokens. Rare. The sums go through
// LDS (mem: a float for each of the lane's, 64 apart), half of them at a time, so
// that this takes no registers of the loop's.
template <int D, bool CAP>
__device__ __forceinline__ void add_left_out(const AttnParams& p, Mx4Page<D> lay, const int* table,
                                              int head, int begin, int end, const Row& row, int h,
                                              float base, float share, float* mem,
                                              v16f (&acc)[D / 32])
{
    constexpr int kHalf = D / 64; // tiles
#pragma unroll
    for (int half = 0; half < 2; half++) {
#pragma unroll
        for (int x = 0; x < kHalf * 16; x++)
            mem[x * 64] = acc[half * kHalf + x / 16][x % 16];
#pragma unroll 1
        for (int t = begin; t < end; t++) {
            const int id = table[t >> p.log2p];
            if (id < 0 || id >= p.num_pages)
                continue;
            const uint8_t* page = p.pages + id * p.stride_page + (size_t)head * lay.bytes();
            const uint32_t in = (uint32_t)t & ((1u << p.log2p) - 1u);
            bool any = false;
#pragma unroll 1
            for (int b = 0; b < D / 32; b++)
                any |= page[lay.v_scale(in / 4, b) + in % 4] >= 253u;
            if (!any || !row.real || t > row.hi || t <= row.lo)
                continue;
            const uint16_t* q = p.q + row.at * p.sq_row + row.head * p.sq_head;
            float s = 0.0f;
#pragma unroll 1
            for (int d = 0; d < D; d++)
                s = fmaf(bf16_to_f32(q[d]),
                         fp4_value(page[lay.k_row(in) + d / 2] >> (d % 2 * 4) & 15u,
                                   page[lay.k_scale(in) + d / 32]),
                         s);
            const float w = exp2_of(score_log2<CAP>(p, p.q_sign ? -s : s) - base) * share;
#pragma unroll 1
            for (int x = 0; x < kHalf * 16; x++) {
                const int d = out_element<D>(half * kHalf + x / 16, x % 16, h);
                const uint32_t i = d / (D / 16), sc = page[lay.v_scale(in / 4, d / 32) + in % 4];
                const uint8_t code =
                    page[lay.v_quad(in / 4, i) + in % 4 * (D / 32) + d % (D / 16) / 2];
                if (sc >= 253u)
                    mem[x * 64] = fmaf(w, fp4_value(code >> (d % 2 * 4) & 15u, sc), mem[x * 64]);
            }
        }
#pragma unroll
        for (int x = 0; x < kHalf * 16; x++)
            acc[half * kHalf + x / 16][x % 16] = mem[x * 64];
    }
}

// BIG: pages of 64 tokens or more, which hold a tile whole, so that its address is a scalar. The two
// measured above: with pages of 64 603 us, of 32 610; D = 64 with pages of 64 620, of 16 652 (D =
// 256: alike).
template <int D, bool CAP, bool BIG>
__global__ __launch_bounds__(64 * PromptShape<D>::kWaves, D == 256 ? 1 : (D == 64 ? 3 : 2))
void mx4_prompt_kernel(AttnParams p)
{
    using S = PromptShape<D>;
    constexpr int NT = S::kTiles;
    __shared__ PromptLds<D> lds;
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (sequence, kv head) innermost: the workgroups that read the same tokens on one XCD where
    // there are a multiple of 8; the last rows, which see the most tokens, first
    const unsigned units = p.seqs * p.kv_heads;
    unsigned rest = blockIdx.x / units;
    const unsigned unit = blockIdx.x - rest * units;
    const int rb = p.row_blocks - 1 - (int)(rest % p.row_blocks);
    const int split = rest / p.row_blocks;
    const int kv_head = unit % p.kv_heads, b = unit / p.kv_heads;
    const Sequence seq(p, b);
    const Mx4Page<D> lay(1 << p.log2p);
    const int* table = p.table + b * p.s_table;
    const PromptThread<D> me(lane, wave);

    for (int first = rb * S::kRows; first < seq.n * p.group; first += p.row_blocks * S::kRows) {
        const Block blk(p, seq, first, S::kRows);
        const int begin = blk.begin() + split * p.chunk;
        const int end = split == p.splits - 1 ? blk.end() : min(blk.end(), begin + p.chunk);
        // this wave's rows; without any it only turns tokens over
        const bool busy = first + 32 * wave < seq.n * p.group;
        const Block mine(p, seq, busy ? first + 32 * wave : first, 32);
        const Row row(p, seq, mine, kv_head, busy ? lane & 31 : 32);
        v4i q[D / 16];
        {
            const uint16_t* src = p.q + row.at * p.sq_row + row.head * p.sq_head + 8 * h;
#pragma unroll
            for (int m = 0; m < D / 16; m++)
                q[m] = *(const v4i*)(src + 16 * m) ^ (int)p.q_sign;
        }
        v16f acc[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                acc[t][r] = 0.0f;
        float m = -INFINITY, base = 0.0f;
        float l = 0.0f, entered = 0.0f; // sums of the probabilities, and of their bf16 terms
        if (threadIdx.x == 0)
            lds.left_out = 0;
        __syncthreads();

        // away: the tokens from t0 on in pages outside the cache, which are hidden too
        auto step = [&](int t0, int buf, uint64_t away) {
            // operands are read kDepth products ahead: left to itself the compiler reads each
            // one right before its product and waits
            constexpr int kDepth = 4;
            v16f s[2];
            {
                auto read = [&](int n) { // products of the halves in turn
                    return lds.k[buf][2 * (n / 2) + h][32 * (n % 2) + (lane & 31)];
                };
                v4i a[kDepth];
#pragma unroll
                for (int n = 0; n < kDepth; n++)
                    a[n] = read(n);
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        s[half][r] = 0.0f;
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    s[n % 2] = mfma_bf16_32x32x16(a[n % kDepth], q[n / 2], s[n % 2]);
                    if (n + kDepth < D / 8)
                        a[n % kDepth] = read(n + kDepth);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            const bool whole = t0 > mine.lo_max && t0 + 63 <= mine.hi_min && (BIG || away == 0);
            if (CAP || !whole) {
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        s[half][r] = score_log2<CAP>(p, s[half][r]);
            }
            if (!whole) {
                const int hi = row.hi - t0 - 4 * h, lo = row.lo - t0 - 4 * h;
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int at = 32 * half + 8 * (r / 4) + r % 4; // + 4 * h
                        s[half][r] = at > hi || at <= lo ? -INFINITY : s[half][r];
                    }
                if (!BIG && away) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const uint32_t w = (uint32_t)(away >> (32 * half)) >> (4 * h);
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            s[half][r] = w & (1u << (8 * (r / 4) + r % 4)) ? -INFINITY : s[half][r];
                    }
                }
            }
            // scores times `by` are in powers of two
            const float by = CAP || !whole ? 1.0f : p.to_log2;
            float top = s[0][0];
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    top = fmaxf(top, s[half][r]);
            top *= by;
            if (__builtin_amdgcn_ballot_w64(top > m + kRaise)) {
                float t = fmaxf(top, m);
                t = fmaxf(t, __shfl_xor(t, 32, 64));
                const float f = m == -INFINITY ? 0.0f : exp2_of(m - t);
                m = t;
                base = t == -INFINITY ? 0.0f : t;
                l *= f;
                entered *= f;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        acc[t][r] *= f;
            }
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    s[half][r] = exp2_of(fmaf(s[half][r], by, -base));
            // four sums of eight, then into l: one running sum of thousands of equal numbers rounds
            // alike at every step
            float part[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                part[i] = s[i / 2][8 * (i % 2)];
#pragma unroll
                for (int r = 1; r < 8; r++)
                    part[i] += s[i / 2][8 * (i % 2) + r];
            }
            l += (part[0] + part[1]) + (part[2] + part[3]);
            v4i pr[2][2];
            auto add = [&]() {
                auto read = [&](int n) {
                    return lds.v[buf][2 * (n / NT) + h][n % NT][lane & 31];
                };
                v4i a[kDepth];
#pragma unroll
                for (int n = 0; n < kDepth; n++)
                    a[n] = read(n);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < 4 * NT; n++) {
                    acc[n % NT] = mfma_bf16_32x32x16(a[n % kDepth], pr[n / NT / 2][n / NT % 2],
                                                     acc[n % NT]);
                    if (n + kDepth < 4 * NT)
                        a[n % kDepth] = read(n + kDepth);
                    __builtin_amdgcn_sched_barrier(0);
                }
                v4f sum[2] = {(v4f){0, 0, 0, 0}, (v4f){0, 0, 0, 0}};
#pragma unroll
                for (int i = 0; i < 8; i++)
                    sum[i % 2] = add_four(pr[i / 4][i / 2 % 2][i % 2 * 2],
                                          pr[i / 4][i / 2 % 2][i % 2 * 2 + 1], sum[i % 2]);
                entered += sum[0][0] + sum[1][0];
                __builtin_amdgcn_sched_barrier(0);
            };
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int r = 0; r < 8; r++)
                    pr[half][r / 4][r % 4] =
                        (int)pack_bf16(s[half][2 * r], s[half][2 * r + 1]);
            add();
            if (__builtin_amdgcn_ballot_w64(!(exp2_of(top - base) <= kShare * l))) {
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        const uint32_t x = (uint32_t)pr[half][r / 4][r % 4];
                        pr[half][r / 4][r % 4] = (int)pack_bf16(
                            s[half][2 * r] - __uint_as_float(x << 16),
                            s[half][2 * r + 1] - __uint_as_float(x & 0xFFFF0000u));
                    }
                add();
            }
        };

        if (begin < end) {
            // Past the end the last tokens are read again and turned into zeros that no row
            // sees: under a branch the loads' registers are copied where it ends, and the copies
            // wait for the loads.
            PromptCodes<D> codes;
            const uint8_t* pages = p.pages + (size_t)kv_head * lay.bytes();
            auto ids = [&](int t0) { return me.template ids<BIG>(p, table, t0, end); };
            auto load = [&](int t0, typename PromptThread<D>::Ids id) {
                return me.template load<BIG>(p, lay, pages, t0, id, codes);
            };
            auto id = ids(begin);
            auto seen = load(begin, id);
            me.turn(lds, 0, begin, end, seen, codes);
            uint64_t next_away = seen.away;
            id = ids(begin + 64);
            seen = load(begin + 64, id);
            id = ids(begin + 128);
            __syncthreads();
            int buf = 0;
            for (int t0 = begin; t0 < end; t0 += 64, buf ^= 1) {
                me.turn(lds, buf ^ 1, t0 + 64, end, seen, codes);
                const uint64_t away = next_away;
                next_away = seen.away;
                seen = load(t0 + 128, id);
                id = ids(t0 + 192);
                if (busy && t0 <= mine.hi_max && t0 + 63 > mine.lo_min && !(BIG && away))
                    step(t0, buf, away);
                barrier_lds();
            }
        }
        l += __shfl_xor(l, 32, 64);
        entered += __shfl_xor(entered, 32, 64);
        if (begin < end && lds.left_out) // the operands are not read any more
            add_left_out<D, CAP>(p, lay, table, kv_head, begin, end, row, h, base,
                                 l == 0.0f ? 1.0f : entered / l,
                                 (float*)&lds + wave * (D / 64 * 16 * 64) + lane, acc);
        if (!row.real) {
        } else if (p.splits == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / entered;
            uint16_t* out = p.out + row.at * p.so_row + row.head * p.so_head;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                uint32_t o[NT];
#pragma unroll
                for (int t = 0; t < NT; t++)
                    o[t] = pack_bf16(acc[t][r] * inv, acc[t][r + 8] * inv);
                uint32_t* dst = (uint32_t*)(out + out_element<D>(0, r, h));
#pragma unroll
                for (int t = 0; t < NT; t += 2)
                    *(uint2*)(dst + t) = make_uint2(o[t], o[t + 1]);
            }
            if (p.lse && h == 0)
                p.lse[row.at * p.sl_row + row.head] = (m + __log2f(l)) * kLn2;
        } else {
            const size_t at = ((size_t)split * p.rows + row.at) * p.heads + row.head;
            if (h == 0)
                *(float2*)(p.ws + at * 2) = make_float2(m, l);
            if (m != -INFINITY || l != 0.0f) { // else nothing seen: the sums are not read
                float* dst = p.ws + stats_floats(p.splits, p.rows, p.heads) + at * D;
                const float f = l / entered; // the join divides by l
#pragma unroll
                for (int r = 0; r < 8; r++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        *(float2*)(dst + out_element<D>(t, r, h)) =
                            make_float2(acc[t][r] * f, acc[t][r + 8] * f);
            }
        }
        __syncthreads(); // lds.left_out is read before the next block of rows clears it
    }
}

int mx4_prompt_rows(int head_dim)
{
    return head_dim == 64 ? PromptShape<64>::kRows
                          : (head_dim == 128 ? PromptShape<128>::kRows : PromptShape<256>::kRows);
}

template <int D, bool CAP>
static void launch_prompt(AttnParams p, hipStream_t stream)
{
    // the kernel takes the maximum before the scale: its sign goes to the queries
    if (p.to_log2 < 0.0f) {
        p.to_log2 = -p.to_log2;
        p.q_sign = 0x80008000u;
    }
    const dim3 grid((unsigned)((long long)p.seqs * p.kv_heads * p.row_blocks * p.splits));
    const dim3 block(64 * PromptShape<D>::kWaves);
    if (p.log2p >= 6)
        hipLaunchKernelGGL((mx4_prompt_kernel<D, CAP, true>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((mx4_prompt_kernel<D, CAP, false>), grid, block, 0, stream, p);
}

void launch_mx4_prompt(const AttnParams& p, int head_dim, bool capped, hipStream_t stream)
{
    if (head_dim == 64)
        capped ? launch_prompt<64, true>(p, stream) : launch_prompt<64, false>(p, stream);
    else if (head_dim == 128)
        capped ? launch_prompt<128, true>(p, stream) : launch_prompt<128, false>(p, stream);
    else
        capped ? launch_prompt<256, true>(p, stream) : launch_prompt<256, false>(p, stream);
}

} // namespace ga

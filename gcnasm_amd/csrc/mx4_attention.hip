// mx4_attention.hip -- attention over the MXFP4 key/value cache, and the weights it gives
// to the cached tokens (layout and operand order: ga_mx4_cache.hpp).
#include "ga_device.hpp"
#include "ga_internal.hpp"
#include "ga_mx4_attention.hpp"

#include <algorithm>

namespace ga {

// A row's D elements as the second operand of D/32 products: lane 16*g + r the
// elements g*D/4 .. (g+1)*D/4 - 1 of row r.
template <int D>
__device__ __forceinline__ void load_q(const AttnParams& p, const Row& row, int g,
                                       v4i (&q)[D / 32])
{
    const uint16_t* src = p.q + row.at * p.sq_row + row.head * p.sq_head + g * (D / 4);
#pragma unroll
    for (int m = 0; m < D / 32; m++)
        q[m] = row.real ? *(const v4i*)(src + 8 * m) : (v4i){0, 0, 0, 0};
}

// Where 16 tokens lie: their page (clamped into the cache, ok says whether it
// was in it) and the place of the first in it.
struct Sixteen {
    const uint8_t* page;
    uint32_t t;
    bool ok;
};
template <int D>
__device__ __forceinline__ Sixteen locate(const AttnParams& p, Mx4Page<D> lay, int head, int t, int id)
{
    const bool ok = id >= 0 && id < p.num_pages;
    return {p.pages + (ok ? id : 0) * p.stride_page + (size_t)head * lay.bytes(),
            (uint32_t)t & ((1u << p.log2p) - 1u), ok};
}
template <int D>
__device__ __forceinline__ Sixteen locate(const AttnParams& p, Mx4Page<D> lay, const int* table,
                                          int head, int t, int end)
{
    return locate<D>(p, lay, head, t, table[min(t, end - 1) >> p.log2p]);
}

// A lane's codes and scales of 16 tokens' keys (row lane % 16), or values.
template <int D>
struct KeyCodes {
    static constexpr int kWords = D / 32;
    uint32_t w[kWords];
    uint32_t scale; // D = 256: two bytes, else one
    __device__ __forceinline__ void load(const Sixteen& s, Mx4Page<D> lay, int lane)
    {
        const uint32_t r = lane & 15, g = lane >> 4, t = s.t + r;
        const uint8_t* src = s.page + lay.k_row(t) + g * (D / 8);
        if constexpr (D == 64) {
            const uint2 x = *(const uint2*)src;
            w[0] = x.x;
            w[1] = x.y;
        } else {
#pragma unroll
            for (int j = 0; j < kWords / 4; j++) {
                const v4i x = *(const v4i*)(src + 16 * j);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    w[4 * j + i] = (uint32_t)x[i];
            }
        }
        const uint8_t* sc = s.page + lay.k_scale(t);
        if constexpr (D == 256)
            scale = *(const uint16_t*)(sc + 2 * g);
        else
            scale = sc[D == 64 ? g / 2 : g];
    }
    // the first operand of product m
    __device__ __forceinline__ v4i operand(int m) const
    {
        return fp4_oct_bf16(w[m], D == 256 && m >= 4 ? e8m0_of<1>(scale) : e8m0_of<0>(scale));
    }
};

// The keys of 16 tokens as operands whose product m sums d = 32m .. 32m + 31, lane 16*g + r
// the eight from 32m + 8g. The queries are then read 64 bytes of a row at a time instead of 16 bytes
// 64 apart, which is four times the rate of the L1, where many queries meet each
// key; the keys' loads are four times as many.
template <int D>
__device__ __forceinline__ void load_keys_in_order(const Sixteen& s, Mx4Page<D> lay, int lane,
                                                   v4i (&k)[D / 32])
{
    const uint32_t g = lane >> 4, t = s.t + (lane & 15);
    const uint8_t* src = s.page + lay.k_row(t) + 4 * g;
    const uint8_t* sc = s.page + lay.k_scale(t);
#pragma unroll
    for (int m = 0; m < D / 32; m++)
        k[m] = fp4_oct_bf16(*(const uint32_t*)(src + 16 * m), e8m0_of<0>(sc[m]));
}

template <int D>
struct ValueCodes {
    static constexpr int kWords = D / 32; // of 4 tokens, D/32 bytes each
    uint32_t w[kWords];
    uint32_t scale; // a byte for each of the 4 tokens
    __device__ __forceinline__ void load(const Sixteen& s, Mx4Page<D> lay, int lane)
    {
        const uint32_t i = lane & 15, quad = s.t / 4 + (lane >> 4);
        const uint8_t* src = s.page + lay.v_quad(quad, i);
        if constexpr (D == 64) {
            const uint2 x = *(const uint2*)src;
            w[0] = x.x;
            w[1] = x.y;
        } else {
#pragma unroll
            for (int j = 0; j < kWords / 4; j++) {
                const v4i x = *(const v4i*)(src + 16 * j);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    w[4 * j + k] = (uint32_t)x[k];
            }
        }
        scale = *(const uint32_t*)(s.page + lay.v_scale(quad, i * (D / 16) / 32));
    }
    // zero the codes of tokens whose scale byte is 253 or more, and that byte
    __device__ __forceinline__ void drop_huge()
    {
        static_for<4>([&](auto u) {
            if ((scale >> (8 * u) & 0xFFu) < 253u)
                return;
            scale &= ~(0xFFu << (8 * u));
            if constexpr (D == 64)
                w[u / 2] &= ~(0xFFFFu << (u % 2 * 16));
            else
                for (int j = 0; j < D / 128; j++)
                    w[u * (D / 128) + j] = 0;
        });
    }
    // byte B (elements 2B and 2B + 1 of the lane's D/16) of the 4 tokens, each a pair of bf16
    template <int B>
    __device__ __forceinline__ void pairs(uint32_t (&x)[4]) const
    {
        constexpr int kBytes = D / 32; // of a token
        static_for<4>([&](auto u) {
            constexpr int at = u * kBytes + B;
            x[u] = fp4_pair_bf16<at % 4>(w[at / 4], e8m0_of<u>(scale));
        });
    }
};

// The two products' first operands of output elements 2B and 2B + 1: eight
// tokens of each.
template <int D, int B>
__device__ __forceinline__ void value_operands(const ValueCodes<D> (&v)[2], v4i& even, v4i& odd)
{
    uint32_t x[2][4];
    v[0].template pairs<B>(x[0]);
    v[1].template pairs<B>(x[1]);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t a = x[j / 2][j % 2 * 2], b = x[j / 2][j % 2 * 2 + 1];
        even[j] = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
        odd[j] = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
    }
}

// 32 tokens of one kv head as a wave holds them.
template <int D>
struct Tile {
    KeyCodes<D> k[2];
    ValueCodes<D> v[2];
    bool ok[2];
    // the pages of its halves, in even and odd lanes
    static __device__ __forceinline__ int ids(const AttnParams& p, const int* table, int t0, int end,
                                              int lane)
    {
        return table[min(t0 + 16 * (lane & 1), end - 1) >> p.log2p];
    }
    __device__ __forceinline__ void load(const AttnParams& p, Mx4Page<D> lay, int head, int t0,
                                         int ids, int lane)
    {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const Sixteen x =
                locate<D>(p, lay, head, t0 + 16 * s, __builtin_amdgcn_readlane(ids, s));
            k[s].load(x, lay, lane);
            v[s].load(x, lay, lane);
            ok[s] = x.ok;
        }
    }
};

// Scores of 16 tokens (first operand) with RT blocks of 16 rows.
template <int D, int RT>
__device__ __forceinline__ void scores16(const KeyCodes<D>& k, const v4i (&q)[RT][D / 32],
                                         v4f (&s)[RT])
{
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
        s[rt] = (v4f){0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
        const v4i a = k.operand(i);
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
            s[rt] = mfma_bf16_16x16x32(a, q[rt][i], s[rt]);
    }
}

// ---- few rows -------------------------------------------------------------------------
// A wave goes over its tiles of 32 tokens with 16 * RT rows, the next tile's loads in
// flight: the scores leave the first product as the second one takes its
// probabilities (a lane: 8 tokens of row lane % 16), so nothing passes through LDS
// until the waves' results are joined. The tokens are split over the waves and over
// p.splits workgroups, whose results mx4_join_kernel joins.
//
// Probabilities enter the second product as two bf16 terms (16 bits of
// significand together): one alone would add as much error as the output's own
// rounding to bf16, and the matrix cores wait for memory here anyway.
//
// Bound by reading the cache: 4 x 131072 tokens (64 heads over 8, D = 128, 570 MB)
// 105 to 113 us by card with the join, 5.0 to 5.4 TB/s, where a copy reaches 5.16; 64 sequences of
// 2048 to 8192 tokens (361 MB) 79 to 85 us, 32 of up to 4096 with 8 kv heads (90 MB) 30, where the first loads, the
// waves' join and the lengths' differences show. The pages' numbers are read a tile
// before the codes and those a tile before their use: read where they are needed,
// each tile waited for its page and the codes before it (100 and 36 us). The scheduling
// barriers keep the operands of one product live at a time: without them and with the rare
// path below inside the loop the registers left room for 2 waves a SIMD instead of 3
// (64 x 8192: 134 us at the time, and 97 with 3).

// What the sums lack: the tokens with a scale byte of 253 or more, whose values
// pass bf16 or are NaN. In a product 0 * infinity would reach rows that do not
// see the token, and the probabilities' second term undo an infinity by its sign; here
// every row adds, in fp32, what it sees. Caches hold such scales only where their
// input was infinite or near the end of fp32, so this is one token at a time.
template <int D, int RT, bool CAP>
__device__ __forceinline__ void add_huge(const AttnParams& p, Mx4Page<D> lay, const int* table,
                                         int head, int from, int step, int end, int lane,
                                         const v4i (&q)[RT][D / 32], const int (&hi)[RT],
                                         const int (&lo)[RT], const float (&base)[RT],
                                         v4f (&acc)[RT][D / 16])
{
    constexpr int NT = D / 16;
    const int g = lane >> 4;
    for (int t0 = from; t0 < end; t0 += step) {
#pragma unroll 1
        for (int half = 0; half < 2; half++) {
            const Sixteen at = locate<D>(p, lay, table, head, t0 + 16 * half, end);
            KeyCodes<D> k;
            k.load(at, lay, lane);
            v4f s[RT];
            scores16<D, RT>(k, q, s);
#pragma unroll 1
            for (int u = 0; u < 16; u++) {
                const int t = t0 + 16 * half + u;
                const uint32_t in = at.t + u;
                const uint8_t own = at.page[lay.v_scale(in / 4, lane % (D / 32)) + in % 4];
                if (!at.ok || !__builtin_amdgcn_ballot_w64(own >= 253u))
                    continue;
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    const float mine = (u & 2) ? ((u & 1) ? s[rt][3] : s[rt][2])
                                               : ((u & 1) ? s[rt][1] : s[rt][0]);
                    const float x = __shfl(mine, u / 4 * 16 + (lane & 15), 64);
                    const float w = exp2_of(score_log2<CAP>(p, x) - base[rt]);
                    const bool sees = t <= hi[rt] && t > lo[rt];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t i = 4 * g + r;
                        const uint32_t sc = at.page[lay.v_scale(in / 4, i * NT / 32) + in % 4];
                        const uint8_t* codes = at.page + lay.v_quad(in / 4, i) + in % 4 * (D / 32);
#pragma unroll
                        for (int j = 0; j < NT; j++)
                            if (sees && sc >= 253u)
                                acc[rt][j][r] = fmaf(
                                    w, fp4_value(codes[j / 2] >> (j % 2 * 4) & 15u, sc),
                                    acc[rt][j][r]);
                    }
                }
            }
        }
    }
}

template <int D, int RT, bool CAP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (D == 64 ? 5 : (D == 128 ? 4 : 3)) - RT)
void mx4_rows_kernel(AttnParams p)
{
    constexpr int NT = D / 16; // output tiles of 16 elements
    constexpr int kRows = 16 * RT;
    __shared__ v4f red[WAVES / 2][RT * NT][64];
    __shared__ float red_m[WAVES][kRows], red_l[WAVES][kRows];
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // splits outermost: the last ones, which short sequences leave empty, start last
    // and spread over the XCDs
    const unsigned units = gridDim.x / p.splits;
    const int split = blockIdx.x / units;
    unsigned unit = blockIdx.x - split * units;
    const int rb = unit % p.row_blocks;
    unit /= p.row_blocks;
    const int kv_head = unit % p.kv_heads, b = unit / p.kv_heads;
    const Sequence seq(p, b);
    const Mx4Page<D> lay(1 << p.log2p);
    const int* table = p.table + b * p.s_table;

    for (int first = rb * kRows; first < seq.n * p.group; first += p.row_blocks * kRows) {
        const Block blk(p, seq, first, kRows);
        const int begin = blk.begin() + split * p.chunk;
        const int end = split == p.splits - 1 ? blk.end() : min(blk.end(), begin + p.chunk);
        v4i q[RT][D / 32];
        int hi[RT], lo[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const Row row(p, seq, blk, kv_head, rt * 16 + (lane & 15));
            load_q<D>(p, row, g, q[rt]);
            hi[rt] = row.hi;
            lo[rt] = row.lo;
        }
        v4f acc[RT][NT];
        float m[RT], base[RT], l[RT]; // base: m, or 0 where no score was finite yet
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            m[rt] = -INFINITY;
            base[rt] = 0.0f;
            l[rt] = 0.0f;
#pragma unroll
            for (int j = 0; j < NT; j++)
                acc[rt][j] = (v4f){0, 0, 0, 0};
        }
        bool huge = false; // a tile had values past bf16, or NaN
        auto step = [&](Tile<D>& tile, int t0) {
            v4f s[2][RT];
            scores16<D, RT>(tile.k[0], q, s[0]);
            __builtin_amdgcn_sched_barrier(0);
            scores16<D, RT>(tile.k[1], q, s[1]);
            __builtin_amdgcn_sched_barrier(0);
            const bool whole = t0 > blk.lo_max && t0 + 31 <= blk.hi_min && tile.ok[0] && tile.ok[1];
            float x[RT][8];
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    x[rt][j] = score_log2<CAP>(p, s[j / 4][rt][j % 4]);
            if (!whole) {
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    uint32_t keep = 0;
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int t = t0 + 16 * half + 4 * g + u;
                        const bool seen = tile.ok[half] && t <= blk.hi_max && t > blk.lo_min;
                        keep |= seen ? 0xFFu << (8 * u) : 0u;
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
                            if (!tile.ok[half] || t > hi[rt] || t <= lo[rt])
                                x[rt][4 * half + u] = -INFINITY;
                    }
                    // hidden from every row: a scale that makes finite values, times 0
                    tile.v[half].scale &= keep;
                }
            }
            if (__builtin_amdgcn_ballot_w64(any_huge(tile.v[0].scale) | any_huge(tile.v[1].scale))) {
                huge = true; // left to the end, one by one
                tile.v[0].drop_huge();
                tile.v[1].drop_huge();
            }
            bool raise = false;
            float top[RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                top[rt] = x[rt][0];
#pragma unroll
                for (int j = 1; j < 8; j++)
                    top[rt] = fmaxf(top[rt], x[rt][j]);
                raise |= top[rt] > m[rt] + kRaise;
            }
            if (__builtin_amdgcn_ballot_w64(raise)) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    float t = fmaxf(top[rt], m[rt]);
                    t = fmaxf(t, __shfl_xor(t, 16, 64));
                    t = fmaxf(t, __shfl_xor(t, 32, 64));
                    const float f = m[rt] == -INFINITY ? 0.0f : exp2_of(m[rt] - t);
                    m[rt] = t;
                    base[rt] = t == -INFINITY ? 0.0f : t;
                    l[rt] *= f;
#pragma unroll
                    for (int j = 0; j < NT; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            acc[rt][j][r] *= f;
                }
            }
            v4i ph[RT], pl[RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[rt][j] = exp2_of(x[rt][j] - base[rt]);
                    l[rt] += x[rt][j];
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t h = pack_bf16(x[rt][2 * j], x[rt][2 * j + 1]);
                    ph[rt][j] = (int)h;
                    pl[rt][j] = (int)pack_bf16(x[rt][2 * j] - __uint_as_float(h << 16),
                                               x[rt][2 * j + 1] - __uint_as_float(h & 0xFFFF0000u));
                }
            }
            static_for<D / 32>([&](auto byte) {
                constexpr int B = decltype(byte)::value;
                v4i even, odd;
                value_operands<D, B>(tile.v, even, odd);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    acc[rt][2 * B] = mfma_bf16_16x16x32(even, ph[rt], acc[rt][2 * B]);
                    acc[rt][2 * B + 1] = mfma_bf16_16x16x32(odd, ph[rt], acc[rt][2 * B + 1]);
                    acc[rt][2 * B] = mfma_bf16_16x16x32(even, pl[rt], acc[rt][2 * B]);
                    acc[rt][2 * B + 1] = mfma_bf16_16x16x32(odd, pl[rt], acc[rt][2 * B + 1]);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        if (int t0 = begin + 32 * wave; t0 < end) {
            // the next tile's codes and the pages of the one after are on their way beside a
            // tile's work; past the end the last tokens' again, not used
            constexpr int kStep = 32 * WAVES;
            Tile<D> cur;
            int ids = Tile<D>::ids(p, table, t0, end, lane);
            const int next = Tile<D>::ids(p, table, t0 + kStep, end, lane);
            cur.load(p, lay, kv_head, t0, ids, lane);
            ids = next;
            for (; t0 < end; t0 += kStep) {
                Tile<D> ahead;
                ahead.load(p, lay, kv_head, t0 + kStep, ids, lane);
                ids = Tile<D>::ids(p, table, t0 + 2 * kStep, end, lane);
                step(cur, t0);
                cur = ahead;
            }
        }
        if (huge)
            add_huge<D, RT, CAP>(p, lay, table, kv_head, begin + 32 * wave, 32 * WAVES, end, lane, q,
                                 hi, lo, base, acc);

        // join the waves: a common maximum, then the sums pairwise
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            l[rt] += __shfl_xor(l[rt], 16, 64);
            l[rt] += __shfl_xor(l[rt], 32, 64);
            if (g == 0) {
                red_m[wave][rt * 16 + lane] = m[rt];
                red_l[wave][rt * 16 + lane] = l[rt];
            }
        }
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const int r = rt * 16 + (lane & 15);
            float top = red_m[0][r];
#pragma unroll
            for (int w = 1; w < WAVES; w++)
                top = fmaxf(top, red_m[w][r]);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++)
                sum += red_m[w][r] == -INFINITY ? red_l[w][r]
                                                : red_l[w][r] * exp2_of(red_m[w][r] - top);
            const float f = m[rt] == -INFINITY ? 1.0f : exp2_of(m[rt] - top);
            m[rt] = top;
            l[rt] = sum;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    acc[rt][j][k] *= f;
        }
        for (int half = WAVES / 2; half >= 1; half /= 2) {
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        red[wave - half][rt * NT + j][lane] = acc[rt][j];
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        const v4f o = red[wave][rt * NT + j][lane];
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            acc[rt][j][k] += o[k];
                    }
            }
            __syncthreads();
        }
        if (wave != 0)
            continue;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const Row row(p, seq, blk, kv_head, rt * 16 + (lane & 15));
            if (!row.real)
                continue;
            if (p.splits == 1) {
                const float inv = l[rt] == 0.0f ? 0.0f : 1.0f / l[rt];
                uint16_t* out = p.out + row.at * p.so_row + row.head * p.so_head;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t o[NT / 2];
#pragma unroll
                    for (int j = 0; j < NT / 2; j++)
                        o[j] = pack_bf16(acc[rt][2 * j][k] * inv, acc[rt][2 * j + 1][k] * inv);
                    uint32_t* dst = (uint32_t*)(out + (4 * g + k) * NT);
#pragma unroll
                    for (int j = 0; j < NT / 2; j += 2)
                        *(uint2*)(dst + j) = make_uint2(o[j], o[j + 1]);
                }
                if (p.lse && g == 0)
                    p.lse[row.at * p.sl_row + row.head] = (m[rt] + __log2f(l[rt])) * kLn2;
            } else {
                const size_t at = ((size_t)split * p.rows + row.at) * p.heads + row.head;
                if (g == 0)
                    *(float2*)(p.ws + at * 2) = make_float2(m[rt], l[rt]);
                if (m[rt] == -INFINITY && l[rt] == 0.0f)
                    continue; // nothing seen: the sums are not read
                float* dst = p.ws + stats_floats(p.splits, p.rows, p.heads) + at * D;
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int j = 0; j < NT; j += 4)
                        *(v4f*)(dst + (4 * g + k) * NT + j) =
                            (v4f){acc[rt][j][k], acc[rt][j + 1][k], acc[rt][j + 2][k],
                                  acc[rt][j + 3][k]};
            }
        }
    }
}

// The splits of a row joined: out = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) l_s. A
// workgroup of WAVES waves a row, each wave every WAVES-th split, then the waves in
// order: the same order on every call. Bound by its launch, and with many splits by
// the latency of reading their sums, so eight are read at a time: about 4 us for a few splits. WAVES: 1
// up to 4 splits, 4 up to 64, then 16 (30000 tokens of two kv heads in 118 splits, the whole call: 13.2 us,
// 14.6 with 4).
template <int D, int WAVES>
__global__ __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) void mx4_join_kernel(AttnParams p)
{
    constexpr int E = D / 64; // elements of a lane
    constexpr int kRows = WAVES > 4 ? 1 : 4 / WAVES;
    __shared__ float part_acc[kRows * WAVES][D], part_sum[kRows * WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long unit = (long long)blockIdx.x * kRows + wave / WAVES;
    const bool real = unit < (long long)p.rows * p.heads;
    const long long row = unit / p.heads;
    const int head = (int)(unit - row * p.heads);
    const size_t step = (size_t)p.rows * p.heads;
    float acc[E] = {}, sum = 0.0f, top = -INFINITY;
    if (real) {
        const float2* stats = (const float2*)p.ws + unit;
        const float* part = p.ws + stats_floats(p.splits, p.rows, p.heads) + unit * D + lane * E;
        for (int s = lane; s < p.splits; s += 64)
            top = fmaxf(top, stats[s * step].x);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1)
            top = fmaxf(top, __shfl_xor(top, o, 64));
        for (int s0 = wave % WAVES; s0 < p.splits; s0 += 8 * WAVES) {
            float2 ml[8];
            float x[8][E];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int s = s0 + i * WAVES;
                ml[i] = s < p.splits ? stats[s * step] : make_float2(-INFINITY, 0.0f);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // splits that saw nothing have written no sums
                const bool none = ml[i].x == -INFINITY && ml[i].y == 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++)
                    x[i][e] = none ? 0.0f : part[(s0 + i * WAVES) * step * D + e];
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float f = ml[i].x == -INFINITY ? 1.0f : exp2_of(ml[i].x - top);
                sum += ml[i].y * f;
#pragma unroll
                for (int e = 0; e < E; e++)
                    acc[e] += x[i][e] * f;
            }
        }
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int e = 0; e < E; e++)
            part_acc[wave][lane * E + e] = acc[e];
        if (lane == 0)
            part_sum[wave] = sum;
        __syncthreads();
        if (wave != 0)
            return;
#pragma unroll
        for (int w = 1; w < WAVES; w++) {
            sum += part_sum[w];
#pragma unroll
            for (int e = 0; e < E; e++)
                acc[e] += part_acc[w][lane * E + e];
        }
    }
    if (!real)
        return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* out = p.out + row * p.so_row + head * p.so_head + lane * E;
    if constexpr (E == 1) {
        out[0] = f32_to_bf16(acc[0] * inv);
    } else {
#pragma unroll
        for (int e = 0; e < E; e += 2)
            *(uint32_t*)(out + e) = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
    }
    if (p.lse && lane == 0)
        p.lse[row * p.sl_row + head] = (top + __log2f(sum)) * kLn2;
}

// ---- the weights of the tokens ------------------------------------------------------------
// w[t] += sum over rows and heads of 2^(x_t - lse log2 e). The scores' product has tokens on its
// rows, so a lane adds up the probabilities of its tokens over its rows (lane % 16 of each 16),
// and the 16 lanes are added once at the end: no atomics, a fixed order.
struct WeightsParams {
    AttnParams a;
    const float* w_in;
    float* w_out;
    long long si_seq, si_head, so_seq, so_head;
    int width, chunk; // chunk: tokens of a workgroup (few rows)
    int splits;       // workgroups along the rows (many)
    float* ws;        // their sums, [splits][seqs][kv heads][width]

    // the weight so far of token t < len of a sequence
    __device__ __forceinline__ float before(int b, int head, int t) const
    {
        return w_in ? w_in[b * si_seq + head * si_head + t] : 0.0f;
    }
    __device__ __forceinline__ void store(const Sequence& s, int b, int head, int t, float x) const
    {
        if (t < width)
            w_out[b * so_seq + head * so_head + t] = t < s.len ? x + before(b, head, t) : 0.0f;
    }
};

// Sum over aligned groups of 16 lanes, in every lane of them.
__device__ __forceinline__ float sum16(float x)
{
    auto dpp = [](float v, auto ctrl) {
        return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
            0, (int)__float_as_uint(v), decltype(ctrl)::value, 0xF, 0xF, false));
    };
    x += dpp(x, std::integral_constant<int, 0xB1>{});  // quad_perm(1,0,3,2)
    x += dpp(x, std::integral_constant<int, 0x4E>{});  // quad_perm(2,3,0,1)
    x += dpp(x, std::integral_constant<int, 0x141>{}); // row_half_mirror
    x += dpp(x, std::integral_constant<int, 0x140>{}); // row_mirror
    return x;
}

// sum[4 * s + u] over its lanes, for token 16 * s + 4 * g + u in lane 16 * g + 4 * s + u.
template <int N>
__device__ __forceinline__ float own_sum(const float (&sum)[N], int lane)
{
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float y = sum16(sum[i]);
        x = (lane & 15) == i ? y : x;
    }
    return x;
}

__device__ __forceinline__ int own_token(int lane)
{
    return 16 * (lane >> 2 & 3) + 4 * (lane >> 4) + (lane & 3);
}

// 16 rows' queries and what their probabilities need.
template <int D>
struct WeightRows {
    v4i q[D / 32];
    float lse2; // lse log2 e
    int hi, lo;
};

// A lane's row of a sequence's n * group (row x: query x / group, head x % group), and steps of
// `step` rows from it without a division.
struct RowCursor {
    long long q, lse;                             // offsets of the row, in elements
    long long q0, lse0;                           // of the sequence's first row
    long long q_step, q_wrap, lse_step, lse_wrap; // of a step, and if the head wraps besides
    int in, d_in, group;                          // head of the kv head's
    int pos, d_pos;                               // position; if not causal the last token
    int top, wrap_pos;
    __device__ __forceinline__ RowCursor(const AttnParams& p, const Sequence& s, int kv_head, int x,
                                         int step, int offset)
    {
        group = p.group;
        const int i = x / group;
        in = x - i * group;
        const int di = step / group;
        d_in = step - di * group;
        q0 = s.q0 * p.sq_row + kv_head * group * p.sq_head + offset;
        lse0 = s.q0 * p.sl_row + kv_head * group;
        q = q0 + i * p.sq_row + in * p.sq_head;
        lse = lse0 + i * p.sl_row + in;
        q_step = di * p.sq_row + d_in * p.sq_head;
        q_wrap = p.sq_row - group * p.sq_head;
        lse_step = di * p.sl_row + d_in;
        lse_wrap = p.sl_row - group;
        top = s.len - 1;
        pos = p.causal ? s.len - s.n + i : top;
        d_pos = p.causal ? di : 0;
        wrap_pos = p.causal ? 1 : 0;
    }
    // the lane's operands; real: the row is one of the sequence's (which has one), otherwise
    // the first row is read, for nothing
    template <int D>
    __device__ __forceinline__ void load(const AttnParams& p, WeightRows<D>& r, bool real) const
    {
        const uint16_t* src = p.q + (real ? q : q0);
#pragma unroll
        for (int m = 0; m < D / 32; m++)
            r.q[m] = *(const v4i*)(src + 8 * m);
        r.lse2 = p.lse[real ? lse : lse0] * kLog2e;
        r.hi = real ? min(pos, top) : -1;
        r.lo = before_first(pos, p.window);
    }
    __device__ __forceinline__ void advance()
    {
        in += d_in;
        const bool wrap = in >= group;
        in -= wrap ? group : 0;
        q += q_step + (wrap ? q_wrap : 0);
        lse += lse_step + (wrap ? lse_wrap : 0);
        pos += d_pos + (wrap ? wrap_pos : 0);
    }
};

// N tiles of 16 tokens' probabilities under 16 rows added to the tokens' sums: all products
// first, so that each one's latency is behind the others.
template <int D, int N, bool CAP>
__device__ __forceinline__ void add_weights(const AttnParams& p, const v4i (&k)[N][D / 32],
                                            const WeightRows<D>& r, bool whole,
                                            const bool (&ok)[N], int t, float (&sum)[4 * N])
{
    v4f s[N];
#pragma unroll
    for (int n = 0; n < N; n++)
        s[n] = (v4f){0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
        for (int n = 0; n < N; n++)
            s[n] = mfma_bf16_16x16x32(k[n][i], r.q[i], s[n]);
    float w[4 * N];
#pragma unroll
    for (int j = 0; j < 4 * N; j++) {
        const float x = s[j / 4][j % 4];
        w[j] = exp2_of(CAP ? score_log2<CAP>(p, x) - r.lse2 : fmaf(x, p.to_log2, -r.lse2));
    }
    if (!whole) {
#pragma unroll
        for (int j = 0; j < 4 * N; j++) {
            const int at = t + 16 * (j / 4) + j % 4;
            w[j] = ok[j / 4] && at <= r.hi && at > r.lo ? w[j] : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < 4 * N; j++)
        sum[j] += w[j];
}

// Few rows (16 of a kv head's; more take the loop inside): a wave goes over its tiles of 32 tokens,
// the next one's keys in flight. Bound by reading the keys and by the vector instructions of a
// tile, three quarters of whose rows are not there with four heads a kv head: 32 sequences of up to
// 4096 tokens (32 heads over 8, D = 128) 20 us, their keys alone 10; 64 of up to 8192
// (64 over 8) 65 and 39.
template <int D, bool CAP>
__global__ __launch_bounds__(256) void mx4_weights_few_kernel(WeightsParams w)
{
    const AttnParams& p = w.a;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned units = p.seqs * p.kv_heads;
    const int part = blockIdx.x / units;
    const unsigned unit = blockIdx.x - part * units;
    const int kv_head = unit % p.kv_heads, b = unit / p.kv_heads;
    const Sequence seq(p, b);
    const Mx4Page<D> lay(1 << p.log2p);
    const int* table = p.table + b * p.s_table;
    const int rows = seq.n * p.group;
    const int end = (int)min((part + 1ll) * w.chunk, (long long)w.width);
    const int last = min(end, seq.len); // of the tokens that have keys
    // a window leaves most tokens behind: their weights stay, without a look at their keys (23
    // sequences of up to 41289 tokens, 20 heads over 4, window 6: 11 us for 77)
    int begin = part * w.chunk;
    if (p.window) {
        const long long seen = (long long)seq.len - seq.n - p.window + 1; // the first
        const int behind = (int)(min(max(seen, (long long)begin), (long long)last) - begin);
        const int skip = behind > 0 ? behind / 128 * 128 : 0;
        const float* in = w.w_in ? w.w_in + b * w.si_seq + kv_head * w.si_head : nullptr;
        float* out = w.w_out + b * w.so_seq + kv_head * w.so_head;
        if (in != out)
#pragma unroll 4
            for (int t = begin + (int)threadIdx.x; t < begin + skip; t += 256)
                out[t] = in ? in[t] : 0.0f;
        begin += skip;
    }
    begin += 32 * wave;
    WeightRows<D> r;
    auto load_rows = [&](int x0) {
        const int x = x0 + (lane & 15);
        RowCursor(p, seq, kv_head, x, 0, g * (D / 4)).load(p, r, x < rows);
    };
    if (rows > 0)
        load_rows(0);
    KeyCodes<D> k[2], ahead[2];
    bool ok[2], ok_ahead[2];
    float old = 0.0f, old_ahead = 0.0f; // weight so far of this lane's token
    auto load_keys = [&](int t0) {
        old_ahead = w.before(b, kv_head, min(t0 + own_token(lane), last - 1));
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const Sixteen x = locate<D>(p, lay, table, kv_head, t0 + 16 * s, last);
            ahead[s].load(x, lay, lane);
            ok_ahead[s] = x.ok;
        }
    };
    if (begin < last)
        load_keys(begin);
    for (int t0 = begin; t0 < end; t0 += 128) {
        float sum[8] = {};
        if (t0 < last) {
#pragma unroll
            for (int s = 0; s < 2; s++) {
                k[s] = ahead[s];
                ok[s] = ok_ahead[s];
            }
            old = old_ahead;
            load_keys(t0 + 128); // past the end: the last tokens again, not used
            v4i kop[2][D / 32];
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < D / 32; i++)
                    kop[s][i] = k[s].operand(i);
            for (int x0 = 0; x0 < rows; x0 += 16) {
                if (rows > 16)
                    load_rows(x0);
                const bool sees = ok[0] && ok[1] && t0 + 31 <= r.hi && t0 > r.lo;
                const bool whole = __builtin_amdgcn_ballot_w64(!sees) == 0;
                add_weights<D, 2, CAP>(p, kop, r, whole, ok, t0 + 4 * g, sum);
            }
        }
        const float x = own_sum<8>(sum, lane);
        const int t = t0 + own_token(lane);
        if ((lane & 15) < 8 && t < w.width)
            w.w_out[b * w.so_seq + kv_head * w.so_head + t] = t < seq.len ? old + x : 0.0f;
    }
}

// Many rows: a workgroup's four waves hold 32 tokens each, their keys as operands, and go over
// the rows together, 32 at a time through LDS, loaded while the 32 before
// are computed; workgroups along the rows leave their sums in the workspace, which
// mx4_weights_join_kernel adds in their order. Bound by issuing the exponentials (a
// quarter of the rate of other vector instructions, together as long as the product) and the product.
// Prompts of 2048 and 8192 tokens (32 heads over 8, D = 128): 39 and 342 us. Where
// those took 46 and 403, 64 tokens a wave, whose operands leave room for two waves a SIMD instead
// of four, took 54 and 410, and every wave reading rows of its own, bound by the L1, 67 and 510.
//
// A row's 16-byte pieces lie in LDS at their number xor (row % 8), so that eight rows' reads of a
// piece meet different banks.
constexpr int kWeightRows = 32, kWeightTiles = 2, kWeightTokens = 64 * kWeightTiles;
constexpr int kWeightChunk = 128; // rows of a workgroup, at least

template <int D, bool CAP>
__global__ __launch_bounds__(256, D == 64 ? 5 : (D == 128 ? 4 : 2))
void mx4_weights_many_kernel(WeightsParams w)
{
    constexpr int N = kWeightTiles;
    constexpr int kPieces = D / 8;        // 16-byte pieces of a row
    constexpr int kPass = 256 / kPieces;  // rows copied by one load of each thread
    __shared__ v4i rows_q[2][kWeightRows][kPieces];
    __shared__ float rows_lse[2][kWeightRows];
    __shared__ int rows_hi[2][kWeightRows], rows_lo[2][kWeightRows];
    __shared__ long long rows_at[2][kWeightRows]; // where q has them
    const AttnParams& p = w.a;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // (sequence, kv head) innermost: the workgroups that read the same rows are apart by a multiple
    // of 8 where there are as many, on one XCD
    const unsigned units = p.seqs * p.kv_heads;
    unsigned part = blockIdx.x / units;
    const unsigned unit = blockIdx.x - part * units;
    const int split = part % w.splits;
    part /= w.splits;
    const int kv_head = unit % p.kv_heads, b = unit / p.kv_heads;
    const Sequence seq(p, b);
    const int first = part * kWeightTokens; // of the workgroup's tokens
    const int t0 = first + 16 * N * wave;
    float sum[4 * N] = {};
    // the queries that see some of the tokens: positions first .. first + kWeightTokens - 1 +
    // window - 1
    const int pos0 = seq.len - seq.n;
    const long long i0 = p.causal ? max((long long)first - pos0, 0ll) : 0;
    const long long far =
        p.window ? (long long)first + kWeightTokens - 1 + p.window - 1 - pos0 : seq.n - 1;
    const long long see = (min((long long)seq.n, far + 1)) * p.group; // end of their rows
    const long long x_first = i0 * p.group;
    const int even = (int)((see - x_first + w.splits - 1) / w.splits);
    const int chunk = max((even + kWeightRows - 1) / kWeightRows * kWeightRows, kWeightChunk);
    const int x_begin = (int)min(see, x_first + (long long)split * chunk);
    const int x_end = (int)min(see, (long long)x_begin + chunk);
    if (first < seq.len && x_begin < x_end) {
        const Mx4Page<D> lay(1 << p.log2p);
        v4i kop[N][D / 32];
        bool ok[N], all_ok = true;
#pragma unroll
        for (int s = 0; s < N; s++) {
            const Sixteen x =
                locate<D>(p, lay, p.table + b * p.s_table, kv_head, t0 + 16 * s, seq.len);
            load_keys_in_order<D>(x, lay, lane, kop[s]);
            ok[s] = x.ok;
            all_ok &= x.ok;
        }
        // a thread carries piece tid % kPieces of row tid / kPieces of each kPass; the first
        // 32 threads know a row each, and say where the others find it, a round before
        constexpr int kLoads = kWeightRows / kPass;
        const int my_row = tid / kPieces, my_piece = tid % kPieces;
        const bool teller = tid < kWeightRows;
        RowCursor at(p, seq, kv_head, x_begin + (tid & (kWeightRows - 1)), kWeightRows, 0);
        v4i held[kLoads];
        float lse;
        int pos;
        auto tell = [&](int x0, int buf) {
            if (teller)
                rows_at[buf][tid] = x0 + tid < x_end ? at.q : at.q0;
        };
        auto fetch = [&](int x0, int buf) {
#pragma unroll
            for (int j = 0; j < kLoads; j++)
                held[j] = *(const v4i*)(p.q + rows_at[buf][j * kPass + my_row] + 8 * my_piece);
            const bool real = x0 + (tid & (kWeightRows - 1)) < x_end;
            lse = p.lse[real ? at.lse : at.lse0];
            pos = real ? at.pos : -1;
            at.advance();
        };
        auto publish = [&](int buf) {
#pragma unroll
            for (int j = 0; j < kLoads; j++) {
                const int r = j * kPass + my_row;
                rows_q[buf][r][my_piece ^ (r & 7)] = held[j];
            }
            if (teller) {
                rows_lse[buf][tid] = lse * kLog2e;
                rows_hi[buf][tid] = min(pos, at.top);
                rows_lo[buf][tid] = before_first(pos, p.window);
            }
        };
        int buf = 0;
        tell(x_begin, 0);
        __syncthreads();
        fetch(x_begin, 0);
        publish(0);
        tell(x_begin + kWeightRows, 1);
        __syncthreads();
        for (int x0 = x_begin; x0 < x_end; x0 += kWeightRows, buf ^= 1) {
            // past the end: the sequence's first row, not used
            fetch(x0 + kWeightRows, buf ^ 1);
#pragma unroll
            for (int half = 0; half < kWeightRows; half += 16) {
                const int r = half + (lane & 15);
                WeightRows<D> rows;
#pragma unroll
                for (int m = 0; m < D / 32; m++)
                    rows.q[m] = rows_q[buf][r][(4 * m + g) ^ (r & 7)];
                rows.lse2 = rows_lse[buf][r];
                rows.hi = rows_hi[buf][r];
                rows.lo = rows_lo[buf][r];
                const bool sees = all_ok && t0 + 16 * N - 1 <= rows.hi && t0 > rows.lo;
                const bool whole = __builtin_amdgcn_ballot_w64(!sees) == 0;
                add_weights<D, N, CAP>(p, kop, rows, whole, ok, t0 + 4 * g, sum);
            }
            publish(buf ^ 1);
            tell(x0 + 2 * kWeightRows, buf);
            __syncthreads();
        }
    }
    const float x = own_sum<4 * N>(sum, lane);
    const int t = t0 + own_token(lane);
    if ((lane & 15) >= 4 * N)
        return;
    if (w.splits == 1)
        w.store(seq, b, kv_head, t, x);
    else if (t < w.width)
        w.ws[((size_t)split * units + unit) * w.width + t] = x;
}

__global__ __launch_bounds__(256) void mx4_weights_join_kernel(WeightsParams w)
{
    const AttnParams& p = w.a;
    const unsigned units = p.seqs * p.kv_heads;
    const unsigned part = blockIdx.x / units, unit = blockIdx.x - part * units;
    const int t = part * 256 + threadIdx.x;
    if (t >= w.width)
        return;
    const int kv_head = unit % p.kv_heads, b = unit / p.kv_heads;
    const float* x = w.ws + (size_t)unit * w.width + t;
    const size_t step = (size_t)units * w.width;
    float sum = 0.0f;
    for (int s0 = 0; s0 < w.splits; s0 += 8) { // eight loads at a time, added in their order
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            y[i] = s0 + i < w.splits ? x[(s0 + i) * step] : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++)
            sum += y[i];
    }
    w.store(Sequence(p, b), b, kv_head, t, sum);
}

// ---- host -------------------------------------------------------------------------------
ga_status mx4_cache_check(const ga_mx4_cache* c);

static ga_status attention_check(const ga_mx4_cache* c, const ga_mx4_attention_args* a,
                                 bool pointers)
{
    if (const ga_status st = mx4_cache_check(c))
        return st;
    if (!a)
        return fail(GA_ERR_ARG, "mx4 attention: null arguments");
    if (a->seqs < 0 || a->rows < 0 || a->table_pages < 0 || a->max_q < 0 || a->max_len < 0 ||
        a->heads <= 0 || a->window < 0 || !(a->softcap >= 0.0f))
        return fail(GA_ERR_ARG, "mx4 attention: negative size, window or softcap");
    if (a->heads % c->kv_heads)
        return fail(GA_ERR_SHAPE, "mx4 attention: %d heads over %d kv heads", a->heads, c->kv_heads);
    if (a->window > 0 && !a->causal)
        return fail(GA_ERR_ARG, "mx4 attention: a window needs causal rows");
    if (!a->q_starts && a->rows != a->seqs)
        return fail(GA_ERR_SHAPE, "mx4 attention: %d rows of %d sequences need q_starts", a->rows,
                    a->seqs);
    // a row's number and the step to the next block of rows together stay below 2^31
    if ((long long)a->rows * a->heads > 0x3FFFFF00ll)
        return fail(GA_ERR_SHAPE, "mx4 attention: too many rows for one call");
    if (!pointers || a->seqs == 0 || a->rows == 0)
        return GA_OK;
    if (!a->q || !a->lens || (!a->table && a->table_pages))
        return fail(GA_ERR_ARG, "mx4 attention: null pointer");
    if ((uintptr_t)a->q % 16 || a->stride_q_row % 8 || a->stride_q_head % 8)
        return fail(GA_ERR_SHAPE, "mx4 attention: q must be 16-byte aligned with strides that are "
                                  "multiples of 8");
    return GA_OK;
}

static AttnParams params_of(const ga_mx4_cache& c, const ga_mx4_attention_args& a)
{
    AttnParams p{};
    p.q = (const uint16_t*)a.q;
    p.out = (uint16_t*)a.out;
    p.lse = a.lse;
    p.table = a.table;
    p.lens = a.lens;
    p.q_starts = a.q_starts;
    p.pages = (const uint8_t*)c.pages;
    p.num_pages = c.num_pages;
    p.stride_page = c.stride_page;
    p.sq_row = a.stride_q_row;
    p.sq_head = a.stride_q_head;
    p.so_row = a.stride_out_row;
    p.so_head = a.stride_out_head;
    p.sl_row = a.stride_lse_row;
    p.s_table = a.stride_table;
    p.seqs = a.seqs;
    p.rows = a.rows;
    p.heads = a.heads;
    p.kv_heads = c.kv_heads;
    p.group = a.heads / c.kv_heads;
    p.table_pages = a.table_pages;
    p.log2p = __builtin_ctz((unsigned)c.page_size);
    p.causal = a.causal != 0;
    p.window = a.window;
    p.to_log2 = (a.softcap > 0.0f ? a.softcap : a.scale) * kLog2e;
    p.to_cap = a.softcap > 0.0f ? a.scale / a.softcap : 0.0f;
    return p;
}

// How a call is cut. A kv head with more than 64 rows in a sequence goes to
// mx4_prompt.hip (32768 tokens, 32 heads over 8, D = 128: 256 rows of each kv head 80 us
// there and 86 here, 64 rows 41 and 39; 8 sequences of 8192 with 64 rows 68 and 59; the times
// there of before it added up the rounded probabilities, 3 to 4 % more since),
// its tokens split as prompt_chunk says. Here row blocks
// of 16 rows while a sequence has no more, else of 32 (D = 256: always 16, two
// blocks' sums do not fit the registers), and tokens in chunks of a multiple of 128, a
// tile for each of four waves:
// - Few tokens stay in one workgroup, of eight waves past 128, which saves the
//   join's launch: 1 x 513 tokens of 8 kv heads (D = 128) 8.7 us against 8.9 split,
//   and 4 us less on the host; 768 tokens 9.5 against 8.9; D = 256 already at 300
//   tokens 10.5 against 10.7, at 520 12.4 against 10.9.
// - Else up to two workgroups a CU, against 4 and 6 in one run: 64 sequences of 2048 to 8192 tokens
//   (64 heads over 8) 87 us, 92 and 96; 32 of up to 4096 31, 30 and 33; 16 of 4000 with 4
//   rows each (32 heads over 8) 23, 28 and 30, with 8 rows (64 heads over 8) 49, 55 and 69; 4 of
//   131072 121, 127 and 122. Four of D = 64, which a CU holds: 53 of up to 99211 (one kv head)
//   79, 91 with two.
// - At least 256 tokens a split (8 of 2000: 13 us, with 128 16) and at most 128 splits, whose join
//   grows: 131072 tokens of one kv head 19 us, with 64 24, with 512 28.
struct RowsPlan {
    bool prompt; // mx4_prompt.hip
    int tiles;   // else: of 16 rows
    int waves, threads; // of a workgroup
    int row_blocks, splits, chunk;
    size_t ws_floats;
};

// Tokens of a split for many rows: the cut with the least time by what was measured, in us. 64 tokens
// take a workgroup alone on its CU 1.1, 1.5, 2.6 (D = 64, 128, 256), two on a CU, of which D = 256
// has no room, 0.85 and 1.15 each; splits cost a launch, and their sums are written and
// read at 2.5 TB/s. (Before the rounded probabilities were added up, which takes all cuts alike 3 to
// 7 % more.) 32 heads over 8, D = 128: 1000 tokens 36 us, 55 in two splits, 500 21 and 29;
// 700 rows over 8000 154 us in two splits, 190 in one; 300 rows 86 in three, 94 in six, 189 in one;
// 100 rows 54 in eight, 188 in one.
static int prompt_chunk(int head_dim, long long span, long long units, int num_cu, double rows)
{
    const double alone = head_dim == 64 ? 1.1 : (head_dim == 128 ? 1.5 : 2.6);
    const double shared = head_dim == 64 ? 0.85 : (head_dim == 128 ? 1.15 : 2.6);
    const long long tiles = (span + 63) / 64;
    const long long most = std::min<long long>(tiles, std::max<long long>(1, 2ll * num_cu / units));
    long long best = tiles;
    double least = 0.0;
    for (long long s = 1; s <= most; s++) {
        const long long n = (tiles + s - 1) / s; // of a split
        const long long per_cu = (units * s + num_cu - 1) / num_cu;
        const double time = n * (per_cu == 1 ? alone : shared * per_cu) +
                            (s == 1 ? 0.0 : 6.0 + s * rows * head_dim * 8 / 2.5e6);
        if (s == 1 || time < least) {
            least = time;
            best = n;
        }
    }
    return (int)std::min<long long>(best * 64, 1 << 30);
}

static RowsPlan rows_plan(const ga_mx4_cache& c, const ga_mx4_attention_args& a, int num_cu)
{
    RowsPlan r{};
    const int group = a.heads / c.kv_heads;
    const long long max_q = a.q_starts ? std::min<long long>(std::max(a.max_q, 1), a.rows) : 1;
    const long long rows = max_q * group;
    r.prompt = rows > 64;
    r.tiles = rows <= 16 || c.head_dim == 256 ? 1 : 2;
    const int block = r.prompt ? mx4_prompt_rows(c.head_dim) : 16 * r.tiles;
    r.row_blocks = (int)((rows + block - 1) / block);
    long long span = std::min<long long>(a.max_len, (long long)a.table_pages * c.page_size);
    if (a.window > 0) // a row block's rows and the alignment of its first token
        span = std::min<long long>(span, (long long)a.window + block / group + 64);
    span = std::min<long long>(std::max<long long>(span, 1), GA_MX4_MAX_TOKENS);
    const long long units = (long long)a.seqs * c.kv_heads * r.row_blocks;
    if (r.prompt) {
        r.chunk = prompt_chunk(c.head_dim, span, units, num_cu, (double)a.rows * a.heads);
    } else {
        const bool one = r.tiles == 1 && units < 2 * num_cu && span * c.head_dim <= 640 * 128;
        r.waves = one && span > 128 ? 8 : 4;
        const long long room = (c.head_dim == 64 && r.tiles == 1 ? 4ll : 2ll) * num_cu / units;
        const long long want = one ? 1 : std::min<long long>(std::max<long long>(1, room), 128);
        r.chunk = (int)(((span + want - 1) / want + 127) / 128 * 128);
        if (want > 1)
            r.chunk = std::max(r.chunk, 256);
    }
    r.splits = (int)((span + r.chunk - 1) / r.chunk);
    // what one launch takes: without splits if their join would be too large; each workgroup
    // goes over its share of a sequence's row blocks
    r.threads = r.prompt ? 256 : 64 * r.waves;
    if (r.splits > 1 && ((long long)a.rows * a.heads + 3) / 4 > most_workgroups(256))
        r.splits = 1;
    const long long others = (long long)a.seqs * c.kv_heads * r.splits;
    r.row_blocks =
        (int)std::min<long long>(r.row_blocks, std::max(1ll, most_workgroups(r.threads) / others));
    if (r.splits > 1)
        r.ws_floats = stats_floats(r.splits, a.rows, a.heads) +
                      (size_t)r.splits * a.rows * a.heads * c.head_dim;
    return r;
}

struct WeightsPlan {
    bool few;
    int chunk, splits;
    long long grid;
    size_t ws_bytes;
};

// Few rows: tokens in chunks of a multiple of 128, up to 4 workgroups a CU, as many as it
// holds (32 sequences of 4096: 21 us, 24 with 8). Many: up to 4 workgroups a CU of at least
// 128 rows each, or up to 8 of 256 (a prompt of 8192 tokens, 32 heads over 8: 342 us, 384 with 4
// a CU, 339 with 16; of 2048: 39, 40 and 46; of 1024: 19, and 24 with 8 of 128). Each block of
// tokens divides the rows that see it: divided alike for all, half of a prompt's
// workgroups have nothing to do and the others differ most (412 and 47 us).
static WeightsPlan weights_plan(const ga_mx4_cache& c, const ga_mx4_attention_args& a, int width,
                                int num_cu)
{
    WeightsPlan r{};
    const long long units = (long long)a.seqs * c.kv_heads;
    const long long max_q = a.q_starts ? std::min(std::max(a.max_q, 1), std::max(a.rows, 1)) : 1;
    const long long rows = max_q * (a.heads / c.kv_heads);
    r.few = rows <= 16;
    r.splits = 1;
    if (r.few) {
        const long long most = std::max<long long>(1, 4ll * num_cu / units);
        r.chunk = (int)(((width + most - 1) / most + 127) / 128 * 128);
        r.grid = units * (((long long)width + r.chunk - 1) / r.chunk);
        return r;
    }
    const long long blocks = ((long long)width + kWeightTokens - 1) / kWeightTokens;
    const auto splits = [&](int per_cu, int least) {
        const long long most = std::max<long long>(1, (long long)per_cu * num_cu / (units * blocks));
        return (int)std::min<long long>(most, (rows + least - 1) / least);
    };
    r.splits = std::max(splits(4, kWeightChunk), splits(8, 2 * kWeightChunk));
    r.grid = units * blocks * r.splits;
    if (r.splits > 1)
        r.ws_bytes = (size_t)r.splits * units * width * 4;
    return r;
}

template <int D, bool CAP>
static void launch_rows(const AttnParams& p, const RowsPlan& r, unsigned grid, hipStream_t s)
{
    if constexpr (D < 256) {
        if (r.tiles == 2) {
            hipLaunchKernelGGL((mx4_rows_kernel<D, 2, CAP, 4>), dim3(grid), dim3(256), 0, s, p);
            return;
        }
    }
    if (r.waves == 8)
        hipLaunchKernelGGL((mx4_rows_kernel<D, 1, CAP, 8>), dim3(grid), dim3(512), 0, s, p);
    else
        hipLaunchKernelGGL((mx4_rows_kernel<D, 1, CAP, 4>), dim3(grid), dim3(256), 0, s, p);
}

// f(std::integral_constant<int, D>, std::bool_constant<capped>)
template <class F>
static void with_dim_cap(int d, bool cap, F&& f)
{
    auto with = [&](auto dim) {
        if (cap)
            f(dim, std::true_type{});
        else
            f(dim, std::false_type{});
    };
    if (d == 64)
        with(std::integral_constant<int, 64>{});
    else if (d == 128)
        with(std::integral_constant<int, 128>{});
    else
        with(std::integral_constant<int, 256>{});
}

} // namespace ga

using namespace ga;

extern "C" {

ga_status ga_mx4_attention_workspace_bytes(const ga_mx4_cache* cache,
                                           const ga_mx4_attention_args* args, size_t* bytes)
{
    if (!bytes)
        return fail(GA_ERR_ARG, "mx4 attention: null pointer");
    if (const ga_status st = attention_check(cache, args, false))
        return st;
    *bytes = 0;
    if (args->seqs == 0 || args->rows == 0)
        return GA_OK;
    int num_cu = 0;
    if (const ga_status st = device_cu_count(&num_cu))
        return st;
    *bytes = rows_plan(*cache, *args, num_cu).ws_floats * 4;
    return GA_OK;
}

ga_status ga_mx4_attention(const ga_mx4_cache* cache, const ga_mx4_attention_args* args,
                           void* workspace, size_t workspace_bytes, void* stream)
{
    if (const ga_status st = attention_check(cache, args, true))
        return st;
    const ga_mx4_attention_args& a = *args;
    if (a.seqs == 0 || a.rows == 0)
        return GA_OK;
    if (!a.out || (uintptr_t)a.out % 16 || a.stride_out_row % 8 || a.stride_out_head % 8)
        return fail(GA_ERR_SHAPE, "mx4 attention: out must be 16-byte aligned with strides that are "
                                  "multiples of 8");
    int num_cu = 0;
    if (const ga_status st = device_cu_count(&num_cu))
        return st;
    const RowsPlan r = rows_plan(*cache, a, num_cu);
    if (r.ws_floats && (!workspace || workspace_bytes < r.ws_floats * 4))
        return fail(GA_ERR_WORKSPACE, "mx4 attention: workspace holds %zu bytes, need %zu",
                    workspace ? workspace_bytes : (size_t)0, r.ws_floats * 4);
    if ((uintptr_t)workspace % 16)
        return fail(GA_ERR_ARG, "mx4 attention: workspace must be 16-byte aligned");
    const long long grid = (long long)a.seqs * cache->kv_heads * r.row_blocks * r.splits;
    if (grid > most_workgroups(r.threads))
        return fail(GA_ERR_SHAPE, "mx4 attention: too many sequences for one call");
    AttnParams p = params_of(*cache, a);
    p.row_blocks = r.row_blocks;
    p.splits = r.splits;
    p.chunk = r.chunk;
    p.ws = (float*)workspace;
    hipStream_t st = (hipStream_t)stream;
    with_dim_cap(cache->head_dim, a.softcap > 0.0f, [&](auto dim, auto cap) {
        constexpr int D = decltype(dim)::value;
        if (r.prompt)
            launch_mx4_prompt(p, D, decltype(cap)::value, st);
        else
            launch_rows<D, decltype(cap)::value>(p, r, (unsigned)grid, st);
        const long long joins = (long long)a.rows * a.heads;
        if (r.splits > 64 && joins <= most_workgroups(1024))
            hipLaunchKernelGGL((mx4_join_kernel<D, 16>), dim3((unsigned)joins), dim3(1024), 0, st,
                               p);
        else if (r.splits > 4 && joins <= most_workgroups(256))
            hipLaunchKernelGGL((mx4_join_kernel<D, 4>), dim3((unsigned)joins), dim3(256), 0, st, p);
        else if (r.splits > 1)
            hipLaunchKernelGGL((mx4_join_kernel<D, 1>), dim3((unsigned)((joins + 3) / 4)), dim3(256),
                               0, st, p);
    });
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

ga_status ga_mx4_attention_weights_workspace_bytes(const ga_mx4_cache* cache,
                                                   const ga_mx4_attention_args* args, int width,
                                                   size_t* bytes)
{
    if (!bytes)
        return fail(GA_ERR_ARG, "mx4 attention weights: null pointer");
    if (const ga_status st = attention_check(cache, args, false))
        return st;
    if (width < 0)
        return fail(GA_ERR_ARG, "mx4 attention weights: negative width");
    if (width > GA_MX4_MAX_TOKENS)
        return fail(GA_ERR_SHAPE, "mx4 attention weights: too many tokens for one call");
    *bytes = 0;
    if (args->seqs == 0 || width == 0)
        return GA_OK;
    int num_cu = 0;
    if (const ga_status st = device_cu_count(&num_cu))
        return st;
    *bytes = weights_plan(*cache, *args, width, num_cu).ws_bytes;
    return GA_OK;
}

ga_status ga_mx4_attention_weights(const ga_mx4_cache* cache, const ga_mx4_attention_args* args,
                                   const float* w_in, long long stride_in_seq,
                                   long long stride_in_head, float* w_out,
                                   long long stride_out_seq, long long stride_out_head, int width,
                                   void* workspace, size_t workspace_bytes, void* stream)
{
    if (const ga_status st = attention_check(cache, args, true))
        return st;
    const ga_mx4_attention_args& a = *args;
    if (width < 0)
        return fail(GA_ERR_ARG, "mx4 attention weights: negative width");
    if (width > GA_MX4_MAX_TOKENS)
        return fail(GA_ERR_SHAPE, "mx4 attention weights: too many tokens for one call");
    if (a.seqs == 0 || width == 0)
        return GA_OK;
    // without rows the kernels still look the tokens' pages up
    if (!w_out || !a.lens || (!a.table && a.table_pages) || (a.rows && !a.lse))
        return fail(GA_ERR_ARG, "mx4 attention weights: null pointer");
    int num_cu = 0;
    if (const ga_status st = device_cu_count(&num_cu))
        return st;
    const WeightsPlan r = weights_plan(*cache, a, width, num_cu);
    if (r.ws_bytes && (!workspace || workspace_bytes < r.ws_bytes))
        return fail(GA_ERR_WORKSPACE, "mx4 attention weights: workspace holds %zu bytes, need %zu",
                    workspace ? workspace_bytes : (size_t)0, r.ws_bytes);
    if ((uintptr_t)workspace % 4)
        return fail(GA_ERR_ARG, "mx4 attention weights: workspace must be 4-byte aligned");
    if (r.grid > most_workgroups(256))
        return fail(GA_ERR_SHAPE, "mx4 attention weights: too many sequences or tokens for one "
                                  "call");
    const WeightsParams w{params_of(*cache, a), w_in,    w_out,    stride_in_seq,
                          stride_in_head,       stride_out_seq, stride_out_head,
                          width,                r.chunk, r.splits, (float*)workspace};
    hipStream_t st = (hipStream_t)stream;
    with_dim_cap(cache->head_dim, a.softcap > 0.0f, [&](auto dim, auto cap) {
        constexpr int D = decltype(dim)::value;
        constexpr bool CAP = decltype(cap)::value;
        if (r.few)
            hipLaunchKernelGGL((mx4_weights_few_kernel<D, CAP>), dim3((unsigned)r.grid), dim3(256),
                               0, st, w);
        else
            hipLaunchKernelGGL((mx4_weights_many_kernel<D, CAP>), dim3((unsigned)r.grid), dim3(256),
                               0, st, w);
    });
    if (r.splits > 1)
        hipLaunchKernelGGL(mx4_weights_join_kernel,
                           dim3((unsigned)((long long)a.seqs * cache->kv_heads *
                                           (((long long)width + 255) / 256))),
                           dim3(256), 0, st, w);
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

} // extern "C"

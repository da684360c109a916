// ga_mx4_attention.hpp -- what the attention kernels over the MXFP4 cache share: their
// arguments, and which tokens a block of rows sees.
//
// For row i (position len - n + i) of a sequence and the tokens t that it sees:
//   x_t = scale q.k_t  (or softcap tanh(scale q.k_t / softcap)),  in powers of two:
//   m = max x_t,  l = sum 2^(x_t - m),  out = sum 2^(x_t - m) v_t / l,  lse = (m + log2 l) ln 2
// kept as running values over the tokens, so the scores are never stored.
#pragma once

#include "ga_mx4_cache.hpp"
#include "ga_mx4_positions.hpp"

namespace ga {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf16 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnParams {
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    const int *table, *lens, *q_starts;
    const uint8_t* pages;
    long long num_pages, stride_page;
    long long sq_row, sq_head, so_row, so_head, sl_row, s_table;
    int seqs, rows, heads, kv_heads, group, table_pages, log2p;
    int causal, window;
    float to_log2; // scores to powers of two: scale * log2(e), or softcap * log2(e)
    float to_cap;  // scale / softcap
    uint32_t q_sign; // prompts: the sign bits of two bf16, or 0
    int row_blocks; // workgroups along a sequence's rows; each takes every row_blocks-th block
    int splits, chunk; // workgroups along the tokens, tokens of each
    float* ws;         // [splits][rows][heads] {m, l}, then [splits][rows][heads][D]
};

__host__ __device__ inline size_t stats_floats(int splits, int rows, int heads)
{
    return ((size_t)splits * rows * heads * 2 + 3) / 4 * 4;
}

// A sequence's rows and tokens; whatever the tables hold, inside the operands.
struct Sequence {
    int q0, n, len;
    __device__ __forceinline__ Sequence(const AttnParams& p, int b)
    {
        q0 = b;
        n = 1;
        if (p.q_starts) {
            q0 = min(max(p.q_starts[b], 0), p.rows);
            n = min(max(p.q_starts[b + 1] - q0, 0), p.rows - q0);
        }
        const long long cap = (long long)p.table_pages << p.log2p;
        len = (int)min((long long)max(p.lens[b], 0), min(cap, (long long)GA_MX4_MAX_TOKENS));
    }
};

// Rows r0 .. r0 + count - 1 of a sequence's n * group (row r: query r / group, head
// r % group) and what they see.
struct Block : Seen {
    int r0, count;
    __device__ __forceinline__ Block(const AttnParams& p, const Sequence& s, int first, int most)
        : Block(p, s, first, min(most, s.n * p.group - first), 0)
    {
    }

private:
    __device__ __forceinline__ Block(const AttnParams& p, const Sequence& s, int first, int rows, int)
        : Seen(s.len, s.n, first / p.group, (first + rows - 1) / p.group, p.causal, p.window),
          r0(first), count(rows)
    {
    }
};

struct Row {
    bool real;
    int head;      // query head
    long long at;  // row of q and out
    int hi, lo;    // sees tokens in (lo, hi]
    __device__ __forceinline__ Row(const AttnParams& p, const Sequence& s, const Block& blk,
                                   int kv_head, int r)
    {
        real = r < blk.count;
        const int x = real ? blk.r0 + r : blk.r0;
        const int i = x / p.group;
        head = kv_head * p.group + (x - i * p.group);
        at = s.q0 + i;
        hi = real ? last_seen(s.len - s.n + i, s.len, p.causal) : -1;
        lo = before_first(s.len - s.n + i, p.window);
    }
};

template <bool CAP>
__device__ __forceinline__ float score_log2(const AttnParams& p, float qk)
{
    return CAP ? tanhf(qk * p.to_cap) * p.to_log2 : qk * p.to_log2;
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, v2bf16));
}

// Nonzero if one of a dword's four scale bytes is 253 or more: its values may pass bf16
// (4 * 2^126), or are NaN.
__device__ __forceinline__ uint32_t any_huge(uint32_t w)
{
    return ((w & 0x7F7F7F7Fu) + 0x03030303u) & w & 0x80808080u;
}

// The running maximum is raised only when a score passes it by 2^8: until then
// probabilities up to 2^8 stand in the same sums, which fp32 holds as exactly, and
// neither the exchange between lanes nor the rescaling is needed.
constexpr float kRaise = 8.0f;

// Prompts (mx4_prompt.hip): rows of a workgroup, and the launch. p.row_blocks and
// p.splits workgroups along rows and tokens, p.chunk a multiple of 64.
int mx4_prompt_rows(int head_dim);
void launch_mx4_prompt(const AttnParams& p, int head_dim, bool capped, hipStream_t stream);

} // namespace ga

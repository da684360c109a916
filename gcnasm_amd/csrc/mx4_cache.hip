// mx4_cache.hip -- writing, reading back and thinning out the MXFP4 key/value cache
// (layout: ga_mx4_cache.hpp).
#include "ga_device.hpp"
#include "ga_internal.hpp"
#include "ga_mx4_cache.hpp"
#include "ga_mx4_positions.hpp"
#include "ga_quant.hpp"

#include <algorithm>

namespace ga {

struct CacheView {
    uint8_t* pages;
    long long num_pages, stride_page;
    int heads, log2p;

    __device__ __forceinline__ int page_size() const { return 1 << log2p; }
    // one head's page; in_cache() has to hold
    __device__ __forceinline__ uint8_t* page(long long id, int head, uint32_t bytes) const
    {
        return pages + id * stride_page + (size_t)head * bytes;
    }
    __device__ __forceinline__ bool in_cache(long long id) const
    {
        return id >= 0 && id < num_pages;
    }
};

static CacheView view_of(const ga_mx4_cache& c)
{
    return {(uint8_t*)c.pages, c.num_pages, c.stride_page, c.kv_heads,
            __builtin_ctz((unsigned)c.page_size)};
}

// ---- append -----------------------------------------------------------------------
// A lane quantises EPL elements of a token's key and the same ones of its value,
// 32 / EPL lanes a block: both loads are in flight before the first maximum is
// taken. Bound by bytes: the input once, 17/32 of a byte per element out (8191 tokens of
// 8 heads, D = 128, from bf16, 42 MB: 12 us).
template <int D, int EPL>
__device__ __forceinline__ void store_value_codes(uint8_t* page, Mx4Page<D> lay, uint32_t t,
                                                  uint32_t d, uint32_t w)
{
    constexpr uint32_t kPer = D / 16; // elements of one i
    const uint32_t u = t % 4 * (D / 32);
    if constexpr (EPL == 8 && D == 64) { // two i's of 4 elements
        *(uint16_t*)(page + lay.v_quad(t / 4, d / kPer) + u) = (uint16_t)w;
        *(uint16_t*)(page + lay.v_quad(t / 4, d / kPer + 1) + u) = (uint16_t)(w >> 16);
    } else {
        uint8_t* dst = page + lay.v_quad(t / 4, d / kPer) + u + d % kPer / 2;
        if constexpr (EPL == 8)
            *(uint32_t*)dst = w;
        else
            *(uint16_t*)dst = (uint16_t)w;
    }
}

template <int EPL, bool NAN_RULE>
__device__ __forceinline__ uint32_t scaled_codes(const float (&v)[EPL], int e)
{
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < EPL; j += 4)
        w |= e2m1_encode4<NAN_RULE>(ldexpf(v[j], -e), ldexpf(v[j + 1], -e), ldexpf(v[j + 2], -e),
                                    ldexpf(v[j + 3], -e))
             << (4 * j);
    return w;
}

template <int IN, int EPL, int D>
__global__ __launch_bounds__(256) void mx4_append_kernel(
    CacheView c, const void* __restrict__ k, const void* __restrict__ v, int tokens,
    long long sk_row, long long sk_head, long long sv_row, long long sv_head,
    const long long* __restrict__ slots, int rule)
{
    constexpr int LPB = 32 / EPL, LPR = D / EPL; // lanes per block, per row
    const long long lane = (long long)blockIdx.x * 256 + threadIdx.x;
    const uint32_t row = (uint32_t)(lane / LPR);
    const uint32_t d = (uint32_t)(lane % LPR) * EPL;
    const uint32_t tok = row / (uint32_t)c.heads;
    const int head = (int)(row - tok * (uint32_t)c.heads);
    const bool real = tok < (uint32_t)tokens;
    Raw<IN, EPL> rk, rv;
    rk.load(k, (size_t)(tok * sk_row + head * sk_head + d), real);
    rv.load(v, (size_t)(tok * sv_row + head * sv_head + d), real);
    const long long slot = real ? slots[tok] : -1;
    const MxScaleRule scale(2, rule);
    float vk[EPL], vv[EPL];
    rk.unpack(real, vk);
    rv.unpack(real, vv);
    bool nan_k, nan_v;
    const int ek = scale.exp(block_amax<LPB, EPL>(vk, nan_k));
    const int ev = scale.exp(block_amax<LPB, EPL>(vv, nan_v));
    const long long id = slot >> c.log2p;
    if (!real || !c.in_cache(id))
        return;
    const Mx4Page<D> lay(c.page_size());
    uint8_t* page = c.page(id, head, lay.bytes());
    const uint32_t t = (uint32_t)slot & (uint32_t)(c.page_size() - 1);
    const uint32_t wk = nan_k ? scaled_codes<EPL, true>(vk, ek) : scaled_codes<EPL, false>(vk, ek);
    const uint32_t wv = nan_v ? scaled_codes<EPL, true>(vv, ev) : scaled_codes<EPL, false>(vv, ev);
    if constexpr (EPL == 8)
        *(uint32_t*)(page + lay.k_row(t) + d / 2) = wk;
    else
        *(uint16_t*)(page + lay.k_row(t) + d / 2) = (uint16_t)wk;
    store_value_codes<D, EPL>(page, lay, t, d, wv);
    if (d % 32 == 0) {
        page[lay.k_scale(t) + d / 32] = (uint8_t)(ek + 127);
        page[lay.v_scale(t / 4, d / 32) + t % 4] = (uint8_t)(ev + 127);
    }
}

// ---- read back ---------------------------------------------------------------------
// Eight elements of a token's key and value per lane; bound by the bytes written (8191 tokens of
// 8 heads, D = 128, as bf16: 10 us).
template <int D>
__device__ __forceinline__ uint32_t value_codes8(const uint8_t* page, Mx4Page<D> lay, uint32_t t,
                                                 uint32_t d)
{
    constexpr uint32_t kPer = D / 16;
    const uint32_t u = t % 4 * (D / 32);
    if constexpr (D == 64)
        return *(const uint16_t*)(page + lay.v_quad(t / 4, d / kPer) + u) |
               (uint32_t) * (const uint16_t*)(page + lay.v_quad(t / 4, d / kPer + 1) + u) << 16;
    else
        return *(const uint32_t*)(page + lay.v_quad(t / 4, d / kPer) + u + d % kPer / 2);
}

typedef float v2f __attribute__((ext_vector_type(2)));

// The converter's results are exact while neither code 0.5 nor 6 leaves the normal range; scale
// bytes outside 2 .. 252 take fp4_value.
template <int OUT>
__device__ __forceinline__ void store_values8(void* dst, size_t at, uint32_t w, uint32_t scale)
{
    const bool usual = scale - 2u <= 250u;
    const float sc = __uint_as_float(scale << 23);
    if constexpr (OUT == GA_DTYPE_BF16) {
        v4i o = fp4_oct_bf16(w, sc);
        if (!usual) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                o[j] = (int)(f32_to_bf16(fp4_value(w >> (8 * j) & 15u, scale)) |
                             (uint32_t)f32_to_bf16(fp4_value(w >> (8 * j + 4) & 15u, scale)) << 16);
        }
        *(v4i*)((uint16_t*)dst + at) = o;
    } else {
        float x[8];
        static_for<4>([&](auto j) {
            const v2f y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, j);
            x[2 * j] = y[0];
            x[2 * j + 1] = y[1];
        });
        if (!usual) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = fp4_value(w >> (4 * j) & 15u, scale);
        }
        *(v4f*)((float*)dst + at) = (v4f){x[0], x[1], x[2], x[3]};
        *(v4f*)((float*)dst + at + 4) = (v4f){x[4], x[5], x[6], x[7]};
    }
}

template <int OUT, int D>
__global__ __launch_bounds__(256) void mx4_read_kernel(CacheView c,
                                                       const long long* __restrict__ slots,
                                                       int tokens, void* __restrict__ k,
                                                       void* __restrict__ v)
{
    const long long lane = (long long)blockIdx.x * 256 + threadIdx.x;
    const uint32_t row = (uint32_t)(lane / (D / 8));
    const uint32_t d = (uint32_t)(lane % (D / 8)) * 8;
    const uint32_t tok = row / (uint32_t)c.heads;
    if (tok >= (uint32_t)tokens)
        return;
    const int head = (int)(row - tok * (uint32_t)c.heads);
    const long long slot = slots[tok], id = slot >> c.log2p;
    const Mx4Page<D> lay(c.page_size());
    uint32_t wk = 0, wv = 0, sk = 0, sv = 0;
    if (c.in_cache(id)) {
        const uint8_t* page = c.page(id, head, lay.bytes());
        const uint32_t t = (uint32_t)slot & (uint32_t)(c.page_size() - 1);
        wk = *(const uint32_t*)(page + lay.k_row(t) + d / 2);
        wv = value_codes8<D>(page, lay, t, d);
        sk = page[lay.k_scale(t) + d / 32];
        sv = page[lay.v_scale(t / 4, d / 32) + t % 4];
    }
    const size_t at = (size_t)row * D + d;
    store_values8<OUT>(k, at, wk, sk);
    store_values8<OUT>(v, at, wv, sv);
}

// ---- eviction: which tokens stay --------------------------------------------------------
struct EvictArgs {
    ga_mx4_evict_args a;
    CacheView c;
};

__device__ __forceinline__ int evict_length(const EvictArgs& e, int b)
{
    const long long cap = min((long long)e.a.table_pages << e.c.log2p, (long long)e.a.width);
    return (int)min((long long)max(e.a.lens[b], 0), cap);
}

// Order of weights as unsigned integers: larger weight, larger key; both zeros
// alike, every NaN above everything.
__device__ __forceinline__ uint32_t weight_key(float x)
{
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u)
        return 0xFFFFFFFFu;
    if ((u & 0x7FFFFFFFu) == 0)
        return 0x80000000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The weight of a key (a zero without its sign, a NaN without its payload).
__device__ __forceinline__ float key_weight(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kSelBins = 2048;

// One workgroup per sequence and kv head. The (keep - recent)-th largest key is
// found by its digits (11, 11 and 10 bits, a histogram each), then every wave
// goes over its stretch of the weights twice: once to count what is above the key and
// equal to it, once to write the indices at the place that the stretches before it
// leave. No atomics on anything but the histograms' counts, so the result does
// not depend on an order. Bound by latency: a lane keeps its keys in registers, up to
// KEYS of them (65536 tokens), so that the weights are loaded once, all at the same time;
// longer sequences (KEYS 0) read them from the L2 in each of the five passes. One sequence of
// 5000 tokens (8 heads) 10 us; 16 of 16384 to 32768 26 us, on half of the CUs by then bound by the
// five passes' instructions (with a branch around each count 31; eight counts a bin instead
// of four 33).
template <int KEYS>
__global__ __launch_bounds__(kSelThreads) void mx4_select_kernel(EvictArgs e)
{
    __shared__ v4i hist[kSelBins]; // four counts of a bin, of every fourth lane each
    __shared__ int wave_sum[kSelWaves], wave_gt[kSelWaves], wave_eq[kSelWaves];
    __shared__ int found_bin, found_left;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = blockIdx.x / e.c.heads, head = blockIdx.x - b * e.c.heads;
    const int len = evict_length(e, b), keep = e.a.keep;
    const float* w = e.a.weights + b * e.a.stride_w_seq + head * e.a.stride_w_head;
    int* kept = e.a.kept + (size_t)blockIdx.x * keep;
    float* nw = e.a.new_weights + b * e.a.stride_new_seq + head * e.a.stride_new_head;
    const int new_len = min(len, keep);
    if (head == 0 && tid == 0)
        e.a.new_lens[b] = new_len;
    for (int j = new_len + tid; j < keep; j += kSelThreads)
        kept[j] = -1;
    for (int j = new_len + tid; j < e.a.new_width; j += kSelThreads)
        nw[j] = 0.0f;
    if (len <= keep) {
        for (int j = tid; j < len; j += kSelThreads) {
            kept[j] = j;
            nw[j] = w[j];
        }
        return;
    }
    const int old = len - e.a.recent, want = keep - e.a.recent; // old > want
    for (int j = tid; j < e.a.recent; j += kSelThreads) {
        kept[want + j] = old + j;
        nw[want + j] = w[old + j];
    }
    if (want == 0)
        return;
    // each wave's stretch of the tokens: lane's are lo + lane, 64 apart
    const Stretch part(old, wave, kSelWaves);
    const int lo = part.lo, hi = part.hi, rows = part.rows;
    uint32_t held[KEYS ? KEYS : 1];
    auto key_of = [&](int i) { // 0, which no weight has, past the stretch's end
        const int j = lo + 64 * i + lane;
        const uint32_t key = weight_key(w[j < hi ? j : 0]);
        return j < hi ? key : 0u;
    };
    if constexpr (KEYS > 0) {
        // a branch for 16 of them: loads under a branch are waited for inside it
        constexpr int kGroup = KEYS < 16 ? KEYS : 16;
#pragma unroll
        for (int i0 = 0; i0 < KEYS; i0 += kGroup)
            if (i0 < rows) {
#pragma unroll
                for (int i = i0; i < i0 + kGroup; i++)
                    held[i] = key_of(i);
            }
    }
    // f(token of the lane, its key) in the tokens' order
    auto each = [&](auto&& f) {
        if constexpr (KEYS > 0) {
#pragma unroll
            for (int i = 0; i < KEYS; i++)
                if (i < rows) // a register's number has to be known: no loop over them
                    f(lo + 64 * i + lane, held[i]);
        } else {
            for (int i = 0; i < rows; i++)
                f(lo + 64 * i + lane, key_of(i));
        }
    };
    uint32_t key_at = 0;
    int left = want; // of the keys that share key_at's digits so far
    static_for<3>([&](auto digit) {
        constexpr int kPass = decltype(digit)::value;
        constexpr int shift = kPass == 0 ? 21 : (kPass == 1 ? 10 : 0);
        constexpr int bits = kPass == 2 ? 10 : 11;
        constexpr uint32_t fixed = kPass == 0 ? 0u : ~0u << (shift + bits < 32 ? shift + bits : 0);
        for (int j = tid; j < kSelBins; j += kSelThreads)
            hist[j] = (v4i){0, 0, 0, 0};
        __syncthreads();
        // without a branch a key, which costs more than to count a 0; the zeros past the
        // stretch's end are below every key and never reached
        each([&](int, uint32_t key) {
            atomicAdd((int*)&hist[key >> shift & ((1u << bits) - 1u)] + (lane & 3),
                      ((key ^ key_at) & fixed) == 0 ? 1 : 0);
        });
        __syncthreads();
        // thread i holds bins top = 2047 - 2i and top - 1: keys above come first
        const int top = kSelBins - 1 - 2 * tid;
        const v4i h1 = hist[top], h0 = hist[top - 1];
        const int n1 = h1[0] + h1[1] + h1[2] + h1[3], n0 = h0[0] + h0[1] + h0[2] + h0[3];
        int sum = n1 + n0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(sum, o, 64);
            sum += lane >= o ? t : 0;
        }
        if (lane == 63)
            wave_sum[wave] = sum;
        __syncthreads();
        int before = sum - n1 - n0; // keys in bins above top
#pragma unroll
        for (int i = 0; i < kSelWaves; i++)
            before += i < wave ? wave_sum[i] : 0;
        if (before < left && left <= before + n1 + n0) {
            const bool upper = left <= before + n1;
            found_bin = upper ? top : top - 1;
            found_left = left - (upper ? before : before + n1);
        }
        __syncthreads();
        key_at |= (uint32_t)found_bin << shift;
        left = found_left;
    });
    int gt = 0, eq = 0;
    each([&](int, uint32_t key) {
        gt += __popcll(__builtin_amdgcn_ballot_w64(key > key_at));
        eq += __popcll(__builtin_amdgcn_ballot_w64(key == key_at));
    });
    if (lane == 0) {
        wave_gt[wave] = gt;
        wave_eq[wave] = eq;
    }
    __syncthreads();
    int at_gt = 0, at_eq = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; i++) {
        at_gt += i < wave ? wave_gt[i] : 0;
        at_eq += i < wave ? wave_eq[i] : 0;
    }
    int at = at_gt + min(at_eq, left);
    const uint64_t below = (1ull << lane) - 1ull;
    each([&](int j, uint32_t key) {
        const uint64_t eqs = __builtin_amdgcn_ballot_w64(key == key_at);
        const bool stays =
            key > key_at || (key == key_at && at_eq + __popcll(eqs & below) < left);
        const uint64_t stay = __builtin_amdgcn_ballot_w64(stays);
        if (stays) {
            const int to = at + __popcll(stay & below);
            kept[to] = j;
            nw[to] = key_weight(key);
        }
        at_eq += __popcll(eqs);
        at += __popcll(stay);
    });
}

// ---- eviction: moving them ---------------------------------------------------------------
// A workgroup moves 64 kept tokens of one head, at their new places in whole
// quads of four, so that a lane writes a value's pieces of four tokens, or their scales, at
// once; the reads are as scattered as the kept tokens are, and of a value's line only a
// quarter is its own. Bound by those lines: 16 sequences' 2048 tokens of 8 heads (D = 128) 34 us,
// 36 MB written and about 130 MB of lines touched.
constexpr int kMoveTokens = 64;

template <int D>
__global__ __launch_bounds__(256) void mx4_move_kernel(EvictArgs e, int blocks)
{
    constexpr int kPiece = D / 32; // code bytes of a token's value under one i; scale bytes of a token
    __shared__ const uint8_t* src_page[kMoveTokens];
    __shared__ uint8_t* dst_page[kMoveTokens / 4]; // of a quad
    __shared__ int src_at[kMoveTokens];
    const Mx4Page<D> lay(e.c.page_size());
    const int unit = blockIdx.x / blocks, first = (blockIdx.x - unit * blocks) * kMoveTokens;
    const int b = unit / e.c.heads, head = unit - b * e.c.heads;
    const int mask = e.c.page_size() - 1;
    const int n = min(min(evict_length(e, b), e.a.keep) - first, kMoveTokens);
    if (n <= 0)
        return;
    if (threadIdx.x < kMoveTokens) {
        const int i = threadIdx.x;
        const uint8_t* sp = nullptr;
        int at = 0;
        if (i < n) {
            const int t = e.a.kept[(size_t)unit * e.a.keep + first + i];
            const long long from = e.a.table[b * e.a.stride_table + (t >> e.c.log2p)];
            if (e.c.in_cache(from))
                sp = e.c.page(from, head, lay.bytes());
            at = t & mask;
        }
        src_page[i] = sp;
        src_at[i] = at;
        if (i % 4 == 0) {
            const int j = (first + i) >> e.c.log2p;
            const long long to =
                i < n && j < e.a.dst_pages ? e.a.dst_table[b * e.a.stride_dst_table + j] : -1;
            dst_page[i / 4] = e.c.in_cache(to) ? e.c.page(to, head, lay.bytes()) : nullptr;
        }
    }
    __syncthreads();
    // keys: 16 bytes a lane, then their scales; a token without a source becomes zeros
    for (int x = threadIdx.x; x < kMoveTokens * (D / 32); x += 256) {
        const int i = x / (D / 32), o = x % (D / 32) * 16;
        uint8_t* dst = dst_page[i / 4];
        if (!dst || i >= n)
            continue;
        v4i w = (v4i){0, 0, 0, 0};
        if (src_page[i])
            w = *(const v4i*)(src_page[i] + lay.k_row(src_at[i]) + o);
        *(v4i*)(dst + lay.k_row((first + i) & mask) + o) = w;
    }
    // values: the four tokens of a quad (those past the last become zeros)
    for (int x = threadIdx.x; x < kMoveTokens / 4 * 16; x += 256) {
        const int quad = x / 16, i = x % 16;
        uint8_t* dst = dst_page[quad];
        if (!dst)
            continue;
        dst += lay.v_quad(((first + 4 * quad) & mask) / 4, i);
        uint32_t w[4 * kPiece / 4] = {};
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int j = quad * 4 + u;
            if (!src_page[j])
                continue;
            const uint8_t* s = src_page[j] + lay.v_quad(src_at[j] / 4, i) + src_at[j] % 4 * kPiece;
            if constexpr (kPiece == 2) {
                w[u / 2] |= (uint32_t) * (const uint16_t*)s << (u % 2 * 16);
            } else if constexpr (kPiece == 4) {
                w[u] = *(const uint32_t*)s;
            } else {
                const uint2 y = *(const uint2*)s;
                w[2 * u] = y.x;
                w[2 * u + 1] = y.y;
            }
        }
        if constexpr (kPiece == 2) {
            *(uint2*)dst = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int o = 0; o < kPiece; o += 4)
                *(v4i*)(dst + 4 * o) =
                    (v4i){(int)w[o], (int)w[o + 1], (int)w[o + 2], (int)w[o + 3]};
        }
    }
    // scales: of a token's key, and of a block of a quad's values
    for (int x = threadIdx.x; x < kMoveTokens + kMoveTokens / 4 * kPiece; x += 256) {
        if (x < kMoveTokens) {
            uint8_t* dst = dst_page[x / 4];
            if (!dst || x >= n)
                continue;
            dst += lay.k_scale((first + x) & mask);
            const uint8_t* s = src_page[x] ? src_page[x] + lay.k_scale(src_at[x]) : nullptr;
            if constexpr (kPiece == 2)
                *(uint16_t*)dst = s ? *(const uint16_t*)s : 0;
            else if constexpr (kPiece == 4)
                *(uint32_t*)dst = s ? *(const uint32_t*)s : 0;
            else
                *(uint2*)dst = s ? *(const uint2*)s : make_uint2(0, 0);
        } else {
            const int quad = (x - kMoveTokens) / kPiece, blk = (x - kMoveTokens) % kPiece;
            uint8_t* dst = dst_page[quad];
            if (!dst)
                continue;
            uint32_t w = 0;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int j = quad * 4 + u;
                if (src_page[j])
                    w |= (uint32_t)src_page[j][lay.v_scale(src_at[j] / 4, blk) + src_at[j] % 4]
                         << (8 * u);
            }
            *(uint32_t*)(dst + lay.v_scale(((first + 4 * quad) & mask) / 4, blk)) = w;
        }
    }
}

ga_status mx4_cache_check(const ga_mx4_cache* c)
{
    if (!c || !c->pages)
        return fail(GA_ERR_ARG, "mx4 cache: null pages");
    const size_t bytes = ga_mx4_page_bytes(c->page_size, c->head_dim);
    if (!bytes)
        return fail(GA_ERR_SHAPE, "mx4 cache: head_dim must be 64, 128 or 256 and page_size 16, 32, "
                                  "64, 128 or 256");
    if (c->num_pages <= 0 || c->kv_heads <= 0)
        return fail(GA_ERR_ARG, "mx4 cache: num_pages and kv_heads must be positive");
    if ((uintptr_t)c->pages % 16 || c->stride_page % 16 ||
        c->stride_page < (long long)bytes * c->kv_heads)
        return fail(GA_ERR_ARG, "mx4 cache: pages must be 16-byte aligned, stride_page a multiple "
                                "of 16 and at least kv_heads pages' bytes");
    return GA_OK;
}

// f(std::integral_constant<int, D>) for the cache's head_dim.
template <class F>
static void with_dim(int d, F&& f)
{
    if (d == 64)
        f(std::integral_constant<int, 64>{});
    else if (d == 128)
        f(std::integral_constant<int, 128>{});
    else
        f(std::integral_constant<int, 256>{});
}

static bool aligned_rows(const void* p, long long row, long long head, int elems, int bytes)
{
    return (uintptr_t)p % bytes == 0 && row % elems == 0 && head % elems == 0;
}

} // namespace ga

using namespace ga;

extern "C" {

size_t ga_mx4_page_bytes(int page_size, int head_dim)
{
    const bool dim = head_dim == 64 || head_dim == 128 || head_dim == 256;
    const bool size = page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0;
    return dim && size ? (size_t)page_size * (size_t)(head_dim + head_dim / 16) : 0;
}

ga_status ga_mx4_append(const ga_mx4_cache* cache, const void* k, const void* v, int in_dtype,
                        int tokens, long long stride_k_row, long long stride_k_head,
                        long long stride_v_row, long long stride_v_head, const long long* slots,
                        int scale_rule, void* stream)
{
    if (const ga_status st = mx4_cache_check(cache))
        return st;
    if (in_dtype != GA_IN_F32 && in_dtype != GA_IN_BF16)
        return fail(GA_ERR_ARG, "mx4_append: input dtype must be GA_IN_F32 or GA_IN_BF16");
    if (tokens < 0 || scale_rule < 0 || scale_rule > 2)
        return fail(GA_ERR_ARG, "mx4_append: bad token count or scale rule");
    if (tokens == 0)
        return GA_OK;
    if (!k || !v || !slots)
        return fail(GA_ERR_ARG, "mx4_append: null pointer");
    const int least = in_dtype == GA_IN_F32 ? 16 : 8;
    if (!aligned_rows(k, stride_k_row, stride_k_head, 4, least) ||
        !aligned_rows(v, stride_v_row, stride_v_head, 4, least))
        return fail(GA_ERR_SHAPE, "mx4_append: k and v must be %d-byte aligned with strides that "
                                  "are multiples of 4", least);
    const bool wide = in_dtype == GA_IN_BF16 &&
                      aligned_rows(k, stride_k_row, stride_k_head, 8, 16) &&
                      aligned_rows(v, stride_v_row, stride_v_head, 8, 16);
    const long long rows = (long long)tokens * cache->kv_heads;
    const long long blocks = (rows * (cache->head_dim / (wide ? 8 : 4)) + 255) / 256;
    if (rows > 0x7FFFFFFFll || blocks > most_workgroups(256))
        return fail(GA_ERR_SHAPE, "mx4_append: too many tokens for one call");
    with_dim(cache->head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                               view_of(*cache), k, v, tokens, stride_k_row, stride_k_head,
                               stride_v_row, stride_v_head, slots, scale_rule);
        };
        if (in_dtype == GA_IN_F32)
            run(mx4_append_kernel<GA_IN_F32, 4, D>);
        else if (wide)
            run(mx4_append_kernel<GA_IN_BF16, 8, D>);
        else
            run(mx4_append_kernel<GA_IN_BF16, 4, D>);
    });
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

ga_status ga_mx4_read(const ga_mx4_cache* cache, const long long* slots, int tokens, void* k,
                      void* v, int out_dtype, void* stream)
{
    if (const ga_status st = mx4_cache_check(cache))
        return st;
    if (out_dtype != GA_DTYPE_F32 && out_dtype != GA_DTYPE_BF16)
        return fail(GA_ERR_ARG, "mx4_read: output dtype must be GA_DTYPE_F32 or GA_DTYPE_BF16");
    if (tokens < 0)
        return fail(GA_ERR_ARG, "mx4_read: bad token count");
    if (tokens == 0)
        return GA_OK;
    if (!slots || !k || !v || (uintptr_t)k % 16 || (uintptr_t)v % 16)
        return fail(GA_ERR_ARG, "mx4_read: k and v must be 16-byte aligned, nothing null");
    const long long rows = (long long)tokens * cache->kv_heads;
    const long long blocks = (rows * (cache->head_dim / 8) + 255) / 256;
    if (rows > 0x7FFFFFFFll || blocks > most_workgroups(256))
        return fail(GA_ERR_SHAPE, "mx4_read: too many tokens for one call");
    with_dim(cache->head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                               view_of(*cache), slots, tokens, k, v);
        };
        if (out_dtype == GA_DTYPE_F32)
            run(mx4_read_kernel<GA_DTYPE_F32, D>);
        else
            run(mx4_read_kernel<GA_DTYPE_BF16, D>);
    });
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

ga_status ga_mx4_evict(const ga_mx4_cache* cache, const ga_mx4_evict_args* args, void* stream)
{
    if (const ga_status st = mx4_cache_check(cache))
        return st;
    if (!args)
        return fail(GA_ERR_ARG, "mx4_evict: null arguments");
    const ga_mx4_evict_args& a = *args;
    if (a.keep <= 0 || a.recent < 0 || a.recent > a.keep)
        return fail(GA_ERR_ARG, "mx4_evict: keep must be positive and recent 0 .. keep");
    if (a.seqs < 0 || a.table_pages < 0 || a.dst_pages < 0 || a.width < 0 || a.new_width < a.keep)
        return fail(GA_ERR_ARG, "mx4_evict: negative size, or new_width below keep");
    if (a.width > GA_MX4_MAX_TOKENS || a.new_width > GA_MX4_MAX_TOKENS)
        return fail(GA_ERR_SHAPE, "mx4_evict: too many tokens for one call");
    if ((long long)a.dst_pages * cache->page_size < std::min(a.keep, a.width))
        return fail(GA_ERR_SHAPE, "mx4_evict: dst_table's pages hold fewer than keep tokens");
    if (a.seqs == 0)
        return GA_OK;
    if (!a.table || !a.lens || !a.dst_table || !a.weights || !a.kept || !a.new_lens ||
        !a.new_weights)
        return fail(GA_ERR_ARG, "mx4_evict: null pointer");
    const long long units = (long long)a.seqs * cache->kv_heads;
    const int blocks = (a.keep + kMoveTokens - 1) / kMoveTokens;
    if (units > most_workgroups(kSelThreads) || units * blocks > most_workgroups(256))
        return fail(GA_ERR_SHAPE, "mx4_evict: too many sequences for one call");
    const EvictArgs e{a, view_of(*cache)};
    // the most tokens that may be looked at decide whether a lane can hold its share
    const long long most = std::min<long long>((long long)a.table_pages * cache->page_size, a.width);
    if (most <= 8ll * kSelThreads)
        hipLaunchKernelGGL((mx4_select_kernel<8>), dim3((unsigned)units), dim3(kSelThreads), 0,
                           (hipStream_t)stream, e);
    else if (most <= 64ll * kSelThreads)
        hipLaunchKernelGGL((mx4_select_kernel<64>), dim3((unsigned)units), dim3(kSelThreads), 0,
                           (hipStream_t)stream, e);
    else
        hipLaunchKernelGGL((mx4_select_kernel<0>), dim3((unsigned)units), dim3(kSelThreads), 0,
                           (hipStream_t)stream, e);
    with_dim(cache->head_dim, [&](auto dim) {
        hipLaunchKernelGGL((mx4_move_kernel<decltype(dim)::value>), dim3((unsigned)(units * blocks)),
                           dim3(256), 0, (hipStream_t)stream, e, blocks);
    });
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

} // extern "C"

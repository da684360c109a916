// experts.hip -- layers of experts around their products: the choice of a token's experts
// (route), the map of rows (arrange), the gated activation that quantises for the second
// product (activate) and the weighted sum that ends the layer (combine). The products:
// gemm_experts.hip.
#include "ga_device.hpp"
#include "ga_experts.hpp"
#include "ga_internal.hpp"
#include "ga_quant.hpp"

#include <algorithm>

namespace ga {
namespace {

// ---- route ------------------------------------------------------------------------
// A wave has one token; lane l holds the experts l, l + 64, ... A choice is a maximum over the
// wave of keys made comparable as integers, then the lowest expert that has it.
//
// Keys with a bias are sums that 32 bits round; the choice is that of 64 bits. It is made in 32
// bits first, with a bound of what they are off by, and again in 64 where two keys that
// decide it lie within that bound (31 of 16384 random tokens): instructions bound
// this kernel, and exponentials and comparisons of 64 bits cost two to four times as many.
// 16384 tokens, 192 experts in 8 groups, sigmoid and bias: 64 bits throughout 25.4 us, so 17.3.

// Exchange between the lanes of a row of 16, then between rows: lane 63 has all.
template <class T, class Op>
__device__ __forceinline__ T wave_all(T a, const Op& op, T none)
{
    auto dpp = [&](T v, auto ctrl, auto rows) {
        return __builtin_bit_cast(
            T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                           decltype(ctrl)::value, decltype(rows)::value, 0xF,
                                           false));
    };
    using std::integral_constant;
    a = op(a, dpp(a, integral_constant<int, 0xB1>{}, integral_constant<int, 0xF>{}));  // xor 1
    a = op(a, dpp(a, integral_constant<int, 0x4E>{}, integral_constant<int, 0xF>{}));  // xor 2
    a = op(a, dpp(a, integral_constant<int, 0x141>{}, integral_constant<int, 0xF>{})); // half mirror
    a = op(a, dpp(a, integral_constant<int, 0x140>{}, integral_constant<int, 0xF>{})); // mirror
    a = op(a, dpp(a, integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{})); // row_bcast 15
    a = op(a, dpp(a, integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{})); // row_bcast 31
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, a), 63));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t a)
{
    return wave_all(a, [](uint32_t x, uint32_t y) { return max(x, y); }, 0u);
}
__device__ __forceinline__ float wave_max(float a)
{
    return wave_all(a, [](float x, float y) { return fmaxf(x, y); }, -__builtin_inff());
}
__device__ __forceinline__ float wave_sum(float a)
{
    return wave_all(a, [](float x, float y) { return x + y; }, 0.0f);
}
__device__ __forceinline__ double wave_sum(double a)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
        a += __shfl_xor(a, d, 64);
    return a;
}

// Integers in the order of the numbers, both zeros alike; 0 for what cannot be chosen.
__device__ __forceinline__ uint32_t ordered(float x)
{
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double x)
{
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ float unordered(uint32_t k)
{
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

constexpr int kRouteWaves = 4;
constexpr float kMinus = -__builtin_inff();

// What keys of scores are off by in 32 bits, apart from the rounding of score + bias: an exponential's
// argument, the exponential and the sum of up to 1024 of them, at most 2^-19 of a score in all,
// taken twice. (What is too wide here sends more tokens to 64 bits, what is too narrow would choose wrongly.)
constexpr float kScoreError = 0x1p-18f;

// A logit: -inf where it is not there (-inf, NaN), +inf as its type's largest finite value.
template <int IN>
__device__ __forceinline__ float logit_at(const void* p, long long i)
{
    const float x =
        IN == GA_IN_F32 ? ((const float*)p)[i] : bf16_to_f32(((const uint16_t*)p)[i]);
    return x > kMinus ? fminf(x, IN == GA_IN_F32 ? 0x1.FFFFFEp127f : 0x1.FEp127f) : kMinus;
}

template <int VPT>
struct RouteToken {
    float x[VPT];
    float largest;
    int lane;
};

// Steps of packed keys to 1: logits, exact, reach 16 down from the largest; scores with a bias 2,
// sums of two of them 4.
constexpr float kLogitSteps = 0x1p18f, kScoreSteps = 0x1p21f, kSumSteps = 0x1p20f;

// The weight of a chosen logit x before it is divided by the sum over the chosen ones, relative to the
// largest of them, `from`; without renormalising its score (sum: a softmax's).
__device__ __forceinline__ float weight_of(const ga_experts_route_args& a, float x, float from,
                                           float largest, float sum)
{
    if (a.scores == GA_EXPERTS_SOFTMAX)
        return a.renormalise ? expf(x - from) : expf(x - largest) / sum;
    const float e = fminf(x, 0.0f) - (a.renormalise ? fminf(from, 0.0f) : 0.0f);
    return expf(e) / (1.0f + expf(-fabsf(x)));
}

// By the hardware's exponential, also for the sum that divides a softmax's weights: its argument x log2(e)
// rounded to 24 bits is off by 1.25 |x| 2^-24 of a term, of the sum, where terms weigh by their size, by
// 1.25 ln(1024) 2^-24, with the exponential's own 2^-23 at most 11 2^-24; the sum's additions in fp32 (16
// a lane, 6 between lanes) can take twice that.
__device__ __forceinline__ float score_of(float x, bool softmax, float largest)
{
    return softmax ? __expf(x - largest) : __builtin_amdgcn_rcpf(1.0f + __expf(-x));
}

// A number and an index in one integer: of the larger number, of equal ones the lower index is the
// larger. Numbers from `top` (the largest) down to top - 2^22 / steps become steps, those below
// step 1; 0 is nothing.
__device__ __forceinline__ uint32_t packed(float x, float top, float steps, int index)
{
    const float d = 4194303.0f - (top - x) * steps;
    return (uint32_t)fmaxf(d, 1.0f) << 10 | (uint32_t)(1023 - index);
}
// Steps that numbers off by so many steps together have to be apart: those of the packing's own roundings
// more, at most all there are.
__device__ __forceinline__ uint32_t steps_apart(float off) { return 2 + (uint32_t)fminf(off, 4194303.0f); }
__device__ __forceinline__ int index_of(uint32_t key) { return 1023 - (int)(key & 1023u); }

// The two largest of a group's values, at its first lane.
template <class T>
__device__ __forceinline__ void two_largest(const ga_experts_route_args& a, const T* by, int lane,
                                            int shift, T& b1, T& b2)
{
    const int size = a.experts / a.groups;
    const int g = lane >> shift, sub = lane & ((1 << shift) - 1);
    b1 = b2 = (T)kMinus;
    if (g < a.groups)
        for (int i = sub; i < size; i += 1 << shift) {
            const T d = by[g * size + i];
            b2 = max(b2, min(b1, d));
            b1 = max(b1, d);
        }
    for (int d = 1; d < 1 << shift; d <<= 1) {
        const T o1 = __shfl_xor(b1, d, 64), o2 = __shfl_xor(b2, d, 64);
        b2 = max(min(b1, o1), max(b2, o2));
        b1 = max(b1, o1);
    }
}

// The value of a group in 32 bits. Two keys can have a sum below the least number, which may not
// become that of a group that is not there; values so far out are within what they can be off by, so that
// 64 bits decide.
__device__ __forceinline__ float group_value(const ga_experts_route_args& a, float b1, float b2)
{
    return a.group_rank == 2 && b2 > kMinus ? fmaxf(b1 + b2, -0x1.FFFFFEp127f) : b1;
}

// The groups that are kept, a bit at each one's first lane (group << shift), by their values.
template <class T>
__device__ __forceinline__ uint64_t kept_groups(const ga_experts_route_args& a, const T* by, int lane,
                                                int shift)
{
    T b1, b2;
    two_largest(a, by, lane, shift, b1, b2);
    const T none = (T)kMinus;
    const T value = a.group_rank == 2 && b2 > none ? b1 + b2 : b1;
    const int g = lane >> shift;
    int before = 0;
    for (int j = 0; j < a.groups; j++) {
        const T o = __shfl(value, j << shift, 64);
        before += o > value || (o == value && j < g);
    }
    return __builtin_amdgcn_ballot_w64(g < a.groups && (lane & ((1 << shift) - 1)) == 0 &&
                                       value > none && before < a.top_groups);
}

// The same one after the other by packed values; sure: no group left out is within `gap` steps of
// a kept one.
__device__ __forceinline__ uint64_t kept_groups_packed(const ga_experts_route_args& a,
                                                       const float* by, int lane, int shift,
                                                       float steps, uint32_t gap, bool& sure)
{
    float b1, b2;
    two_largest(a, by, lane, shift, b1, b2);
    const float value = group_value(a, b1, b2);
    const int g = lane >> shift;
    const bool there =
        g < a.groups && (lane & ((1 << shift) - 1)) == 0 && value > kMinus;
    const float top = unordered(wave_max(there ? ordered(value) : 0u));
    uint32_t key = there ? packed(value, top, steps, g) : 0u, last = 0;
    uint64_t kept = 0;
    for (int j = 0; j <= a.top_groups; j++) {
        const uint32_t best = wave_max(key);
        if (best == 0)
            break;
        if (j == a.top_groups) {
            sure &= (last >> 10) - (best >> 10) > gap;
            break;
        }
        kept |= 1ull << (index_of(best) << shift);
        key = key == best ? 0u : key;
        last = best;
    }
    sure &= top < __builtin_inff();
    return kept;
}

// Whether expert v * 64 + lane is in a kept group: e / size by a multiplication, exact for e and
// size up to 1024.
__device__ __forceinline__ bool in_kept(uint64_t kept, int shift, int size, int e)
{
    const uint32_t inv = ((1u << 20) + size - 1) / size;
    return kept >> ((((uint32_t)e * inv) >> 20) << shift) & 1;
}

// The experts of largest keys one after the other, choice j's expert in lane j. Keys of 64 bits, or
// (WIDE false) the first 32 alone.
template <int VPT, bool WIDE>
__device__ __forceinline__ int choose(int lane, uint32_t (&key)[VPT], uint32_t (&low)[VPT], int top)
{
    int id = -1;
    for (int j = 0; j < top; j++) {
        uint32_t best = key[0], second = 0;
#pragma unroll
        for (int v = 1; v < VPT; v++)
            best = max(best, key[v]);
        best = wave_max(best);
        if (best == 0)
            break;
        if constexpr (WIDE) {
#pragma unroll
            for (int v = 0; v < VPT; v++)
                second = key[v] == best ? max(second, low[v]) : second;
            second = wave_max(second);
        }
        bool found = false;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const uint64_t has =
                __builtin_amdgcn_ballot_w64(key[v] == best && (!WIDE || low[v] == second));
            if (!found && has != 0) {
                const int l = __builtin_ctzll(has);
                found = true;
                if (lane == l)
                    key[v] = low[v] = 0u;
                if (lane == j)
                    id = v * 64 + l;
            }
        }
    }
    return id;
}

// The same by packed keys. sure: consecutive ones, and the first that is left, are further apart
// than `gap` steps, so that they are in the order of what they stand for.
template <int VPT>
__device__ __forceinline__ int choose_packed(int lane, uint32_t (&key)[VPT], int top, uint32_t gap,
                                             bool& sure)
{
    int id = -1;
    uint32_t last = ~0u;
    for (int j = 0; j <= top; j++) {
        uint32_t best = key[0];
#pragma unroll
        for (int v = 1; v < VPT; v++)
            best = max(best, key[v]);
        best = wave_max(best);
        if (best == 0)
            break;
        sure &= j == 0 || (last >> 10) - (best >> 10) > gap;
        if (j == top)
            break;
#pragma unroll
        for (int v = 0; v < VPT; v++)
            key[v] = key[v] == best ? 0u : key[v];
        id = lane == j ? index_of(best) : id;
        last = best;
    }
    return id;
}

// The choice by keys of 64 bits.
template <int VPT>
__device__ __forceinline__ int choose64(const ga_experts_route_args& a, const RouteToken<VPT>& t,
                                        double* by, int shift)
{
    const bool softmax = a.scores == GA_EXPERTS_SOFTMAX;
    const int lane = t.lane, E = a.experts, size = E / a.groups;
    double score[VPT], sum = 0.0;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const double d = (double)t.x[v];
        score[v] = softmax ? (t.x[v] > kMinus ? exp(d - (double)t.largest) : 0.0)
                           : 1.0 / (1.0 + exp(-d));
        sum += score[v];
    }
    if (softmax) {
        sum = wave_sum(sum);
#pragma unroll
        for (int v = 0; v < VPT; v++)
            score[v] /= sum;
    }
    uint32_t key[VPT], low[VPT];
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const int e = v * 64 + lane;
        bool there = t.x[v] > kMinus;
        if (a.bias) {
            score[v] += e < E ? (double)a.bias[e] : 0.0;
            there = there && score[v] > (double)kMinus;
            const uint64_t u = ordered(score[v]);
            key[v] = there ? (uint32_t)(u >> 32) : 0u;
            low[v] = there ? (uint32_t)u : 0u;
        } else {
            key[v] = there ? ordered(t.x[v]) : 0u;
            low[v] = 0u;
        }
        // groups go by the largest key, without a bias a logit: scores of 64 bits can be
        // alike where logits differ; only the sum of two is one of scores
        if (!a.bias && a.group_rank == 1)
            score[v] = (double)t.x[v];
        if (!there)
            score[v] = (double)kMinus;
    }
    if (a.top_groups < a.groups) {
#pragma unroll
        for (int v = 0; v < VPT; v++)
            if (v * 64 + lane < E)
                by[v * 64 + lane] = score[v];
        wave_lds_fence();
        const uint64_t kept = kept_groups(a, by, lane, shift);
#pragma unroll
        for (int v = 0; v < VPT; v++)
            if (!in_kept(kept, shift, size, v * 64 + lane))
                key[v] = low[v] = 0u;
    }
    return a.bias ? choose<VPT, true>(lane, key, low, a.top)
                  : choose<VPT, false>(lane, key, low, a.top);
}

template <int VPT, int IN>
__global__ __launch_bounds__(64 * kRouteWaves) void route_kernel(ga_experts_route_args a)
{
    extern __shared__ double by_all[]; // [wave][expert], with groups
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long token = (long long)blockIdx.x * kRouteWaves + wave;
    if (token >= a.tokens)
        return;
    const int E = a.experts, size = E / a.groups;
    const bool softmax = a.scores == GA_EXPERTS_SOFTMAX, grouped = a.top_groups < a.groups;
    // scores decide, not the logits alone
    const bool by_group = grouped && a.group_rank == 2, by_score = a.bias || by_group;
    const int shift = 31 - __builtin_clz(64 / a.groups); // log2 of the lanes of a group

    const long long row = token * a.stride_logits;
    auto logit = [&](int e) { return logit_at<IN>(a.logits, row + e); };
    RouteToken<VPT> t;
    t.lane = lane;
    float top = kMinus;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const int e = v * 64 + lane;
        t.x[v] = e < E ? logit(min(e, E - 1)) : kMinus;
        top = fmaxf(top, t.x[v]);
    }
    t.largest = wave_max(top);

    // in 32 bits: the keys, and what the groups go by
    float key[VPT], by[VPT], sum = 0.0f;
#pragma unroll
    for (int v = 0; v < VPT; v++)
        key[v] = by[v] = t.x[v];
    if (by_score || (softmax && !a.renormalise)) {
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            by[v] = t.x[v] > kMinus ? score_of(t.x[v], softmax, t.largest) : 0.0f;
            sum += by[v];
        }
        sum = wave_sum(sum);
    }
    // the steps of packed keys, and what two keys can be off by
    float steps = kLogitSteps, off = 0.0f;
    if (by_score) {
        const float scale = softmax ? 1.0f / sum : 1.0f;
        float most = 0.0f; // the largest |score + bias|
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            float s = by[v] * scale;
            if (a.bias) {
                s += a.bias[min(v * 64 + lane, E - 1)];
                key[v] = t.x[v] > kMinus && s > kMinus ? s : kMinus;
                s = key[v];
                most = s > kMinus ? fmaxf(most, fabsf(s)) : most;
            }
            by[v] = t.x[v] > kMinus ? s : kMinus;
        }
        most = a.bias ? wave_max(most) : 1.0f;
        off = 2.0f * (kScoreError + 0x1p-23f * most);
        if (a.bias)
            steps = kScoreSteps;
    } else {
#pragma unroll
        for (int v = 0; v < VPT; v++)
            by[v] = t.x[v];
    }

    bool sure = true;
    uint64_t kept = ~0ull;
    double* lds = by_all + wave * E;
    if (grouped) {
        float* f = (float*)lds;
#pragma unroll
        for (int v = 0; v < VPT; v++)
            if (v * 64 + lane < E)
                f[v * 64 + lane] = by[v];
        wave_lds_fence();
        const float gsteps = by_score ? kSumSteps : steps; // sums are off by twice as much
        kept = kept_groups_packed(a, f, lane, shift, gsteps, steps_apart(2.0f * off * gsteps),
                                  sure);
        wave_lds_fence(); // read before 64 bits are written there
#pragma unroll
        for (int v = 0; v < VPT; v++)
            if (!in_kept(kept, shift, size, v * 64 + lane))
                key[v] = kMinus;
    }
    int id = -1;
    if (sure) {
        float best = kMinus;
#pragma unroll
        for (int v = 0; v < VPT; v++)
            best = fmaxf(best, key[v]);
        best = wave_max(best);
        uint32_t pack[VPT];
        const bool bf16 = IN == GA_IN_BF16 && !a.bias; // 16 bits and the index hold all of it
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const int e = v * 64 + lane;
            pack[v] = !(key[v] > kMinus) ? 0u
                      : bf16             ? (ordered(key[v]) >> 16) << 10 | (uint32_t)(1023 - e)
                                         : packed(key[v], best, steps, e);
        }
        sure = best < __builtin_inff();
        bool apart = true;
        id = choose_packed<VPT>(lane, pack, a.top, steps_apart(off * steps), apart);
        sure &= bf16 || apart;
    }
    if (!sure)
        id = choose64(a, t, lds, shift);

    // weights: each relative to the largest of the chosen logits, which so cancels
    const float xi = id >= 0 ? logit(id) : kMinus;
    const float from = wave_max(xi);
    float w = id >= 0 ? weight_of(a, xi, from, t.largest, sum) : 0.0f;
    if (a.renormalise) {
        const float all = wave_sum(w);
        w = id >= 0 ? w / all : 0.0f;
    }
    if (lane < a.top) {
        a.ids[token * a.top + lane] = id;
        a.weights[token * a.top + lane] = w * a.scale;
    }
}

// ---- route, four tokens a wave -----------------------------------------------------------
// Up to 256 experts, 16 groups and 16 choices: a token has a row of 16 lanes, runs of four experts
// each (lane r the experts 64 c + 4 r + i), so that the reductions, which take as many instructions
// for one token as for four, are shared. Tokens that 32 bits do not decide are gone over again, one
// at a time, by the whole wave.
template <class T, class Op>
__device__ __forceinline__ T row_all(T a, const Op& op)
{
    auto dpp = [](T v, auto ctrl) {
        return __builtin_bit_cast(
            T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF,
                                           0xF, false));
    };
    a = op(a, dpp(a, std::integral_constant<int, 0xB1>{}));  // xor 1
    a = op(a, dpp(a, std::integral_constant<int, 0x4E>{}));  // xor 2
    a = op(a, dpp(a, std::integral_constant<int, 0x141>{})); // half mirror
    return op(a, dpp(a, std::integral_constant<int, 0x140>{})); // mirror
}
__device__ __forceinline__ uint32_t row_max(uint32_t a)
{
    return row_all(a, [](uint32_t x, uint32_t y) { return max(x, y); });
}
__device__ __forceinline__ float row_max(float a)
{
    return row_all(a, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float row_sum(float a)
{
    return row_all(a, [](float x, float y) { return x + y; });
}

template <int C, int IN>
__global__ __launch_bounds__(64 * kRouteWaves) void route_rows_kernel(ga_experts_route_args a,
                                                                      int vector)
{
    constexpr int VPT = 4 * C;
    extern __shared__ double by_all[]; // [wave][2 E], with groups
    const int lane = threadIdx.x & 63, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long first = ((long long)blockIdx.x * kRouteWaves + wave) * 4;
    if (first >= a.tokens)
        return;
    const long long token = min(first + (lane >> 4), (long long)a.tokens - 1);
    const int E = a.experts, size = E / a.groups;
    const bool softmax = a.scores == GA_EXPERTS_SOFTMAX, grouped = a.top_groups < a.groups;
    const bool by_score = a.bias || (grouped && a.group_rank == 2);

    const long long row = token * a.stride_logits;
    float x[VPT], largest = kMinus;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = c * 64 + r * 4;
        if (vector) { // E a multiple of 4, rows aligned
            const long long f = row + min(e, E - 4);
            const float none = kMinus;
            if constexpr (IN == GA_IN_F32) {
                const v4f d = *(const v4f*)((const float*)a.logits + f);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    x[4 * c + i] = e < E && d[i] > none ? fminf(d[i], 0x1.FFFFFEp127f) : none;
            } else {
                const uint2 d = *(const uint2*)((const uint16_t*)a.logits + f);
                const uint32_t u[4] = {d.x << 16, d.x & 0xFFFF0000u, d.y << 16, d.y & 0xFFFF0000u};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float y = __uint_as_float(u[i]);
                    x[4 * c + i] = e < E && y > none ? fminf(y, 0x1.FEp127f) : none;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                x[4 * c + i] =
                    e + i < E ? logit_at<IN>(a.logits, row + min(e + i, E - 1)) : kMinus;
        }
    }
#pragma unroll
    for (int v = 0; v < VPT; v++)
        largest = fmaxf(largest, x[v]);
    largest = row_max(largest);

    float key[VPT], by[VPT], sum = 0.0f;
#pragma unroll
    for (int v = 0; v < VPT; v++)
        key[v] = by[v] = x[v];
    if (by_score || (softmax && !a.renormalise)) {
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            by[v] = x[v] > kMinus ? score_of(x[v], softmax, largest) : 0.0f;
            sum += by[v];
        }
        sum = row_sum(sum);
    }
    float steps = kLogitSteps, off = 0.0f;
    if (by_score) {
        const float scale = softmax ? 1.0f / sum : 1.0f;
        float most = 0.0f;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            float s = by[v] * scale;
            if (a.bias) {
                s += a.bias[min(v / 4 * 64 + r * 4 + v % 4, E - 1)];
                key[v] = x[v] > kMinus && s > kMinus ? s : kMinus;
                s = key[v];
                most = s > kMinus ? fmaxf(most, fabsf(s)) : most;
            }
            by[v] = x[v] > kMinus ? s : kMinus;
        }
        most = a.bias ? row_max(most) : 1.0f;
        off = 2.0f * (kScoreError + 0x1p-23f * most);
        if (a.bias)
            steps = kScoreSteps;
    } else {
#pragma unroll
        for (int v = 0; v < VPT; v++)
            by[v] = x[v];
    }

    bool sure = true;
    double* lds = by_all + (size_t)wave * 2 * E;
    if (grouped) {
        float* f = (float*)lds + (lane >> 4) * E;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const int e = v / 4 * 64 + r * 4 + v % 4;
            if (e < E)
                f[e] = by[v];
        }
        wave_lds_fence();
        const int shift = 31 - __builtin_clz(16 / a.groups); // log2 of the lanes of a group
        float b1, b2;
        two_largest(a, f, r, shift, b1, b2);
        const float value = group_value(a, b1, b2);
        const int g = r >> shift;
        const bool leads = g < a.groups && (r & ((1 << shift) - 1)) == 0 && value > kMinus;
        const float top = row_max(leads ? value : kMinus);
        const float gsteps = by_score ? kSumSteps : steps;
        const uint32_t gap = steps_apart(2.0f * off * gsteps);
        uint32_t gkey = leads ? packed(value, top, gsteps, g) : 0u, last = 0, kept = 0;
        for (int j = 0; j <= a.top_groups; j++) {
            const uint32_t best = row_max(gkey);
            if (j == a.top_groups)
                sure &= best == 0 || (last >> 10) - (best >> 10) > gap;
            else if (best != 0)
                kept |= 1u << index_of(best);
            gkey = gkey == best ? 0u : gkey;
            last = best;
        }
        sure &= top < __builtin_inff();
        // e / size by a multiplication, exact for e and size up to 1024; a run's at once where it can be
        const uint32_t inv = ((1u << 20) + size - 1) / size;
        if (size % 4 == 0) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                const bool in = kept >> (((uint32_t)(c * 64 + r * 4) * inv) >> 20) & 1;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    key[4 * c + i] = in ? key[4 * c + i] : kMinus;
            }
        } else {
#pragma unroll
            for (int v = 0; v < VPT; v++) {
                const uint32_t e = v / 4 * 64 + r * 4 + v % 4;
                if (!(kept >> ((e * inv) >> 20) & 1))
                    key[v] = kMinus;
            }
        }
    }

    float best_key = kMinus;
#pragma unroll
    for (int v = 0; v < VPT; v++)
        best_key = fmaxf(best_key, key[v]);
    best_key = row_max(best_key);
    const bool bf16 = IN == GA_IN_BF16 && !a.bias; // 16 bits and the index hold all of it
    uint32_t pack[VPT];
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const int e = v / 4 * 64 + r * 4 + v % 4;
        pack[v] = !(key[v] > kMinus) ? 0u
                  : bf16             ? (ordered(key[v]) >> 16) << 10 | (uint32_t)(1023 - e)
                                     : packed(key[v], best_key, steps, e);
    }
    // The next key after `last` is last + the largest of (key - last) mod 2^32: of keys below last,
    // which wrap, the largest is the nearest, and any of them is above those that do not wrap. So
    // nothing has to be taken out.
    const uint32_t gap = steps_apart(off * steps);
    bool apart = true;
    uint32_t last = 0;
    int id = -1;
    for (int j = 0; j <= a.top; j++) {
        uint32_t best = pack[0] - last;
#pragma unroll
        for (int v = 1; v < VPT; v++)
            best = max(best, pack[v] - last);
        best = row_max(best) + last;
        best = j > 0 && best >= last ? 0u : best; // none is left
        apart &= j == 0 || best == 0 || (last >> 10) - (best >> 10) > gap;
        if (j == a.top)
            break;
        id = r == j && best != 0 ? index_of(best) : id;
        last = best;
    }
    sure &= (bf16 || apart) && best_key < __builtin_inff();

    for (uint64_t again = __builtin_amdgcn_ballot_w64(!sure); again;) {
        const int lead = __builtin_ctzll(again) & ~15; // of the token's lanes
        again &= ~(0xFFFFull << lead);
        RouteToken<C> t;
        t.lane = lane;
        t.largest = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(largest), lead));
        const long long at = min(first + lead / 16, (long long)a.tokens - 1) * a.stride_logits;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int e = c * 64 + lane;
            t.x[c] = e < E ? logit_at<IN>(a.logits, at + min(e, E - 1)) : kMinus;
        }
        if (grouped)
            wave_lds_fence(); // what was there has been read
        const int id64 = choose64(a, t, lds, 31 - __builtin_clz(64 / a.groups));
        const int mine = __shfl(id64, r, 64);
        if ((lane & ~15) == lead)
            id = mine;
    }

    // weights: each relative to the largest of the chosen logits, which so cancels
    const float xi = id >= 0 ? logit_at<IN>(a.logits, row + id) : kMinus;
    const float from = row_max(xi);
    float w = id >= 0 ? weight_of(a, xi, from, largest, sum) : 0.0f;
    if (a.renormalise) {
        const float all = row_sum(w);
        w = id >= 0 ? w / all : 0.0f;
    }
    if (r < a.top && first + (lane >> 4) < a.tokens) {
        a.ids[token * a.top + r] = id;
        a.weights[token * a.top + r] = w * a.scale;
    }
}

template <int IN>
void launch_route(const ga_experts_route_args& a, hipStream_t st)
{
    const int v = (a.experts + 63) / 64;
    const bool grouped = a.top_groups < a.groups;
    if (v <= 4 && a.groups <= 16 && a.top <= 16) {
        const int el = IN == GA_IN_F32 ? 4 : 2;
        const int vector = a.experts % 4 == 0 && (uintptr_t)a.logits % (4 * el) == 0 &&
                           (a.tokens == 1 || a.stride_logits % 4 == 0);
        const dim3 grid((unsigned)((a.tokens + 4ll * kRouteWaves - 1) / (4 * kRouteWaves)));
        const size_t lds = grouped ? 2 * sizeof(double) * kRouteWaves * a.experts : 0;
        auto go = [&](auto C) {
            hipLaunchKernelGGL((route_rows_kernel<decltype(C)::value, IN>), grid,
                               dim3(64 * kRouteWaves), lds, st, a, vector);
        };
        v == 1   ? go(std::integral_constant<int, 1>{})
        : v == 2 ? go(std::integral_constant<int, 2>{})
        : v == 3 ? go(std::integral_constant<int, 3>{})
                 : go(std::integral_constant<int, 4>{});
        return;
    }
    const dim3 grid((unsigned)((a.tokens + (long long)kRouteWaves - 1) / kRouteWaves));
    const size_t lds = grouped ? sizeof(double) * kRouteWaves * a.experts : 0;
    auto go = [&](auto V) {
        hipLaunchKernelGGL((route_kernel<decltype(V)::value, IN>), grid, dim3(64 * kRouteWaves), lds,
                           st, a);
    };
    v <= 4   ? go(std::integral_constant<int, 4>{})
    : v <= 8 ? go(std::integral_constant<int, 8>{})
             : go(std::integral_constant<int, 16>{});
}

// ---- arrange ----------------------------------------------------------------------
// A workgroup has one expert and goes over all ids: those of smaller experts give its first row,
// its own are listed by each wave, which has a run of the pairs, and written in order once the waves
// before are known. No atomics: the same ids give the same rows. Every expert goes over every id; not
// the loads bound it (as long if they all hit L1) but the instructions: 98304 pairs of 192 experts
// 15.5 us, of which an empty launch takes 2.5, the comparisons 4, listing what is found 3, writing
// it 4; 8 pairs 3.4 us. Bits kept for 256 pairs at a time and gone over by a thread each took 42 us
// with a load in flight, 18 with 32.
constexpr int kArrangeList = 512; // a wave's own pairs that LDS holds; more are looked for again
constexpr int kAhead = 4;         // blocks of 256 pairs whose loads are in flight

template <int NT>
__global__ __launch_bounds__(NT) void arrange_kernel(const int* __restrict__ ids, int pairs,
                                                     int top, int experts, int first,
                                                     int* __restrict__ starts,
                                                     int* __restrict__ row_tokens,
                                                     int* __restrict__ place)
{
    constexpr int NW = NT / 64;
    __shared__ int lists[NW][kArrangeList];
    __shared__ int part[2][NW];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int me = blockIdx.x;
    const uint32_t mine = (uint32_t)first + me;
    const int blocks = (int)(((long long)pairs + 255) / 256);
    const int per = (blocks + NW - 1) / NW;
    const int b0 = min(blocks, wave * per), b1 = min(blocks, b0 + per);
    int* list = lists[wave];

    // pair 64 i + lane of a block is a lane's i-th; those behind the last are nobody's
    auto load = [&](int b, uint32_t (&e)[4]) {
        const int* p = ids + (size_t)b * 256 + lane;
        if ((long long)b * 256 + 256 <= pairs) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                e[i] = (uint32_t)p[i * 64];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                e[i] = (long long)b * 256 + i * 64 + lane < pairs ? (uint32_t)p[i * 64] : ~0u;
        }
    };
    // this wave's own pairs in order, to take(pair, its number); the pairs of smaller experts
    int less = 0, count = 0; // uniform
    auto pass = [&](auto&& take) {
        less = count = 0;
        for (int b = b0; b < b1; b += kAhead) {
            uint32_t e[kAhead][4];
#pragma unroll
            for (int u = 0; u < kAhead; u++)
                load(min(b + u, b1 - 1), e[u]);
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                if (b + u >= b1)
                    break;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    less += __builtin_popcountll(__builtin_amdgcn_ballot_w64(e[u][i] < mine));
                    if (first > 0)
                        less -= __builtin_popcountll(
                            __builtin_amdgcn_ballot_w64(e[u][i] < (uint32_t)first));
                    const uint64_t has = __builtin_amdgcn_ballot_w64(e[u][i] == mine);
                    if (has != 0) {
                        if (e[u][i] == mine)
                            take((b + u) * 256 + i * 64 + lane,
                                 count + (int)__builtin_amdgcn_mbcnt_hi(
                                             (uint32_t)(has >> 32),
                                             __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0)));
                        count += __builtin_popcountll(has);
                    }
                }
            }
        }
    };
    pass([&](int p, int k) {
        if (k < kArrangeList)
            list[k] = p;
    });
    if (lane == 0) {
        part[0][wave] = less;
        part[1][wave] = count;
    }
    // choices that are left out: every workgroup looks at some blocks
    for (int b = me + wave * experts; b < blocks; b += experts * NW) {
        uint32_t e[4];
        load(b, e);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const long long p = (long long)b * 256 + i * 64 + lane;
            if (p < pairs && e[i] - (uint32_t)first >= (uint32_t)experts)
                place[p] = -1;
        }
    }
    __syncthreads();
    int start = 0, base = 0, end = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        start += part[0][i];
        base += i < wave ? part[1][i] : 0;
        end += part[1][i];
    }
    base += start;
    end += start;
    if (threadIdx.x == 0)
        starts[me] = start;
    auto put = [&](int p, int k) {
        row_tokens[base + k] = p / top;
        place[p] = base + k;
    };
    if (count <= kArrangeList) {
        for (int k = lane; k < count; k += 64)
            put(list[k], k);
    } else {
        pass(put);
    }
    if (me == experts - 1) {
        if (threadIdx.x == 0)
            starts[experts] = end;
        for (long long r = (long long)end + threadIdx.x; r < pairs; r += NT) // nobody's rows
            row_tokens[r] = -1;
    }
}

// ---- activate ---------------------------------------------------------------------
// A workgroup has kActRows rows of kActBlocks blocks of 128, a wave the blocks of a row at a time:
// sixteen lanes a block, eight elements of gate and up each, all loads before the first use. The
// scales, which lie row by row within a block, go through LDS. With the library's exponential and a
// division instructions bound the kernel, 65536 rows of 2048 from bf16 167 us; with the hardware's,
// made as exact, HBM does, 125 to 130 us. Eight rows a workgroup took as long.
constexpr int kActBlocks = 4;
constexpr int kActRows = 16;

template <int IN>
__device__ __forceinline__ void load8(const void* x, size_t i, float (&v)[8])
{
    if constexpr (IN == GA_IN_F32) {
        const v4f_any* p = (const v4f_any*)((const float*)x + i);
        const v4f a = p[0], b = p[1];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = a[j];
            v[4 + j] = b[j];
        }
    } else {
        const v4i a = *(const v4i_any*)((const uint16_t*)x + i);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[2 * j] = __uint_as_float((uint32_t)a[j] << 16);
            v[2 * j + 1] = __uint_as_float((uint32_t)a[j] & 0xFFFF0000u);
        }
    }
}

// g / (1 + exp(-g)) for g from -87 on, off by at most 2^-21.4 of itself (the hardware's exponential
// 2^-23, four roundings): the exponential's argument in two parts, a Newton step for the
// reciprocal. +inf gives itself.
__device__ __forceinline__ float gated(float g)
{
    constexpr float kLog2e = 0x1.715476p+0f, kLess = 0x1.4ae0c0p-26f; // to fp32, and what it leaves
    const float x = -__builtin_amdgcn_fmed3f(g, -88.6f, 200.0f); // beyond, 1 / (1 + exp) is 0 or 1
    const float t = x * kLog2e;
    const float rest = fmaf(x, kLess, fmaf(x, kLog2e, -t));
    float e = __builtin_amdgcn_exp2f(t);
    e = fmaf(e, rest * 0x1.62e430p-1f, e); // 2^rest = 1 + rest ln 2
    const float d = 1.0f + e;
    float r = __builtin_amdgcn_rcpf(d);
    r = fmaf(fmaf(-d, r, 1.0f), r, r);
    return g * r;
}

// The same for g below -87, where 1 / (1 + exp(-g)), exp(g) there, is denormal though the result is not:
// exp(g + 20), of which the argument is exact, and the rest behind the product. Denormal from g =
// -91.8 down, zero from -108.7; -inf gives NaN.
constexpr float kFar = -87.0f;

__device__ __forceinline__ float gated_far(float g)
{
    return g * expf(g + 20.0f) * 0x1.1b4866p-29f; // exp(-20)
}

template <int IN>
__global__ __launch_bounds__(256) void activate_kernel(const void* __restrict__ x, int rows,
                                                       int inner, long long stride_x,
                                                       uint8_t* __restrict__ q, long long stride_q,
                                                       float* __restrict__ scales,
                                                       long long stride_scales,
                                                       const int* __restrict__ limit, int parts)
{
    constexpr int U = kActRows / 4;
    __shared__ float s_of[kActBlocks][kActRows];
    const int live = limit ? min(rows, max(0, *limit)) : rows;
    const int g0 = blockIdx.x % parts * kActBlocks;
    const long long r0 = (long long)(blockIdx.x / parts) * kActRows;
    if (r0 >= live)
        return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = g0 + (lane >> 4), sub = lane & 15;
    const int gc = min(g, inner / 128 - 1); // blocks and rows past the last: the last again
    float gate[U][8], up[U][8];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long long r = min(r0 + u * 4 + wave, (long long)live - 1);
        const size_t at = (size_t)r * stride_x + gc * 128 + sub * 8;
        load8<IN>(x, at, gate[u]);
        load8<IN>(x, at + inner, up[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long long r = r0 + u * 4 + wave;
        float y[8];
        float least = gate[u][0];
#pragma unroll
        for (int j = 1; j < 8; j++)
            least = fminf(least, gate[u][j]);
#pragma unroll
        for (int j = 0; j < 8; j++)
            y[j] = gated(gate[u][j]);
        if (__builtin_amdgcn_ballot_w64(least < kFar) != 0)
#pragma unroll
            for (int j = 0; j < 8; j++)
                y[j] = gate[u][j] < kFar ? gated_far(gate[u][j]) : y[j];
#pragma unroll
        for (int j = 0; j < 8; j++)
            y[j] *= up[u][j];
        bool nan;
        const float s = ds_scale(__uint_as_float(block_amax<16, 8>(y, nan)));
        const ScaleDiv d(s);
        const bool nan_rule = nan || __builtin_amdgcn_ballot_w64(!d.fast) != 0;
        if (sub == 0)
            s_of[lane >> 4][u * 4 + wave] = s;
        if (r >= live || g != gc)
            continue;
        uint8_t* dst = q + (size_t)r * stride_q + g * 128 + sub * 8;
        if (nan_rule)
            fp8_store_codes<true>(d, y, dst);
        else
            fp8_store_codes<false>(d, y, dst);
    }
    __syncthreads();
    const int b = threadIdx.x / kActRows, m = threadIdx.x % kActRows;
    if (b < kActBlocks && g0 + b < inner / 128 && r0 + m < live)
        scales[(size_t)(g0 + b) * stride_scales + r0 + m] = s_of[b][m];
}

// ---- combine ----------------------------------------------------------------------
// A thread has eight elements of a token and adds up its rows', eight rows' loads at a time; the
// last elements of a row that are fewer go one by one. HBM bounds it: 8191 tokens x 8 rows of 4096
// 119 us, 5.1 TB/s.
template <int OUT>
__global__ __launch_bounds__(256) void combine_kernel(const uint16_t* __restrict__ y, int rows,
                                                      int n, long long stride_y,
                                                      const int* __restrict__ place,
                                                      const float* __restrict__ weights, int top,
                                                      void* __restrict__ out, long long stride_out,
                                                      int parts)
{
    const int t = blockIdx.x / parts;
    const int c = ((blockIdx.x % parts) * 256 + threadIdx.x) * 8;
    if (c >= n)
        return;
    const int here = min(8, n - c);
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        acc[i] = 0.0f;
    constexpr int B = 8;
    for (int j0 = 0; j0 < top; j0 += B) {
        v4i raw[B];
        float w[B];
        bool ok[B];
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int j = min(j0 + b, top - 1);
            const int r = place[(size_t)t * top + j];
            ok[b] = j0 + b < top && r >= 0 && r < rows;
            w[b] = weights[(size_t)t * top + j];
            const uint16_t* p = y + (size_t)(ok[b] ? r : 0) * stride_y + c;
            if (here == 8) {
                raw[b] = *(const v4i_any*)p;
            } else {
                raw[b] = (v4i){0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 7; i++)
                    if (i < here)
                        raw[b][i / 2] |= (int)((uint32_t)p[i] << (i % 2 * 16));
            }
        }
#pragma unroll
        for (int b = 0; b < B; b++)
            if (ok[b])
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t u = (uint32_t)raw[b][i / 2];
                    acc[i] = fmaf(w[b], __uint_as_float(i & 1 ? u & 0xFFFF0000u : u << 16), acc[i]);
                }
    }
    const size_t o = (size_t)t * stride_out + c;
    if constexpr (OUT == GA_DTYPE_F32) {
        float* p = (float*)out + o;
        if (here == 8) {
            *(v4f_any*)p = (v4f){acc[0], acc[1], acc[2], acc[3]};
            *(v4f_any*)(p + 4) = (v4f){acc[4], acc[5], acc[6], acc[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 7; i++)
                if (i < here)
                    p[i] = acc[i];
        }
    } else {
        uint16_t* p = (uint16_t*)out + o;
        if (here == 8) {
            v4i d;
#pragma unroll
            for (int i = 0; i < 4; i++)
                d[i] = (int)((uint32_t)f32_to_bf16(acc[2 * i]) |
                             ((uint32_t)f32_to_bf16(acc[2 * i + 1]) << 16));
            *(v4i_any*)p = d;
        } else {
#pragma unroll
            for (int i = 0; i < 7; i++)
                if (i < here)
                    p[i] = f32_to_bf16(acc[i]);
        }
    }
}

} // namespace
} // namespace ga

using namespace ga;

extern "C" {

ga_status ga_experts_route(const ga_experts_route_args* args, void* stream)
{
    if (!args)
        return fail(GA_ERR_ARG, "experts_route: null argument");
    const ga_experts_route_args& a = *args;
    if (a.in_dtype != GA_IN_F32 && a.in_dtype != GA_IN_BF16)
        return fail(GA_ERR_ARG, "experts_route: in_dtype must be GA_IN_F32 or GA_IN_BF16");
    if (a.scores != GA_EXPERTS_SOFTMAX && a.scores != GA_EXPERTS_SIGMOID)
        return fail(GA_ERR_ARG, "experts_route: scores must be GA_EXPERTS_SOFTMAX or _SIGMOID");
    if (a.tokens < 0 || a.experts <= 0 || a.top <= 0 || a.groups <= 0 || a.top_groups <= 0 ||
        a.top_groups > a.groups || (a.group_rank != 1 && a.group_rank != 2))
        return fail(GA_ERR_ARG, "experts_route: bad count (groups %d, top_groups %d, group_rank %d)",
                    a.groups, a.top_groups, a.group_rank);
    if (a.experts > GA_EXPERTS_MAX || a.top > GA_EXPERTS_MAX_TOP ||
        a.groups > GA_EXPERTS_MAX_GROUPS)
        return fail(GA_ERR_SHAPE, "experts_route: more than %d experts, %d choices or %d groups",
                    GA_EXPERTS_MAX, GA_EXPERTS_MAX_TOP, GA_EXPERTS_MAX_GROUPS);
    if (a.experts % a.groups || a.top > a.experts / a.groups * a.top_groups)
        return fail(GA_ERR_SHAPE, "experts_route: %d experts in %d groups, %d of %d groups' chosen",
                    a.experts, a.groups, a.top, a.top_groups);
    if (!(a.scale - a.scale == 0.0f))
        return fail(GA_ERR_ARG, "experts_route: scale must be finite");
    if (a.tokens == 0)
        return GA_OK;
    if (!a.logits || !a.ids || !a.weights)
        return fail(GA_ERR_ARG, "experts_route: null pointer");
    if (a.stride_logits < (a.tokens > 1 ? a.experts : 0))
        return fail(GA_ERR_SHAPE, "experts_route: stride_logits must be >= experts");
    hipStream_t st = (hipStream_t)stream;
    a.in_dtype == GA_IN_F32 ? launch_route<GA_IN_F32>(a, st) : launch_route<GA_IN_BF16>(a, st);
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

ga_status ga_experts_arrange(const int* ids, int tokens, int top, int experts, int first,
                             int* starts, int* row_tokens, int* place, void* stream)
{
    if (tokens < 0 || top <= 0 || experts <= 0 || first < 0)
        return fail(GA_ERR_ARG, "experts_arrange: bad count");
    if (experts > GA_EXPERTS_MAX || top > GA_EXPERTS_MAX_TOP)
        return fail(GA_ERR_SHAPE, "experts_arrange: more than %d experts or %d choices",
                    GA_EXPERTS_MAX, GA_EXPERTS_MAX_TOP);
    const long long pairs = (long long)tokens * top;
    if (pairs > 0x7FFF0000ll || first > 0x7FFFFFFF - experts)
        return fail(GA_ERR_SHAPE, "experts_arrange: tokens * top and ids must fit in an int");
    if (!starts || (pairs > 0 && (!ids || !row_tokens || !place)))
        return fail(GA_ERR_ARG, "experts_arrange: null pointer");
    hipStream_t st = (hipStream_t)stream;
    if (pairs <= 4096)
        hipLaunchKernelGGL((arrange_kernel<256>), dim3(experts), dim3(256), 0, st, ids, (int)pairs,
                           top, experts, first, starts, row_tokens, place);
    else
        hipLaunchKernelGGL((arrange_kernel<1024>), dim3(experts), dim3(1024), 0, st, ids,
                           (int)pairs, top, experts, first, starts, row_tokens, place);
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

ga_status ga_experts_activate(const void* x, int in_dtype, int rows, int inner, long long stride_x,
                              void* q, long long stride_q, float* scales, long long stride_scales,
                              const int* limit, void* stream)
{
    if (in_dtype != GA_IN_F32 && in_dtype != GA_IN_BF16)
        return fail(GA_ERR_ARG, "experts_activate: in_dtype must be GA_IN_F32 or GA_IN_BF16");
    if (rows < 0 || inner <= 0)
        return fail(GA_ERR_ARG, "experts_activate: bad count");
    if (inner % 128 || inner > 0x3FFFFFFF)
        return fail(GA_ERR_SHAPE, "experts_activate: inner must be a multiple of 128");
    if (rows == 0)
        return GA_OK;
    if (!x || !q || !scales)
        return fail(GA_ERR_ARG, "experts_activate: null pointer");
    const bool one = rows == 1;
    if ((!one && (stride_x < 2ll * inner || stride_q < inner)) || stride_scales < rows)
        return fail(GA_ERR_SHAPE, "experts_activate: rows overlap");
    if ((uintptr_t)x % (in_dtype == GA_IN_F32 ? 4 : 2))
        return fail(GA_ERR_SHAPE, "experts_activate: x must have its elements' alignment");
    if ((uintptr_t)q % 8 || (!one && stride_q % 8))
        return fail(GA_ERR_SHAPE, "experts_activate: q must be 8-byte aligned, its stride too");
    const int parts = (inner / 128 + kActBlocks - 1) / kActBlocks;
    const long long groups = parts * ((rows + (long long)kActRows - 1) / kActRows);
    if (groups > most_workgroups(256))
        return fail(GA_ERR_SHAPE, "experts_activate: too many elements for one call");
    const dim3 grid((unsigned)groups);
    hipStream_t st = (hipStream_t)stream;
    if (in_dtype == GA_IN_F32)
        hipLaunchKernelGGL((activate_kernel<GA_IN_F32>), grid, dim3(256), 0, st, x, rows, inner,
                           stride_x, (uint8_t*)q, stride_q, scales, stride_scales, limit, parts);
    else
        hipLaunchKernelGGL((activate_kernel<GA_IN_BF16>), grid, dim3(256), 0, st, x, rows, inner,
                           stride_x, (uint8_t*)q, stride_q, scales, stride_scales, limit, parts);
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

ga_status ga_experts_combine(const void* y, int rows, int n, long long stride_y, const int* place,
                             const float* weights, int tokens, int top, void* out, int out_dtype,
                             long long stride_out, void* stream)
{
    if (out_dtype != GA_DTYPE_F32 && out_dtype != GA_DTYPE_BF16)
        return fail(GA_ERR_ARG, "experts_combine: out_dtype must be GA_DTYPE_F32 or GA_DTYPE_BF16");
    if (rows < 0 || n <= 0 || tokens < 0 || top <= 0)
        return fail(GA_ERR_ARG, "experts_combine: bad count");
    if (tokens == 0)
        return GA_OK;
    if ((!y && rows > 0) || !place || !weights || !out)
        return fail(GA_ERR_ARG, "experts_combine: null pointer");
    if ((rows > 1 && stride_y < n) || (tokens > 1 && stride_out < n))
        return fail(GA_ERR_SHAPE, "experts_combine: rows overlap");
    if (n > 0x7FFF0000)
        return fail(GA_ERR_SHAPE, "experts_combine: rows of %d elements", n);
    if (rows == 0) // every place is left out; what is loaded for it has to be readable
        y = out;
    if ((uintptr_t)y % 2 || (uintptr_t)out % (out_dtype == GA_DTYPE_F32 ? 4 : 2))
        return fail(GA_ERR_SHAPE, "experts_combine: y and out must have their elements' alignment");
    const int parts = (n - 1) / 2048 + 1;
    if ((long long)tokens * parts > most_workgroups(256))
        return fail(GA_ERR_SHAPE, "experts_combine: too many elements for one call");
    const dim3 grid((unsigned)(tokens * (long long)parts));
    hipStream_t st = (hipStream_t)stream;
    if (out_dtype == GA_DTYPE_F32)
        hipLaunchKernelGGL((combine_kernel<GA_DTYPE_F32>), grid, dim3(256), 0, st,
                           (const uint16_t*)y, rows, n, stride_y, place, weights, top, out,
                           stride_out, parts);
    else
        hipLaunchKernelGGL((combine_kernel<GA_DTYPE_BF16>), grid, dim3(256), 0, st,
                           (const uint16_t*)y, rows, n, stride_y, place, weights, top, out,
                           stride_out, parts);
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

} // extern "C"

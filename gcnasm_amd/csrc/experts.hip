// experts.hip -- layers of experts around their products: the choice of a token's experts
// (route), the map of rows (arrange), the gated activation that quantises for the second
// product (activate) and the weighted sum that ends the layer (combine). The products:
// gemm_experts.hip.
#include "ga_device.hpp"
#include "ga_internal.hpp"
#include "ga_quant.hpp"

#include <algorithm>

namespace ga {
namespace {

// ---- route ------------------------------------------------------------------------
// A wave has one token; lane l holds the experts l, l + 64, ... A choice is a maximum over the
// wave of keys made comparable as integers, then the lowest expert that has it.

// The wave's maximum, uniform.
__device__ __forceinline__ uint32_t wave_max(uint32_t a)
{
    a = group_max_dpp<16>(a);
    const uint32_t x = max((uint32_t)__builtin_amdgcn_readlane(a, 0),
                           (uint32_t)__builtin_amdgcn_readlane(a, 16));
    const uint32_t y = max((uint32_t)__builtin_amdgcn_readlane(a, 32),
                           (uint32_t)__builtin_amdgcn_readlane(a, 48));
    return max(x, y);
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
constexpr double kMinus = -__builtin_inf();

// WIDE: keys in 64 bits (a bias), else the logits in 32.
template <int VPT, int IN, bool WIDE>
__global__ __launch_bounds__(64 * kRouteWaves) void route_kernel(ga_experts_route_args a)
{
    extern __shared__ double by_all[]; // [wave][expert], with groups
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long t = (long long)blockIdx.x * kRouteWaves + wave;
    if (t >= a.tokens)
        return;
    const int E = a.experts;
    const bool softmax = a.scores == GA_EXPERTS_SOFTMAX;

    // logits: NaN and -inf to -inf (not there), +inf to the largest finite value
    auto logit = [&](int e) {
        const long long i = t * a.stride_logits + e;
        const float x = IN == GA_IN_F32 ? ((const float*)a.logits)[i]
                                        : bf16_to_f32(((const uint16_t*)a.logits)[i]);
        return x > -__builtin_inff() ? fminf(x, 3.40282347e38f) : -__builtin_inff();
    };
    float x[VPT];
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const int e = v * 64 + lane;
        x[v] = e < E ? logit(e) : -__builtin_inff();
    }
    uint32_t top = 0;
#pragma unroll
    for (int v = 0; v < VPT; v++)
        top = max(top, ordered(x[v]));
    const float m = unordered(wave_max(top)); // the largest logit

    // scores in 64 bits where the choice goes by them
    const bool grouped = a.top_groups < a.groups;
    const bool by_score = grouped && a.group_rank == 2;
    double score[VPT];
    if (WIDE || by_score) {
        double sum = 0.0;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const double d = (double)x[v];
            if (softmax) {
                score[v] = x[v] > -__builtin_inff() ? exp(d - (double)m) : 0.0;
                sum += score[v];
            } else {
                score[v] = 1.0 / (1.0 + exp(-d));
            }
        }
        if (softmax) {
            sum = wave_sum(sum);
#pragma unroll
            for (int v = 0; v < VPT; v++)
                score[v] /= sum;
        }
    }

    uint32_t key[VPT], low[VPT];
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const int e = v * 64 + lane;
        if constexpr (WIDE) {
            const double k = score[v] + (e < E ? (double)a.bias[e] : 0.0);
            const bool there = x[v] > -__builtin_inff() && k > kMinus;
            const uint64_t u = there ? ordered(k) : 0;
            key[v] = (uint32_t)(u >> 32);
            low[v] = (uint32_t)u;
            score[v] = there ? k : kMinus;
        } else {
            key[v] = x[v] > -__builtin_inff() ? ordered(x[v]) : 0u;
            low[v] = 0u;
        }
    }

    if (grouped) {
        // lanes of a group go over its experts, the two largest of each joined
        double* by = by_all + wave * E;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const int e = v * 64 + lane;
            if (e < E)
                by[e] = WIDE || (by_score && key[v]) ? score[v]
                        : key[v]                     ? (double)x[v]
                                                     : kMinus;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int size = E / a.groups;
        const int shift = 31 - __builtin_clz(64 / a.groups); // log2 of the lanes of a group
        const int g = lane >> shift, sub = lane & ((1 << shift) - 1);
        double b1 = kMinus, b2 = kMinus;
        if (g < a.groups)
            for (int i = sub; i < size; i += 1 << shift) {
                const double d = by[g * size + i];
                b2 = fmax(b2, fmin(b1, d));
                b1 = fmax(b1, d);
            }
        for (int d = 1; d < 1 << shift; d <<= 1) {
            const double o1 = __shfl_xor(b1, d, 64), o2 = __shfl_xor(b2, d, 64);
            b2 = fmax(fmin(b1, o1), fmax(b2, o2));
            b1 = fmax(b1, o1);
        }
        const double value = a.group_rank == 2 && b2 > kMinus ? b1 + b2 : b1;
        int before = 0;
        for (int j = 0; j < a.groups; j++) {
            const double o = __shfl(value, j << shift, 64);
            before += o > value || (o == value && j < g);
        }
        const uint64_t kept = __builtin_amdgcn_ballot_w64(g < a.groups && sub == 0 &&
                                                          value > kMinus && before < a.top_groups);
        // e / size by a multiplication, exact for e and size up to 1024
        const uint32_t inv = ((1u << 20) + size - 1) / size;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const uint32_t of = ((uint32_t)(v * 64 + lane) * inv) >> 20;
            if (!((kept >> (of << shift)) & 1))
                key[v] = low[v] = 0u;
        }
    }

    int id = -1; // of choice `lane`
    for (int j = 0; j < a.top; j++) {
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
        int e = -1;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const uint64_t has =
                __builtin_amdgcn_ballot_w64(key[v] == best && (!WIDE || low[v] == second));
            if (e < 0 && has != 0) {
                const int l = __builtin_ctzll(has);
                e = v * 64 + l;
                if (lane == l)
                    key[v] = low[v] = 0u;
            }
        }
        if (lane == j)
            id = e;
    }

    // weights of the chosen ones, in 64 bits
    double w = 0.0;
    if (softmax) {
        const float xi = id >= 0 ? logit(id) : -__builtin_inff();
        float from = m;
        if (a.renormalise)
            from = unordered(wave_max(ordered(xi)));
        w = id >= 0 ? exp((double)xi - (double)from) : 0.0;
        if (a.renormalise) {
            const double sum = wave_sum(w);
            w = sum > 0.0 ? w / sum : 0.0;
        } else {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < VPT; v++)
                sum += x[v] > -__builtin_inff() ? expf(x[v] - m) : 0.0f;
            const double all = wave_sum((double)sum);
            w = id >= 0 ? w / all : 0.0;
        }
    } else {
        w = id >= 0 ? 1.0 / (1.0 + exp(-(double)logit(id))) : 0.0;
        if (a.renormalise) {
            const double sum = wave_sum(w);
            w = sum > 0.0 ? w / sum : 0.0;
        }
    }
    if (lane < a.top) {
        a.ids[t * a.top + lane] = id;
        a.weights[t * a.top + lane] = id >= 0 ? (float)(w * (double)a.scale) : 0.0f;
    }
}

template <int IN, bool WIDE>
void launch_route(const ga_experts_route_args& a, hipStream_t st)
{
    const dim3 grid((unsigned)((a.tokens + (long long)kRouteWaves - 1) / kRouteWaves));
    const size_t lds = a.top_groups < a.groups ? sizeof(double) * kRouteWaves * a.experts : 0;
    auto go = [&](auto V) {
        hipLaunchKernelGGL((route_kernel<decltype(V)::value, IN, WIDE>), grid,
                           dim3(64 * kRouteWaves), lds, st, a);
    };
    const int v = (a.experts + 63) / 64;
    if (v <= 1)
        go(std::integral_constant<int, 1>{});
    else if (v <= 2)
        go(std::integral_constant<int, 2>{});
    else if (v <= 3)
        go(std::integral_constant<int, 3>{});
    else if (v <= 4)
        go(std::integral_constant<int, 4>{});
    else if (v <= 8)
        go(std::integral_constant<int, 8>{});
    else
        go(std::integral_constant<int, 16>{});
}

// ---- arrange ----------------------------------------------------------------------
// A workgroup has one expert and reads all ids: those of smaller experts give its first row,
// its own become bits, one word for 64 pairs, from which the rows are written in order. No
// atomics: the same ids give the same rows.
constexpr int kMaskWords = 4096; // bits of 262144 pairs at a time

template <int NT>
__global__ __launch_bounds__(NT) void arrange_kernel(const int* __restrict__ ids, int pairs,
                                                     int top, int experts, int first,
                                                     int* __restrict__ starts,
                                                     int* __restrict__ row_tokens,
                                                     int* __restrict__ place)
{
    constexpr int NW = NT / 64;
    __shared__ uint64_t mask[kMaskWords];
    __shared__ int part[3][NW];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t me = blockIdx.x;
    const long long words = ((long long)pairs + 63) / 64;

    int less = 0, valid = 0;
    // the words w0 .. w1 - 1: bits of this expert's pairs, and counts
    auto pass = [&](long long w0, long long w1, bool counts) {
        for (long long w = w0 + wave; w < w1; w += NW) {
            const long long p = w * 64 + lane;
            const uint32_t e = p < pairs ? (uint32_t)ids[p] - (uint32_t)first : ~0u;
            const uint64_t has = __builtin_amdgcn_ballot_w64(e == me);
            if (counts) {
                less += __builtin_popcountll(__builtin_amdgcn_ballot_w64(e < me));
                valid += __builtin_popcountll(__builtin_amdgcn_ballot_w64(e < (uint32_t)experts));
                if (w % experts == (long long)me && p < pairs && e >= (uint32_t)experts)
                    place[p] = -1;
            }
            if (lane == 0 && w - w0 < kMaskWords)
                mask[w - w0] = has;
        }
    };
    pass(0, words, true);
    if (lane == 0) {
        part[0][wave] = less;
        part[1][wave] = valid;
    }
    __syncthreads();
    less = valid = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        less += part[0][i];
        valid += part[1][i];
    }
    if (threadIdx.x == 0) {
        starts[me] = less;
        if (me == (uint32_t)experts - 1)
            starts[experts] = valid;
    }
    // rows behind the last expert's
    for (long long r = valid + (long long)me * NT + threadIdx.x; r < pairs;
         r += (long long)experts * NT)
        row_tokens[r] = -1;

    long long base = less;
    for (long long w0 = 0; w0 < words; w0 += kMaskWords) {
        const long long w1 = min(words, w0 + kMaskWords);
        if (w0 > 0) {
            __syncthreads(); // the words before have been read
            pass(w0, w1, false);
            __syncthreads();
        }
        const int n = (int)(w1 - w0), per = (n + NT - 1) / NT;
        const int b = min(n, (int)threadIdx.x * per), e = min(n, b + per);
        int count = 0;
        for (int i = b; i < e; i++)
            count += __builtin_popcountll(mask[i]);
        int before = count;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(before, d, 64);
            before += lane >= d ? o : 0;
        }
        if (lane == 63)
            part[2][wave] = before;
        __syncthreads();
        int all = 0;
        before -= count;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            before += i < wave ? part[2][i] : 0;
            all += part[2][i];
        }
        long long row = base + before;
        for (int i = b; i < e; i++)
            for (uint64_t bits = mask[i]; bits; bits &= bits - 1) {
                const long long p = (w0 + i) * 64 + __builtin_ctzll(bits);
                row_tokens[row] = (int)(p / top);
                place[p] = (int)row;
                row++;
            }
        base += all;
    }
}

// ---- activate ---------------------------------------------------------------------
// A workgroup has 32 rows of a block of 128: sixteen lanes a row, eight elements of gate and up
// each; the rows' scales lie side by side, one line of the transposed scales.
constexpr int kActRows = 32;

template <int IN>
__device__ __forceinline__ void load8(const void* x, size_t i, bool wide, float (&v)[8])
{
    if constexpr (IN == GA_IN_F32) {
        const float* p = (const float*)x + i;
        if (wide) {
            const v4f a = *(const v4f*)p, b = *(const v4f*)(p + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = a[j];
                v[4 + j] = b[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                v[j] = p[j];
        }
    } else {
        const uint16_t* p = (const uint16_t*)x + i;
        if (wide) {
            const v4i a = *(const v4i*)p;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[2 * j] = __uint_as_float((uint32_t)a[j] << 16);
                v[2 * j + 1] = __uint_as_float((uint32_t)a[j] & 0xFFFF0000u);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                v[j] = bf16_to_f32(p[j]);
        }
    }
}

template <int IN, bool WIDE>
__global__ __launch_bounds__(256) void activate_kernel(const void* __restrict__ x, int rows,
                                                       int inner, long long stride_x,
                                                       uint8_t* __restrict__ q, long long stride_q,
                                                       float* __restrict__ scales,
                                                       long long stride_scales,
                                                       const int* __restrict__ limit)
{
    constexpr int U = kActRows / 16;
    const int live = limit ? min(rows, max(0, *limit)) : rows;
    const int blocks = inner / 128;
    const int g = blockIdx.x % blocks;
    const long long r0 = (long long)(blockIdx.x / blocks) * kActRows;
    if (r0 >= live)
        return;
    const int sub = threadIdx.x & 15;
    float gate[U][8], up[U][8];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long long r = min(r0 + u * 16 + (threadIdx.x >> 4), (long long)live - 1);
        const size_t at = (size_t)r * stride_x + g * 128 + sub * 8;
        load8<IN>(x, at, WIDE, gate[u]);
        load8<IN>(x, at + inner, WIDE, up[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long long r = r0 + u * 16 + (threadIdx.x >> 4);
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            y[j] = gate[u][j] / (1.0f + expf(-gate[u][j])) * up[u][j];
        bool nan;
        const float s = ds_scale(__uint_as_float(block_amax<16, 8>(y, nan)));
        const ScaleDiv d(s);
        const bool nan_rule = nan || __builtin_amdgcn_ballot_w64(!d.fast) != 0;
        if (r >= live)
            continue;
        uint8_t* dst = q + (size_t)r * stride_q + g * 128 + sub * 8;
        if (nan_rule)
            fp8_store_codes<true>(d, y, dst);
        else
            fp8_store_codes<false>(d, y, dst);
        if (sub == 0)
            scales[(size_t)g * stride_scales + r] = s;
    }
}

// ---- combine ----------------------------------------------------------------------
// A thread has EL elements of a token and adds up its rows', eight rows' loads at a time.
template <int EL, int OUT>
__global__ __launch_bounds__(256) void combine_kernel(const uint16_t* __restrict__ y, int rows,
                                                      int n, long long stride_y,
                                                      const int* __restrict__ place,
                                                      const float* __restrict__ weights, int top,
                                                      void* __restrict__ out, long long stride_out,
                                                      int parts)
{
    const int t = blockIdx.x / parts;
    const int c = ((blockIdx.x % parts) * 256 + threadIdx.x) * EL;
    if (c >= n)
        return;
    float acc[EL];
#pragma unroll
    for (int i = 0; i < EL; i++)
        acc[i] = 0.0f;
    constexpr int B = 8;
    for (int j0 = 0; j0 < top; j0 += B) {
        uint32_t raw[B][(EL + 1) / 2];
        float w[B];
        bool ok[B];
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int j = min(j0 + b, top - 1);
            const int r = place[(size_t)t * top + j];
            ok[b] = j0 + b < top && r >= 0 && r < rows;
            w[b] = weights[(size_t)t * top + j];
            const uint16_t* p = y + (size_t)(ok[b] ? r : 0) * stride_y + c;
            if constexpr (EL == 8) {
                const v4i d = *(const v4i*)p;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    raw[b][i] = (uint32_t)d[i];
            } else {
                raw[b][0] = *p;
            }
        }
#pragma unroll
        for (int b = 0; b < B; b++)
            if (ok[b])
#pragma unroll
                for (int i = 0; i < EL; i++) {
                    const uint32_t u = raw[b][i / 2];
                    acc[i] = fmaf(w[b], __uint_as_float(i & 1 ? u & 0xFFFF0000u : u << 16), acc[i]);
                }
    }
    const size_t o = (size_t)t * stride_out + c;
    if constexpr (OUT == GA_DTYPE_F32) {
        float* p = (float*)out + o;
#pragma unroll
        for (int i = 0; i < EL; i += 4)
            if constexpr (EL == 8)
                *(v4f*)(p + i) = (v4f){acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
            else
                p[i] = acc[i];
    } else {
        uint16_t* p = (uint16_t*)out + o;
        if constexpr (EL == 8) {
            v4i d;
#pragma unroll
            for (int i = 0; i < 4; i++)
                d[i] = (int)((uint32_t)f32_to_bf16(acc[2 * i]) |
                             ((uint32_t)f32_to_bf16(acc[2 * i + 1]) << 16));
            *(v4i*)p = d;
        } else {
            *p = f32_to_bf16(acc[0]);
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
    if (a.in_dtype == GA_IN_F32)
        a.bias ? launch_route<GA_IN_F32, true>(a, st) : launch_route<GA_IN_F32, false>(a, st);
    else
        a.bias ? launch_route<GA_IN_BF16, true>(a, st) : launch_route<GA_IN_BF16, false>(a, st);
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
    if ((uintptr_t)q % 8 || (!one && stride_q % 8))
        return fail(GA_ERR_SHAPE, "experts_activate: q must be 8-byte aligned, its stride too");
    const long long groups = (long long)(inner / 128) * ((rows + (long long)kActRows - 1) / kActRows);
    if (groups > most_workgroups(256))
        return fail(GA_ERR_SHAPE, "experts_activate: too many elements for one call");
    const int el = in_dtype == GA_IN_F32 ? 4 : 8; // elements of 16 bytes
    const bool wide = (uintptr_t)x % 16 == 0 && (one || stride_x % el == 0);
    const dim3 grid((unsigned)groups);
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto IN, auto WIDE) {
        hipLaunchKernelGGL((activate_kernel<decltype(IN)::value, decltype(WIDE)::value>), grid,
                           dim3(256), 0, st, x, rows, inner, stride_x, (uint8_t*)q, stride_q,
                           scales, stride_scales, limit);
    };
    auto kind = [&](auto IN) {
        wide ? go(IN, std::true_type{}) : go(IN, std::false_type{});
    };
    if (in_dtype == GA_IN_F32)
        kind(std::integral_constant<int, GA_IN_F32>{});
    else
        kind(std::integral_constant<int, GA_IN_BF16>{});
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
    const bool wide = n % 8 == 0 && (uintptr_t)y % 16 == 0 && (uintptr_t)out % 16 == 0 &&
                      (rows == 1 || stride_y % 8 == 0) && (tokens == 1 || stride_out % 8 == 0);
    const int el = wide ? 8 : 1;
    const int parts = (int)(((long long)n + 256 * el - 1) / (256 * el));
    if ((long long)tokens * parts > most_workgroups(256))
        return fail(GA_ERR_SHAPE, "experts_combine: too many elements for one call");
    const dim3 grid((unsigned)(tokens * (long long)parts));
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto EL, auto OUT) {
        hipLaunchKernelGGL((combine_kernel<decltype(EL)::value, decltype(OUT)::value>), grid,
                           dim3(256), 0, st, (const uint16_t*)y, rows, n, stride_y, place, weights,
                           top, out, stride_out, parts);
    };
    auto kind = [&](auto EL) {
        if (out_dtype == GA_DTYPE_F32)
            go(EL, std::integral_constant<int, GA_DTYPE_F32>{});
        else
            go(EL, std::integral_constant<int, GA_DTYPE_BF16>{});
    };
    wide ? kind(std::integral_constant<int, 8>{}) : kind(std::integral_constant<int, 1>{});
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

} // extern "C"

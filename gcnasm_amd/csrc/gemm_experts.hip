// gemm_experts.hip -- the block-scale product of each expert's rows with its weights:
//   out[r, n] = sum_g P_g[r, n] * SFA[g, m] * SFB[e, n/128, g],  m = rows_of[r] or r,
// expert e of row r by starts, P_g the MFMA's sum over 128-K group g (unit E8M0 scales),
// acc = fmaf(P_g, SFA * SFB, acc) per group as in the other block-scale kernels.
//
// Counts are on the GPU: the grid has a workgroup for every tile that there can be, each finds
// its expert (ga_experts.hpp), those past the last tile end at once. Rows are gathered by the
// copies into LDS, whose addresses are a lane's own.
#include "ga_bs_decode.hpp"
#include "ga_device.hpp"
#include "ga_experts.hpp"
#include "ga_internal.hpp"
#include "ga_pp.hpp"

#include <algorithm>

namespace ga {
namespace {

// Operands span less than this, so an offset kNowhere is past the end of a descriptor, and
// stays so when the steps along K are added: such a load gives zeros.
constexpr uint32_t kNowhere = 0xF0000000u;
constexpr unsigned long long kMostBytes = 0xE0000000ull;
constexpr unsigned long long kMostScaleBytes = 0x0FFF0000ull;

// A tile's rows: row `local` of it, counted from x.first's tile, in a. Gathered rows that are
// not in a, and rows behind the expert's last, are nowhere.
__device__ __forceinline__ uint32_t row_offset(const ga_experts_product_args& a, int row0, int count,
                                               int local, uint32_t ld)
{
    if (local >= count)
        return kNowhere;
    if (a.rows_of == nullptr)
        return (uint32_t)local * ld;
    const int m = a.rows_of[row0 + local];
    return m >= 0 && m < a.a_rows ? (uint32_t)m * ld : kNowhere;
}

// ---- few rows: weights streamed, K slices over the waves of a workgroup --------------
template <int TM, int NG>
__global__ __attribute__((amdgpu_flat_work_group_size(64, 512), amdgpu_waves_per_eu(1, 2)))
void experts_few_kernel(ga_experts_product_args a, int shares, int ks, int gps)
{
    using Cfg = BdCfg<TM, NG>;
    __shared__ __attribute__((aligned(1024))) char smem[8 * Cfg::kWave];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slice = wave % ks, tl = wave / ks;
    int total;
    const int t = blockIdx.x / shares, share = blockIdx.x % shares;
    const ExpertTile x = find_expert(a.starts, a.experts, a.rows, 16 * TM, lane, t, &total);
    if (t >= total)
        return;
    const int row0 = x.first + (t - x.before) * 16 * TM;
    const int M = min(16 * TM, x.last - row0), N = a.n;
    const int ngroups = (N + 15) / 16;
    const int g_end = (int)(((long long)(share + 1) * ngroups) / shares);
    const int cg0 = (int)(((long long)share * ngroups) / shares) + tl * NG;
    const int ng_here = min(NG, g_end - cg0);
    const bool live = ng_here > 0;
    const int G = a.k / 128;
    const int gb = slice * gps;
    const int ge = min(G, gb + gps);
    const int nsteps = live ? max(0, ge - gb) : 0;
    const int r = lane & 15, g = lane >> 4;
    char* ring = smem + wave * Cfg::kWave;

    v4f acc[NG][TM];
#pragma unroll
    for (int c = 0; c < NG; c++)
#pragma unroll
        for (int i = 0; i < TM; i++)
            acc[c][i] = (v4f){0.f, 0.f, 0.f, 0.f};

    if (nsteps > 0) {
        const uint32_t lda = (uint32_t)a.stride_a, ldb = (uint32_t)a.stride_b;
        const bool gathered = a.rows_of != nullptr;
        const auto ra = make_rsrc((const char*)a.a + (gathered ? 0 : (size_t)row0 * lda),
                                  rows_bytes(gathered ? a.a_rows : M, lda, a.k));
        const char* pb = (const char*)a.b + (size_t)x.expert * a.stride_b_expert +
                         (size_t)cg0 * 16 * ldb;
        const auto rb = make_rsrc(pb, rows_bytes(min(ng_here * 16, N - cg0 * 16), ldb, a.k));
        // copy h (0, 1) of a 16-row block: lane l fetches row 8h + l / 8 from
        // whole 128-byte lines into slot l % 8
        const uint32_t crow = (uint32_t)lane >> 3, cslot = lane & 7;
        const uint32_t c0 = (cslot ^ ((crow >> 1) & 7)) * 16, c1 = c0 ^ 64u;
        uint32_t va[TM][2];
#pragma unroll
        for (int i = 0; i < TM; i++) {
            va[i][0] = row_offset(a, row0, M, i * 16 + crow, lda) + c0 + (uint32_t)gb * 128;
            va[i][1] = row_offset(a, row0, M, i * 16 + 8 + crow, lda) + c1 + (uint32_t)gb * 128;
        }
        const uint32_t vb0 = crow * ldb + c0 + (uint32_t)gb * 128;
        const uint32_t vb1 = (crow + 8) * ldb + c1 + (uint32_t)gb * 128;

        // scales: lane l that of row l, and of the 128-column block of group l % NG
        const auto rsa = make_rsrc(a.sfa + (gathered ? 0 : row0),
                                   rows_bytes_f32(G, a.stride_sfa, gathered ? a.a_rows : M));
        const uint32_t sa_step = (uint32_t)a.stride_sfa * 4;
        const uint32_t vsa = row_offset(a, row0, M, gathered ? lane : min(lane, M - 1), 4) +
                             (uint32_t)gb * sa_step;
        const int nblk = (N + 127) / 128;
        const auto rsb = make_rsrc(a.sfb + (size_t)x.expert * a.stride_sfb_expert,
                                   rows_bytes_f32(nblk, a.stride_sfb, G));
        const uint32_t vsb = ((uint32_t)min(((cg0 + lane % NG) * 16) / 128, nblk - 1) *
                                  (uint32_t)a.stride_sfb + gb) * 4;

        // step s into a ring slot, every operand and scale by direct-to-LDS copies
        auto load = [&](int s, char* slot) {
            const uint32_t ok = (uint32_t)s * 128;
#pragma unroll
            for (int i = 0; i < TM; i++) {
                char* dst = slot + i * 2048;
                lds_load16(ra, (lds_void*)dst, va[i][0] + bd_uni(ok), 0);
                lds_load16(ra, (lds_void*)(dst + 1024), va[i][1] + bd_uni(ok), 0);
            }
#pragma unroll
            for (int c = 0; c < NG; c++) {
                const uint32_t ob = ok + (uint32_t)c * 16 * ldb;
                char* dst = slot + (TM + c) * 2048;
                lds_load16(rb, (lds_void*)dst, vb0 + bd_uni(ob), 0);
                lds_load16(rb, (lds_void*)(dst + 1024), vb1 + bd_uni(ob), 0);
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsa, (lds_void*)(slot + Cfg::kScales), 4,
                                                     vsa + bd_uni((uint32_t)s * sa_step), 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsb, (lds_void*)(slot + Cfg::kScales + 256), 4,
                                                     vsb + bd_uni((uint32_t)s * 4), 0, 0, 0);
        };
        bd_chain<TM, NG, BD_GROUP128>(ring, lane, nsteps, load, acc);
    }

    // lane holds out[m][n .. n+3], m = 16i + lane%16, n = 16cg + 4(lane/16)
    uint16_t* out = (uint16_t*)a.out + (size_t)row0 * a.stride_out;
    const bool even = ((uintptr_t)a.out & 7) == 0 && (a.stride_out & 3) == 0;
    auto store = [&](int c, int i, const v4f& v) {
        const int n = (cg0 + c) * 16 + g * 4;
        const int m = i * 16 + r;
        if (c >= ng_here || n >= N || m >= M)
            return;
        uint16_t* o = out + (size_t)m * a.stride_out + n;
        if (even && n + 4 <= N) {
            *(uint2*)o = make_uint2((uint32_t)f32_to_bf16(v[0]) | ((uint32_t)f32_to_bf16(v[1]) << 16),
                                    (uint32_t)f32_to_bf16(v[2]) | ((uint32_t)f32_to_bf16(v[3]) << 16));
        } else {
            for (int e = 0; e < 4 && n + e < N; e++)
                o[e] = f32_to_bf16(v[e]);
        }
    };
    bd_join<TM, NG>(smem, wave, lane, slice, tl, ks, live, acc, store);
}

template <int TM, int NG>
ga_status launch_few(const ga_experts_product_args& a, hipStream_t st)
{
    const int G = a.k / 128, groups = (a.n + 15) / 16;
    const int ks = G >= 8 ? 4 : G >= 2 ? 2 : 1;
    const int gps = (G + ks - 1) / ks;
    const int tasks = std::min(8 / ks, (groups + NG - 1) / NG);
    const int shares = (groups + tasks * NG - 1) / (tasks * NG);
    const long long grid = most_expert_tiles(a.rows, a.experts, 16 * TM) * shares;
    if (grid > most_workgroups(64 * tasks * ks))
        return fail(GA_ERR_SHAPE, "experts_product: too many tiles for one call");
    hipLaunchKernelGGL((experts_few_kernel<TM, NG>), dim3((unsigned)grid), dim3(64 * tasks * ks), 0,
                       st, a, shares, ks, gps);
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

} // namespace
} // namespace ga

using namespace ga;

extern "C" ga_status ga_experts_product(const ga_experts_product_args* args, void* stream)
{
    if (!args)
        return fail(GA_ERR_ARG, "experts_product: null argument");
    const ga_experts_product_args& a = *args;
    if (a.experts <= 0 || a.rows < 0 || a.n <= 0 || a.k <= 0 || a.a_rows < 0)
        return fail(GA_ERR_ARG, "experts_product: bad count");
    if (a.experts > GA_EXPERTS_MAX)
        return fail(GA_ERR_SHAPE, "experts_product: more than %d experts", GA_EXPERTS_MAX);
    if (a.k % 128)
        return fail(GA_ERR_GROUP, "K must be a multiple of GROUP_K (128), got %d", a.k);
    if (a.rows == 0)
        return GA_OK;
    if (!a.a || !a.sfa || !a.b || !a.sfb || !a.starts || !a.out)
        return fail(GA_ERR_ARG, "experts_product: null pointer");
    if (a.a_rows < (a.rows_of ? 1 : a.rows))
        return fail(GA_ERR_SHAPE, "experts_product: a has %lld rows", a.a_rows);
    if (((uintptr_t)a.a | (uintptr_t)a.b | (unsigned long long)a.stride_a |
         (unsigned long long)a.stride_b | (unsigned long long)a.stride_b_expert) % 16)
        return fail(GA_ERR_SHAPE, "experts_product: a, b and their strides must be multiples of 16");
    const int blocks = (a.n - 1) / 128 + 1;
    if (a.stride_a < a.k || a.stride_b < a.k || a.stride_out < a.n || a.stride_sfa < a.a_rows ||
        a.stride_sfb < a.k / 128 || a.stride_b_expert < 0 || a.stride_sfb_expert < 0)
        return fail(GA_ERR_SHAPE, "experts_product: rows overlap");
    // 32-bit offsets into a tile's rows, and into all of a where rows are gathered
    const unsigned long long lim = kMostBytes;
    if ((unsigned long long)a.stride_a > lim / 256 || (unsigned long long)a.stride_b > lim / 256)
        return fail(GA_ERR_SHAPE, "experts_product: 256 rows of a or b pass 0xE0000000 bytes");
    const unsigned long long G = a.k / 128;
    const unsigned long long most_sfa = a.rows_of ? kMostScaleBytes : 0xFFFFFFF0ull;
    if (a.rows_of && (unsigned long long)a.a_rows > lim / (unsigned long long)a.stride_a)
        return fail(GA_ERR_SHAPE, "experts_product: gathered rows of a pass 0xE0000000 bytes");
    if ((unsigned long long)a.stride_sfa > most_sfa / 4 / G ||
        (unsigned long long)a.stride_sfb > 0xFFFFFFF0ull / 4 / blocks)
        return fail(GA_ERR_SHAPE, "experts_product: scales pass 4 GiB, or 0x0FFF0000 bytes with "
                                  "gathered rows");
    hipStream_t st = (hipStream_t)stream;
    const long long each = ((long long)a.rows + a.experts - 1) / a.experts;
    if (each <= 16)
        return launch_few<1, 2>(a, st);
    if (each <= 32)
        return launch_few<2, 2>(a, st);
    return launch_few<4, 4>(a, st);
}

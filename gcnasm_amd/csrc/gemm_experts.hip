// gemm_experts.hip -- the block-scale product of each expert's rows with its weights:
//   out[r, n] = sum_g P_g[r, n] * SFA[g, m] * SFB[e, n/128, g],  m = rows_of[r] or r,
// expert e of row r by starts, P_g the MFMA's sum over 128-K group g (unit E8M0 scales),
// acc = fmaf(P_g, SFA * SFB, acc) per group as in the other block-scale kernels.
//
// Counts are on the GPU: the grid has a workgroup for every tile that there can be, each finds
// its expert (ga_experts.hpp), those past the last tile end at once. Rows are gathered by the
// copies into LDS, whose addresses are a lane's own.
#include "ga_bs_decode.hpp"
#include "ga_bs_pp.hpp"
#include "ga_device.hpp"
#include "ga_experts.hpp"
#include "ga_internal.hpp"
#include "ga_pp.hpp"

#include <algorithm>
#include <cmath>

namespace ga {
namespace {

// Operands span less than this, so an offset kNowhere is past the end of a descriptor, and
// stays so when the steps along K are added: such a load gives zeros. The copies past K can take
// the scales' sum past 2^32. In the hardware's two offsets that is out of range too (checked on
// MI355X); added up in 32 bits it may come to lie in the operand again, and what is copied
// from there is not used.
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

// The hardware's conversion (v_cvt_pk_bf16_f32, to the nearest, ties to even): in integer operations it
// was 4 to 20 % of a call, 65536 rows of 64 experts of 4096x4096 1153 -> 1100 us, of 4096x1024 438 -> 373.
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint2 bf16x4(const v4f& v)
{
    return __builtin_bit_cast(uint2, __builtin_convertvector(v, v4bf));
}

// Four results of row m, columns n .. n + 3, those below N.
__device__ __forceinline__ void expert_store4(uint16_t* out, long long ld, int m, int n, int N,
                                              const v4f& v)
{
    uint16_t* o = out + (size_t)m * ld + n;
    if (n + 4 <= N) {
        const uint2 d = bf16x4(v);
        *(v2i_any*)o = (v2i){(int)d.x, (int)d.y};
    } else {
        for (int e = 0; e < 4 && n + e < N; e++)
            o[e] = f32_to_bf16(v[e]);
    }
}

// ---- few rows: weights streamed, K slices over the waves of a workgroup --------------
constexpr int kFewWaves = 4;

template <int TM, int NG>
__global__ __attribute__((amdgpu_flat_work_group_size(64, 64 * kFewWaves), amdgpu_waves_per_eu(1, 2)))
void experts_few_kernel(ga_experts_product_args a, int shares, int ks, int gps)
{
    using Cfg = BdCfg<TM, NG>;
    __shared__ __attribute__((aligned(1024))) char smem[kFewWaves * Cfg::kWave];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slice = wave % ks, tl = wave / ks;
    const int t = blockIdx.x / shares, share = blockIdx.x % shares;
    ExpertTile x;
    if (!find_expert(a.starts, a.experts, a.rows, 16 * TM, lane, [&](int) { return t; }, x))
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
    auto store = [&](int c, int i, const v4f& v) {
        const int n = (cg0 + c) * 16 + g * 4;
        const int m = i * 16 + r;
        if (c >= ng_here || n >= N || m >= M)
            return;
        expert_store4(out, a.stride_out, m, n, N, v);
    };
    bd_join<TM, NG>(smem, wave, lane, slice, tl, ks, live, acc, store);
}

template <int TM, int NG>
ga_status launch_few(const ga_experts_product_args& a, int ks, hipStream_t st)
{
    const int G = a.k / 128, groups = (a.n - 1) / 16 + 1;
    while (ks > G)
        ks /= 2;
    const int gps = (G + ks - 1) / ks;
    const int tasks = std::min(kFewWaves / ks, (groups + NG - 1) / NG);
    const int shares = (groups + tasks * NG - 1) / (tasks * NG);
    const long long grid = most_expert_tiles(a.rows, a.experts, 16 * TM) * shares;
    if (grid > most_workgroups(64 * tasks * ks))
        return fail(GA_ERR_SHAPE, "experts_product: too many tiles for one call");
    hipLaunchKernelGGL((experts_few_kernel<TM, NG>), dim3((unsigned)grid), dim3(64 * tasks * ks), 0,
                       st, a, shares, ks, gps);
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

// ---- many rows: eight-wave tiles -------------------------------------------------------
// The chains of the dense kernels (ga_bs_pp.hpp), with rows gathered: a lane of the copies has a row
// offset for each 64 rows of the tile.
template <bool GATHER>
struct ExpertLoad : bspp::BsLoad {
    uint32_t vrow[4];
};

template <bool GATHER>
__device__ __forceinline__ void issue_a(const ExpertLoad<GATHER>& L, char* smem, int h, int t,
                                        int wave)
{
    if constexpr (!GATHER) {
        bspp::issue_a((const bspp::BsLoad&)L, smem, h, t, wave);
    } else {
        char* dst = smem + pp::kARegion + (t & 1) * pp::kOpSlot + h * pp::kHalf + wave * 1024;
        const uint32_t o = pp::uni((uint32_t)t * 128);
        lds_load16(L.ra, (lds_void*)dst, L.vrow[2 * h], o);
        lds_load16(L.ra, (lds_void*)(dst + 8192), L.vrow[2 * h + 1], o);
    }
}

// Steps of 32 columns to copy c (0 .. 3) of 64 positions (expert_column).
__device__ __forceinline__ constexpr uint32_t column_step(int c) { return (c >> 1) + 4 * (c & 1); }

template <bool GATHER>
__device__ __forceinline__ void issue_b(const ExpertLoad<GATHER>& L, char* smem, int h, int t,
                                        int wave)
{
    char* dst = smem + pp::kBRegion + (t & 1) * pp::kOpSlot + h * pp::kHalf + wave * 1024;
    const uint32_t o = (uint32_t)t * 128;
    lds_load16(L.rb, (lds_void*)dst, L.vb, pp::uni(o + column_step(2 * h) * L.b_hstep));
    lds_load16(L.rb, (lds_void*)(dst + 8192), L.vb,
               pp::uni(o + column_step(2 * h + 1) * L.b_hstep));
}

template <int NB, int MODE, bool GATHER>
__device__ __forceinline__ void issue_half(const ExpertLoad<GATHER>& L, char* smem, int t, int slot,
                                           int wave)
{
    using H = bspp::BsHalfCfg<NB>;
    char* dst = smem + slot * H::kSlot + wave * 1024;
    const uint32_t o = (uint32_t)t * 128;
    lds_load16(L.ra, (lds_void*)dst, (GATHER ? L.vrow[0] : L.va) + pp::uni(o), 0);
    lds_load16(L.ra, (lds_void*)(dst + 8192),
               GATHER ? L.vrow[1] + pp::uni(o) : L.va + pp::uni(o + L.a_hstep), 0);
#pragma unroll
    for (int c = 0; c < 2 * NB; c++)
        lds_load16(L.rb, (lds_void*)(dst + pp::kHalf + c * 8192),
                   L.vb + pp::uni(o + (NB == 2 ? column_step(c) : c) * L.b_hstep), 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        L.rs, (lds_void*)(smem + H::kScaleBase + (t & (H::kRing - 1)) * bspp::kSSlot + wave * 256),
        4, L.vs + pp::uni((uint32_t)t * L.s_kstep), 0, 0, 0);
}

// Column of position p of the first 64 of a tile of 256 columns. Position 128 h + 32 w + 16 t + j, which
// is wave w's element j of MFMA tile t of column half h, has column 64 w + 32 h + 8 (j / 4) + 4 t +
// j % 4: so a wave has whole 128-byte lines of out and a lane eight consecutive columns of two tiles.
__device__ __forceinline__ uint32_t expert_column(uint32_t p)
{
    return (p & 32) << 1 | (p & 12) << 1 | (p & 16) >> 2 | (p & 3);
}

// The copies of the tile of M rows from row0 on, columns from n0 on.
template <int ROWS, int NB, bool GATHER>
__device__ __forceinline__ void expert_load_setup(const ga_experts_product_args& a, int expert,
                                                  int row0, int M, int n0, int wave, int lane,
                                                  ExpertLoad<GATHER>& L)
{
    const uint32_t lda = (uint32_t)a.stride_a, ldb = (uint32_t)a.stride_b;
    const int N = a.n, G = a.k / 128;
    int crow, ckc;
    pp::copy_lane(wave, lane, crow, ckc);
    L.ra = make_rsrc((const char*)a.a + (GATHER ? 0 : (size_t)row0 * lda),
                     rows_bytes(GATHER ? a.a_rows : M, lda, a.k));
    L.va = (uint32_t)crow * lda + ckc * 16;
    L.a_hstep = 64 * lda;
    if constexpr (GATHER)
#pragma unroll
        for (int i = 0; i < ROWS / 64; i++)
            L.vrow[i] = row_offset(a, row0, M, i * 64 + crow, lda) + ckc * 16;
    L.rb = make_rsrc((const char*)a.b + (size_t)expert * a.stride_b_expert + (size_t)n0 * ldb,
                     rows_bytes(N - n0, ldb, a.k));
    L.vb = (NB == 2 ? expert_column(crow) : (uint32_t)crow) * ldb + ckc * 16;
    L.b_hstep = (NB == 2 ? 32 : 64) * ldb;
    if (wave < 4) {
        // position w*64 + l holds row w*64 + (l%4)*16 + l/4, those past M the last one
        L.rs = make_rsrc(a.sfa + (GATHER ? 0 : row0),
                         rows_bytes_f32(G, a.stride_sfa, GATHER ? a.a_rows : M));
        L.vs = row_offset(a, row0, M, min(wave * 64 + (lane & 3) * 16 + (lane >> 2), M - 1), 4);
        L.s_kstep = (uint32_t)a.stride_sfa * 4;
    } else {
        const int nblk = (N + 127) / 128;
        L.rs = make_rsrc(a.sfb + (size_t)expert * a.stride_sfb_expert,
                         rows_bytes_f32(nblk, a.stride_sfb, G));
        // of each column half (which has the same columns' scales): waves 0 and 1 of four, 2 and 3
        L.vs = (uint32_t)min(n0 / 128 + (NB == 2 ? lane >> 1 & 1 : 0), nblk - 1) * (uint32_t)a.stride_sfb * 4;
        L.s_kstep = 4;
    }
}

__device__ __forceinline__ bspp::BsRead expert_read_setup(char* smem, int lane, int grp, int simd,
                                                          int b_region, int scales)
{
    bspp::BsRead rb;
    uint32_t o, o64;
    pp::operand_lane(lane, o, o64);
    rb.a0 = smem + grp * 64 * 128 + o;
    rb.a1 = smem + grp * 64 * 128 + o64;
    rb.b0 = smem + b_region + simd * 32 * 128 + o;
    rb.b1 = smem + b_region + simd * 32 * 128 + o64;
    rb.sa = smem + scales + grp * 256 + (lane & 15) * 16;
    rb.sb = smem + scales + 1024 + simd / 2 * 8;
    return rb;
}

// Eight results of a row, those below n.
__device__ __forceinline__ void expert_store8(uint16_t* o, const v4i& d, int n)
{
    if (n >= 8)
        // non-temporal: 6000 rows of 60 experts of 2048x1408 65.3 -> 61.7 us, 65536 of 64 of
        // 4096x4096 1 % less; a layer, whose activation reads them next, no slower
        __builtin_nontemporal_store(d, (v4i_any*)o);
    else
#pragma unroll
        for (int e = 0; e < 7; e++)
            if (e < n)
                o[e] = (uint16_t)((uint32_t)d[e / 2] >> e % 2 * 16);
}

// The results of 128 rows and columns to out, `result(i, t)` of 16x16 tile i, t: lane l holds row
// l % 16, columns 4 (l / 16) on. Through LDS, so that whole rows are written (those below M, columns
// below N).
template <class Result>
__device__ __forceinline__ void expert_store128(const ga_experts_product_args& a, char* smem, int row0,
                                             int M, int n0, int wave, int lane, const Result& result)
{
    const int grp = wave >> 2, simd = wave & 3, N = a.n - n0;
    const long long ld = a.stride_out;
    uint16_t* out = (uint16_t*)a.out + (size_t)row0 * ld + n0;
    barrier_lds(); // every wave's operand and scale reads are done
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int m = grp * 64 + i * 16 + (lane & 15);
            const int n = simd * 32 + t * 16 + (lane >> 4) * 4;
            *(uint2*)(smem + m * pp::kStagePitch + n * 2) = bf16x4(result(i, t));
        }
    barrier_lds();
    constexpr int kLanes = 16; // of a row
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const int row = wave * 16 + it * (64 / kLanes) + lane / kLanes;
        const int col = lane % kLanes * 8;
        if (row >= M || col >= N)
            continue;
        uint16_t* o = out + (size_t)row * ld + col;
        const char* from = smem + row * pp::kStagePitch + col * 2;
        expert_store8(o, *(const v4i*)from, N - col);
    }
}

constexpr int kOwnPitch = 128 + 16;
constexpr int kOwnBytes = 16 * kOwnPitch; // of LDS, a wave's own

// The results of ROWS rows and 256 columns: quadrant q of ROWS / 128 * 2, rows first, `result(q, i, t)`
// of its 16x16 tile i, t: lane l holds row l % 16, four columns (expert_column). A wave turns
// its own 16 rows of 64 columns at a time in LDS of its own (`own`), so that whole lines are
// written and no wave waits for another: 65536 rows of 64 experts of 4096x512 251 us, 269 in one piece
// with barriers (of 4096x4096 1100, 1110), 292 from the registers in half lines.
template <int ROWS, class Result>
__device__ __forceinline__ void expert_store(const ga_experts_product_args& a, char* own, int row0,
                                             int M, int n0, int wave, int lane, const Result& result)
{
    const int grp = wave >> 2, simd = wave & 3, N = a.n - n0;
    const long long ld = a.stride_out;
    uint16_t* out = (uint16_t*)a.out + (size_t)row0 * ld + n0;
    char* to = own + (lane & 15) * kOwnPitch + (lane >> 4) * 16;
    const int col = simd * 64 + lane % 8 * 8;
#pragma unroll
    for (int r = 0; r < ROWS / 128; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint2 d0 = bf16x4(result(2 * r + h, i, 0)), d1 = bf16x4(result(2 * r + h, i, 1));
                *(v4i*)(to + h * 64) = (v4i){(int)d0.x, (int)d0.y, (int)d1.x, (int)d1.y};
            }
            wave_lds_fence();
#pragma unroll
            for (int it = 0; it < 2; it++) {
                const int row = it * 8 + lane / 8, m = r * 128 + grp * 64 + i * 16 + row;
                const v4i d = *(const v4i*)(own + row * kOwnPitch + lane % 8 * 16);
                if (m < M && col < N)
                    expert_store8(out + (size_t)m * ld + col, d, N - col);
            }
            wave_lds_fence();
        }
}

// Which tile a workgroup has: XCD by XCD a run of tiles, an expert's column by column within
// bands of `band` row tiles, so that what runs at a time on an XCD shares weights and rows in its L2.
// False: none.
__device__ __forceinline__ bool expert_tile(const ga_experts_product_args& a, int height, int tn,
                                            int lane, int band, ExpertTile& x, int& tile_m,
                                            int& tile_n)
{
    int lin = blockIdx.x;
    auto pick = [&](int tiles) { // the grid has most_expert_tiles() * tn workgroups, an int
        const int total = tiles * tn;
        if (lin >= total)
            return -1;
        if (lin < total / 8 * 8)
            lin = lin % 8 * (total / 8) + lin / 8;
        return lin / tn;
    };
    if (!find_expert(a.starts, a.experts, a.rows, height, lane, pick, x))
        return false;
    const int r = lin - x.before * tn;
    const int first = r / (band * tn) * band;
    const int q = r - first * tn, h = min(x.tiles - first, band);
    tile_m = first + q % h;
    tile_n = q / h;
    return true;
}

constexpr int kExpertBand = 4;

// A tile of 128 rows (M of them there) and NB * 128 columns.
template <int NB, bool GATHER>
__device__ __forceinline__ void expert_half_tile(const ga_experts_product_args& a, char* smem,
                                                 int expert, int row0, int M, int n0, int wave,
                                                 int lane)
{
    using namespace bspp;
    using H = BsHalfCfg<NB>;
    const int grp = wave >> 2, simd = wave & 3;
    v4f acc[NB][4][2];
#pragma unroll
    for (int q = 0; q < NB; q++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int t = 0; t < 2; t++)
                acc[q][i][t] = (v4f){0.f, 0.f, 0.f, 0.f};
    ExpertLoad<GATHER> L;
    expert_load_setup<128, NB>(a, expert, row0, M, n0, wave, lane, L);
    const BsRead rb = expert_read_setup(smem, lane, grp, simd, pp::kHalf, H::kScaleBase);
    bs_half_chain<NB, PS_GROUP128>(L, rb, smem, a.k / 128, wave, grp, acc);
    if constexpr (NB == 2) {
        barrier_lds(); // every wave's operand and scale reads are done
        expert_store<128>(a, smem + wave * kOwnBytes, row0, M, n0, wave, lane,
                          [&](int q, int i, int t) { return acc[q][i][t]; });
    } else {
        expert_store128(a, smem, row0, M, n0, wave, lane,
                        [&](int i, int t) { return acc[0][i][t]; });
    }
}

// 256x256 tiles; of an expert's last, if at most 128 rows are left, the upper half alone.
template <bool GATHER>
__global__ __attribute__((amdgpu_flat_work_group_size(pp::kNT, pp::kNT), amdgpu_waves_per_eu(2, 2)))
void experts_tile_kernel(ga_experts_product_args a, int tn)
{
    using namespace bspp;
    constexpr int kLds = std::max(kLdsBs + 8 * kOwnBytes, BsHalfCfg<2>::kLds);
    static_assert(kLds <= 160 * 1024, "LDS budget");
    __shared__ __attribute__((aligned(1024))) char smem[kLds];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wave >> 2, simd = wave & 3;
    ExpertTile x;
    int tile_m, tile_n;
    if (!expert_tile(a, 256, tn, lane, kExpertBand, x, tile_m, tile_n))
        return;
    const int row0 = x.first + tile_m * 256, n0 = tile_n * 256;
    const int M = min(256, x.last - row0);
    if (M <= 128) {
        expert_half_tile<2, GATHER>(a, smem, x.expert, row0, M, n0, wave, lane);
        return;
    }

    v4f acc[4][4][2];
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int t = 0; t < 2; t++)
                acc[q][i][t] = (v4f){0.f, 0.f, 0.f, 0.f};
    ExpertLoad<GATHER> L;
    expert_load_setup<256, 2>(a, x.expert, row0, M, n0, wave, lane, L);
    const BsRead rb = expert_read_setup(smem, lane, grp, simd, kBRegion, kSBase);
    bs_pp_chain<PS_GROUP128>(L, rb, smem, a.k / 128, wave, grp, acc);
    expert_store<256>(a, smem + kLdsBs + wave * kOwnBytes, row0, M, n0, wave, lane,
                      [&](int q, int i, int t) { return acc[q][i][t]; });
}

template <int NB, bool GATHER>
__global__ __attribute__((amdgpu_flat_work_group_size(pp::kNT, pp::kNT), amdgpu_waves_per_eu(2, 2)))
void experts_half_kernel(ga_experts_product_args a, int tn)
{
    __shared__ __attribute__((aligned(1024))) char smem[bspp::BsHalfCfg<NB>::kLds];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    ExpertTile x;
    int tile_m, tile_n;
    if (!expert_tile(a, 128, tn, lane, kExpertBand, x, tile_m, tile_n))
        return;
    const int row0 = x.first + tile_m * 128;
    expert_half_tile<NB, GATHER>(a, smem, x.expert, row0, min(128, x.last - row0),
                                 tile_n * 128 * NB, wave, lane);
}

template <bool GATHER>
ga_status launch_tiles(const ga_experts_product_args& a, int height, int width, hipStream_t st)
{
    const int tn = (a.n - 1) / width + 1;
    const long long grid = most_expert_tiles(a.rows, a.experts, height) * tn;
    if (grid > most_workgroups(pp::kNT))
        return fail(GA_ERR_SHAPE, "experts_product: too many tiles for one call");
    const dim3 g((unsigned)grid), b(pp::kNT);
    if (height == 256)
        hipLaunchKernelGGL((experts_tile_kernel<GATHER>), g, b, 0, st, a, tn);
    else if (width == 256)
        hipLaunchKernelGGL((experts_half_kernel<2, GATHER>), g, b, 0, st, a, tn);
    else
        hipLaunchKernelGGL((experts_half_kernel<1, GATHER>), g, b, 0, st, a, tn);
    GA_HIP_CHECK(hipGetLastError());
    return GA_OK;
}

// How a product is cut: a workgroup's rows and columns, its slices of K (0: an eight-wave tile),
// how many a CU has at a time, its start and its time for a 128-K step in us, and a CU's time for
// a whole tile's 128 of K when all CUs are busy for long.
struct ExpertCut {
    int height, width, ks, at_once;
    float start, step, full;
};

// The cut with the smallest estimated time. The counts are on the GPU, so the tiles are those of
// rows spread over the experts by chance, and all rows count as live: of a process that holds some of the
// experts they are too many (1/2, 1/4, 1/8 of them held, 120 problems by chance: 8, 11, 10 % slower than
// the fastest cut on average, at the worst 1.95 times; `cut` names another). A call takes its rounds of workgroups (a last one that is
// not full counts as between its part and a whole one) or, where that is longer, its tiles at full
// rate; about where they are equal it takes longer than both, as the fourth root of the sum of
// fourth powers does. The coefficients are a fit to 2359 problems measured on MI355X with every
// cut (2-256 experts, 1-4000 rows each, N 64-7168, K 256-7168): the cut it picks is on average 2 %
// slower than the fastest, at the worst 1.43 times, of 99 in 100 at most 1.26; of 200 others by chance,
// K from 128 on, 5 %, at the worst 1.31. One cut for all takes 1.34 (64x64) to 1.92 (16x32)
// times the fastest on average: 256 experts of 7168x512 with 4 rows each take 132 us in
// 16x256, 250 in 128x256, 342 in 16x32 workgroups; 8 of 2048x7168 with 300 rows 173 in 16x32, 62 in
// 128x256, 83 in 256x256; 64 of 4096x4096 with 64 rows 498, 198, 198, and 285 in 64x256; with 1024
// rows 6450, 1315, 1100; 60 of 99x6272 with 1354 rows 400, 143, 151, and 104 in 128x128.
const ExpertCut& expert_cut(const ga_experts_product_args& a, int num_cu)
{
    static const ExpertCut kCuts[GA_EXPERTS_CUTS] = {
        {16, 64, 2, 2, 3.83f, 0.14f, 0.15f},   {16, 32, 4, 2, 3.60f, 0.26f, 0.12f},
        {16, 256, 1, 2, 2.14f, 0.43f, 0.96f},  {64, 256, 1, 2, 3.41f, 1.31f, 0.84f},
        {64, 64, 4, 2, 4.14f, 0.61f, 0.37f},   {128, 128, 0, 1, 2.39f, 0.39f, 0.59f},
        {128, 256, 0, 1, 3.49f, 0.63f, 0.75f}, {256, 256, 0, 1, 3.62f, 1.03f, 0.88f}};
    if (a.cut)
        return kCuts[a.cut - 1];
    const double rows = a.rows;
    const double active = a.experts * (1.0 - std::exp(-rows / a.experts));
    const ExpertCut* best = nullptr;
    double least = 0.0;
    for (const ExpertCut& c : kCuts) {
        const double tiles = std::max(active, rows / c.height + 0.5 * active);
        const double groups = tiles * ((a.n - 1) / c.width + 1);
        const int slices = std::max(1, c.ks), steps = (a.k / 128 + slices - 1) / slices;
        const double part = groups / (num_cu * c.at_once);
        const double rounds = part > 1.0 ? 0.5 * (part + std::ceil(part)) : 1.0;
        const double in_rounds = rounds * (c.start + steps * c.step);
        const double at_full = groups / num_cu * (a.k / 128) * c.full;
        const double t = in_rounds * in_rounds * in_rounds * in_rounds +
                         at_full * at_full * at_full * at_full;
        if (!best || t < least) {
            best = &c;
            least = t;
        }
    }
    return *best;
}

} // namespace
} // namespace ga

using namespace ga;

extern "C" ga_status ga_experts_product(const ga_experts_product_args* args, void* stream)
{
    if (!args)
        return fail(GA_ERR_ARG, "experts_product: null argument");
    const ga_experts_product_args& a = *args;
    if (a.experts <= 0 || a.rows < 0 || a.n <= 0 || a.k <= 0 || a.a_rows < 0 || a.cut < 0 ||
        a.cut > GA_EXPERTS_CUTS)
        return fail(GA_ERR_ARG, "experts_product: bad count");
    if (a.experts > GA_EXPERTS_MAX || a.rows > 0x7FFF0000)
        return fail(GA_ERR_SHAPE, "experts_product: more than %d experts or 0x7FFF0000 rows",
                    GA_EXPERTS_MAX);
    if (a.k % 128)
        return fail(GA_ERR_GROUP, "K must be a multiple of GROUP_K (128), got %d", a.k);
    if (a.rows == 0)
        return GA_OK;
    if (!a.a || !a.sfa || !a.b || !a.sfb || !a.starts || !a.out)
        return fail(GA_ERR_ARG, "experts_product: null pointer");
    if ((uintptr_t)a.out % 2)
        return fail(GA_ERR_SHAPE, "experts_product: out must have its elements' alignment");
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
    int num_cu = 0;
    const ga_status status = device_cu_count(&num_cu);
    if (status != GA_OK)
        return status;
    const ExpertCut& c = expert_cut(a, num_cu);
    if (c.ks == 0)
        return a.rows_of ? launch_tiles<true>(a, c.height, c.width, st)
                         : launch_tiles<false>(a, c.height, c.width, st);
    if (c.height == 64)
        return launch_few<4, 4>(a, c.ks, st);
    return c.ks == 1 ? launch_few<1, 4>(a, c.ks, st) : launch_few<1, 2>(a, c.ks, st);
}

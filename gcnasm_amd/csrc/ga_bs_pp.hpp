// ga_bs_pp.hpp -- pieces of the eight-wave fp32-scaled FP8 GEMMs (gemm_bs_pp.hip:
// one tile per workgroup; gemm_bs_sk.hip: stream-K; gemm_experts.hip: experts'
// rows): the LDS plan, the copies of A, B and the scales, the operand reads, the
// scale fold, one quadrant's MFMA slot, and the chains of a 256x256 tile and of
// tiles of 128 rows.
#pragma once

#include "ga_device.hpp"
#include "ga_pp.hpp"

namespace ga {
namespace bspp {

using namespace pp;

enum { PS_GROUP128 = 0, PS_GROUP1 = 1, PS_TENSOR = 2 };

constexpr int kSSlot = 2048; // SFA (1 KB) + SFB (1 KB) of one K group
constexpr int kSRing = 4;    // scale slots: group s in slot s % 4
constexpr int kSBase = kOperandBytes;
constexpr int kLdsBs = kSBase + kSRing * kSSlot;
static_assert(kLdsBs <= 160 * 1024, "LDS budget");
constexpr int kBsGroupM = 4;
// fp32 epilogue staging: 128 rows of 1024 + 16 bytes (the 16 rows of one
// ds_write_b128 quarter-wave start 4 banks apart).
constexpr int kStagePitchF32 = 1040;

struct BsLoad {
    __amdgpu_buffer_rsrc_t ra, rb, rs; // rs: SFA (waves 0-3) or SFB (waves 4-7)
    uint32_t va, vb, vs;               // per-lane offsets (half 0, copy 0, K group 0)
    uint32_t a_hstep, b_hstep;         // bytes between copies 0 and 1 (64 rows)
    uint32_t s_kstep;                  // scale bytes per K group
};

// The copies take their wave-uniform offsets in the SGPR soffset: the
// VALU adds they cost as VGPR offsets sit in a loop whose time is VALU and
// MFMA issue (block scale 8192^3 on the reference driver's data 440.6 ->
// 437.4 us, 4096x2112x7168 77.6 -> 76.6 us on one box; the MXFP8 and MXFP4
// kernel ran slower that way and keeps VGPR offsets).
__device__ __forceinline__ void issue_a(const BsLoad& L, char* smem, int h, int t, int wave)
{
    char* dst = smem + kARegion + (t & 1) * kOpSlot + h * kHalf + wave * 1024;
    const uint32_t o = (uint32_t)h * 2 * L.a_hstep + (uint32_t)t * 128;
    lds_load16(L.ra, (lds_void*)dst, L.va, uni(o));
    lds_load16(L.ra, (lds_void*)(dst + 8192), L.va, uni(o + L.a_hstep));
}

__device__ __forceinline__ void issue_b(const BsLoad& L, char* smem, int h, int t, int wave)
{
    char* dst = smem + kBRegion + (t & 1) * kOpSlot + h * kHalf + wave * 1024;
    const uint32_t o = (uint32_t)h * 2 * L.b_hstep + (uint32_t)t * 128;
    lds_load16(L.rb, (lds_void*)dst, L.vb, uni(o));
    lds_load16(L.rb, (lds_void*)(dst + 8192), L.vb, uni(o + L.b_hstep));
}

// Scales of K group t into ring slot `ring`: one 4-byte copy per lane.
__device__ __forceinline__ void issue_s(const BsLoad& L, char* smem, int t, int ring, int wave)
{
    char* dst = smem + kSBase + ring * kSSlot + wave * 256;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(L.rs, (lds_void*)dst, 4, L.vs,
                                             uni((uint32_t)t * L.s_kstep), 0, 0);
}

struct BsRead {
    const char* a0;
    const char* a1;
    const char* b0;
    const char* b1;
    const char* sa; // this lane's four rows of group grp
    const char* sb; // GROUP_N 1: this lane's four columns of tile 0 (simd block)
};

template <int H>
__device__ __forceinline__ void read_a(const BsRead& rb, int slot, v8i (&a)[4])
{
    const int off = kARegion + slot * kOpSlot + H * kHalf;
#pragma unroll
    for (int i = 0; i < 4; i++)
        a[i] = lds_frag(rb.a0 + off + i * 2048, rb.a1 + off + i * 2048);
}

template <int H>
__device__ __forceinline__ void read_b(const BsRead& rb, int slot, v8i (&b)[2])
{
    const int off = slot * kOpSlot + H * kHalf; // base includes the B region
#pragma unroll
    for (int t = 0; t < 2; t++)
        b[t] = lds_frag(rb.b0 + off + t * 2048, rb.b1 + off + t * 2048);
}

// Scales of quadrant (HM, HN) of the K group in ring slot `ring`: this
// lane's four SFA rows and its SFB value(s).
struct ScaleVals {
    v4f sa;
    v4f sb0, sb1; // GROUP_N 1: columns of tiles 0 and 1; GROUP_N 128: sb0[0]
};

template <int MODE, int HM, int HN>
__device__ __forceinline__ ScaleVals read_scales(const BsRead& rb, int ring)
{
    ScaleVals v;
    if constexpr (MODE != PS_TENSOR) {
        v.sa = *(const v4f*)(rb.sa + ring * kSSlot + HM * 2 * 256);
        if constexpr (MODE == PS_GROUP128) {
            v.sb0[0] = *(const float*)(rb.sb + ring * kSSlot + HN * 4);
        } else {
            const char* sbp = rb.sb + ring * kSSlot + HN * 128 * 4;
            v.sb0 = *(const v4f*)sbp;
            v.sb1 = *(const v4f*)(sbp + 64);
        }
    }
    return v;
}

// acc += p * (SFA * SFB), the product rounded to fp32 first.
template <int MODE>
__device__ __forceinline__ void apply_scales(const ScaleVals& v, v4f (&acc)[4][2],
                                             const v4f (&p)[4][2])
{
    if constexpr (MODE == PS_GROUP128) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float s = v.sa[i] * v.sb0[0];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    acc[i][t][j] = __builtin_fmaf(p[i][t][j], s, acc[i][t][j]);
        }
    } else if constexpr (MODE == PS_GROUP1) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                acc[i][0][j] = __builtin_fmaf(p[i][0][j], v.sa[i] * v.sb0[j], acc[i][0][j]);
                acc[i][1][j] = __builtin_fmaf(p[i][1][j], v.sa[i] * v.sb1[j], acc[i][1][j]);
            }
    }
}

// The tiles of a quadrant with t = 1 (GROUP_N 128), folded by the memory
// slot that follows the quadrant's MFMA slot when the fold is split.
template <int MODE>
__device__ __forceinline__ void apply_scales_t1(const ScaleVals& v, v4f (&acc)[4][2],
                                                const v4f (&p)[4][2])
{
    static_assert(MODE == PS_GROUP128, "split fold: one SFB value per quadrant");
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float s = v.sa[i] * v.sb0[0];
#pragma unroll
        for (int j = 0; j < 4; j++)
            acc[i][1][j] = __builtin_fmaf(p[i][1][j], s, acc[i][1][j]);
    }
}

// MFMA slot: the quadrant's 8 MFMAs (4 A tiles x 2 B tiles of one 128-K
// group; unit E8M0 scales). For the block-scale modes each MFMA writes a
// zeroed temporary p[i][t], and just before it the previous quadrant's
// p[i][t] is folded into its accumulator (acc += p * SFA*SFB): the VALU work
// of a tile issues while the MFMA pipe runs the previous tile's MFMA. With
// SPLIT only the t = 0 tiles are folded here; the memory slot before this
// one folded the t = 1 tiles (BS_MEM_SLOT_SPLIT). The B tiles alternate
// direction from one A tile to the next, so consecutive MFMAs differ in one
// operand (fewer operand bits change in the MFMA pipe; every tile's fold
// still comes just before its own MFMA).
template <int MODE, bool APPLY, bool SPLIT = false>
__device__ __forceinline__ void mma_quadrant(v4f (&acc)[4][2], v4f (&p)[4][2], const v8i (&a)[4],
                                             const v8i (&b)[2], v4f (&acc_prev)[4][2],
                                             const ScaleVals& sv)
{
    static_assert(!SPLIT || MODE == PS_GROUP128, "split fold: GROUP_N 128 only");
    __builtin_amdgcn_s_setprio(1);
    static_for<4>([&](auto I) {
        constexpr int i = decltype(I)::value;
        static_for<2>([&](auto T) {
            constexpr int t = (i & 1) ? 1 - decltype(T)::value : decltype(T)::value;
            constexpr bool fold = APPLY && !(SPLIT && t == 1);
            if constexpr (MODE == PS_TENSOR) {
                acc[i][t] = mfma_mx16<0, 0>(b[t], a[i], acc[i][t], 127, 127);
            } else {
                // keep the order fold(tile) -> MFMA(tile), tile by tile
                if constexpr (fold)
                    __builtin_amdgcn_sched_group_barrier(
                        0x2, MODE == PS_GROUP128 ? (t == 0 ? 5 : 4) : 8, 0);
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                if constexpr (fold) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float s = MODE == PS_GROUP128 ? sv.sa[i] * sv.sb0[0]
                                                            : sv.sa[i] * (t ? sv.sb1[j] : sv.sb0[j]);
                        acc_prev[i][t][j] = __builtin_fmaf(p[i][t][j], s, acc_prev[i][t][j]);
                    }
                }
                p[i][t] = mfma_mx16<0, 0>(b[t], a[i], (v4f){0.f, 0.f, 0.f, 0.f}, 127, 127);
            }
        });
    });
    __builtin_amdgcn_s_setprio(0);
}

// Memory slot: the copy, the scales of the quadrant the next MFMA slot
// folds in, then the operand read (the MFMA slot's first fold waits only for
// the scale reads, each MFMA only for its own operand), then the phase
// boundary.
#define BS_MEM_SLOT(HMP, HNP, RING, COPIES, READS, WAITN)                                    \
    {                                                                                        \
        COPIES;                                                                              \
        sv = read_scales<MODE, HMP, HNP>(rb, RING);                                          \
        __builtin_amdgcn_sched_barrier(0);                                                   \
        READS;                                                                               \
        __builtin_amdgcn_sched_barrier(0);                                                   \
        phase_sync<WAITN>();                                                                 \
    }

// Memory slot of the split fold (GROUP_N 128): the scales of quadrant (HM,
// HN), which the coming MFMA slot computes, are read one memory slot ahead
// into `svn`; the scales read by the previous memory slot (`sv`) serve this
// slot's fold of the t = 1 tiles of ACCP, the quadrant the previous MFMA
// slot computed, after the operand reads, and the coming MFMA slot's fold of
// its t = 0 tiles. Half of the fold's VALU work so leaves the MFMA slot
// without delaying the operand reads.
#define BS_MEM_SLOT_SPLIT(HM, HN, RING, COPIES, READS, WAITN, ACCP, DOFOLD)                  \
    {                                                                                        \
        sv = svn;                                                                            \
        COPIES;                                                                              \
        svn = read_scales<MODE, HM, HN>(rb, RING);                                           \
        __builtin_amdgcn_sched_barrier(0);                                                   \
        READS;                                                                               \
        __builtin_amdgcn_sched_barrier(0);                                                   \
        if (DOFOLD)                                                                          \
            apply_scales_t1<MODE>(sv, ACCP, p);                                              \
        __builtin_amdgcn_sched_barrier(0);                                                   \
        phase_sync<WAITN>();                                                                 \
    }

// The chain of a 256x256 tile: acc += the products of nsteps 128-K groups, for block scale with
// its scales. Load has the copies (issue_a, issue_b, issue_s).
template <int MODE, class Load>
__device__ __forceinline__ void bs_pp_chain(const Load& L, const BsRead& rb, char* smem, int nsteps,
                                            int wave, int grp, v4f (&acc)[4][4][2])
{
    constexpr int S = MODE == PS_TENSOR ? 0 : 1; // scale copies per wave per K group
    v4f p[4][2]; // MFMA results of the last quadrant, folded before the next MFMA slot reuses them
    v8i fa[4], fb0[2], fb1[2];

    // Prologue: copies in steady-state order (B0+S, A0, B1, A1 of group 0;
    // B0+S, A0, B1 of group 1), then the B0 read of the phase before step 0.
    issue_b(L, smem, 0, 0, wave);
    if (S)
        issue_s(L, smem, 0, 0, wave);
    issue_a(L, smem, 0, 0, wave);
    issue_b(L, smem, 1, 0, wave);
    issue_a(L, smem, 1, 0, wave);
    issue_b(L, smem, 0, 1, wave);
    if (S)
        issue_s(L, smem, 1, 1, wave);
    issue_a(L, smem, 0, 1, wave);
    issue_b(L, smem, 1, 1, wave);
    phase_sync<12 + S>(); // B0 (+ scales) of group 0
    read_b<0>(rb, 0, fb0);
    phase_sync<10 + S>(); // A0 of group 0
    if (grp == 1)
        slot_sync(); // second group runs one barrier behind

    // K group s (LDS slot s & 1, scale ring slot r0). A memory slot issues
    // its copy, reads scales, then its operand read, then waits:
    //   phase  read      copy            quadrant   younger copies
    //   1      A0(s)     A1(s+1)         00         10 + S
    //   2      B1(s)     B0+S(s+2)       01         10 + 2S
    //   3      A1(s)     A0(s+2)         10         10 + S
    //   4      B0(s+1)   B1(s+2)         11         10 + S
    // The loop's first quadrant has nothing to fold in: peel it.
    // Scale ring slot of group s: s % 4. The copy of group s+2 (phase 2 of
    // group s) overwrites group s-2's slot, last read for the fold in phase 1
    // of group s-1 (unsplit fold) or in phase 4 of group s-2 (split).
    ScaleVals sv;
    if constexpr (MODE == PS_GROUP128) {
        // Split fold: each memory slot reads the scales of the quadrant the
        // coming MFMA slot computes and folds the t = 1 tiles of the quadrant
        // the previous MFMA slot computed after its operand reads; the MFMA
        // slot folds the t = 0 tiles between its MFMAs. Phase 1 reads group
        // s's scales, which landed before A0(s) (copied after them), and the
        // last read of a ring slot (phase 4 of its group) precedes its
        // overwrite (phase 2 of the group two later). Same fmaf per tile and
        // group, in the same order, as the unsplit fold.
        ScaleVals svn = {};
        sv = svn;
        // two K groups per iteration: the LDS slot is a compile-time read
        // offset instead of a VALU add per read base
        auto group = [&](int s, auto SLOT) {
            constexpr int slot = decltype(SLOT)::value;
            const int r0 = s & 3, r2 = (s + 2) & 3;
            // phase 1 (folds in quadrant 11 of the previous group)
            BS_MEM_SLOT_SPLIT(0, 0, r0, issue_a(L, smem, 1, s + 1, wave),
                              read_a<0>(rb, slot, fa), 10 + S, acc[3], s > 0);
            if (s > 0)
                mma_quadrant<MODE, true, true>(acc[0], p, fa, fb0, acc[3], sv);
            else
                mma_quadrant<MODE, false, true>(acc[0], p, fa, fb0, acc[3], sv);
            slot_sync();
            // phase 2
            BS_MEM_SLOT_SPLIT(0, 1, r0,
                              issue_b(L, smem, 0, s + 2, wave);
                              issue_s(L, smem, s + 2, r2, wave), read_b<1>(rb, slot, fb1),
                              10 + 2 * S, acc[0], true);
            mma_quadrant<MODE, true, true>(acc[1], p, fa, fb1, acc[0], sv);
            slot_sync();
            // phase 3
            BS_MEM_SLOT_SPLIT(1, 0, r0, issue_a(L, smem, 0, s + 2, wave),
                              read_a<1>(rb, slot, fa), 10 + S, acc[1], true);
            mma_quadrant<MODE, true, true>(acc[2], p, fa, fb0, acc[1], sv);
            slot_sync();
            // phase 4
            BS_MEM_SLOT_SPLIT(1, 1, r0, issue_b(L, smem, 1, s + 2, wave),
                              read_b<0>(rb, slot ^ 1, fb0), 10 + S, acc[2], true);
            mma_quadrant<MODE, true, true>(acc[3], p, fa, fb1, acc[2], sv);
            slot_sync();
        };
        int s = 0;
        for (; s + 1 < nsteps; s += 2) {
            group(s, std::integral_constant<int, 0>{});
            group(s + 1, std::integral_constant<int, 1>{});
        }
        if (s < nsteps)
            group(s, std::integral_constant<int, 0>{});
        if (grp == 0)
            slot_sync(); // matches the second group's extra barrier
        apply_scales<MODE>(svn, acc[3], p);
    } else {
        auto group = [&](int s, auto SLOT) {
            const int slot = SLOT;
            const int r0 = s & 3, r2 = (s + 2) & 3, rprev = (s - 1) & 3;
            // phase 1 (folds in quadrant 11 of the previous group)
            BS_MEM_SLOT(1, 1, rprev, issue_a(L, smem, 1, s + 1, wave), read_a<0>(rb, slot, fa),
                        10 + S);
            if (s > 0)
                mma_quadrant<MODE, true>(acc[0], p, fa, fb0, acc[3], sv);
            else
                mma_quadrant<MODE, false>(acc[0], p, fa, fb0, acc[3], sv);
            slot_sync();
            // phase 2
            BS_MEM_SLOT(0, 0, r0,
                        issue_b(L, smem, 0, s + 2, wave); if (S) issue_s(L, smem, s + 2, r2, wave),
                        read_b<1>(rb, slot, fb1), 10 + 2 * S);
            mma_quadrant<MODE, true>(acc[1], p, fa, fb1, acc[0], sv);
            slot_sync();
            // phase 3
            BS_MEM_SLOT(0, 1, r0, issue_a(L, smem, 0, s + 2, wave), read_a<1>(rb, slot, fa),
                        10 + S);
            mma_quadrant<MODE, true>(acc[2], p, fa, fb0, acc[1], sv);
            slot_sync();
            // phase 4
            BS_MEM_SLOT(1, 0, r0, issue_b(L, smem, 1, s + 2, wave), read_b<0>(rb, slot ^ 1, fb0),
                        10 + S);
            mma_quadrant<MODE, true>(acc[3], p, fa, fb1, acc[2], sv);
            slot_sync();
        };
        if constexpr (MODE == PS_GROUP1) {
            // one group per iteration: two need more registers than there are
            // (832 spilled: 1536x8192x8192, bf16 C, 1457 us against 126 now)
            for (int s = 0; s < nsteps; s++)
                group(s, s & 1);
        } else {
            int s = 0;
            for (; s + 1 < nsteps; s += 2) {
                group(s, std::integral_constant<int, 0>{});
                group(s + 1, std::integral_constant<int, 1>{});
            }
            if (s < nsteps)
                group(s, std::integral_constant<int, 0>{});
        }
        if (grp == 0)
            slot_sync(); // matches the second group's extra barrier
        const ScaleVals last = read_scales<MODE, 1, 1>(rb, (nsteps - 1) & 3);
        apply_scales<MODE>(last, acc[3], p);
    }
    wait_vmcnt<0>(); // copies past K land before the LDS is used again, and before exit
}

template <int NB>
struct BsHalfCfg {
    static constexpr int kSlot = (1 + NB) * kHalf; // A, then the B halves
    static constexpr int NS = NB == 2 ? 3 : 4;
    static constexpr int kRing = NB == 2 ? 4 : 8; // scale slots: group s in s % kRing
    static constexpr int kScaleBase = NS * kSlot;
    static constexpr int kLds = kScaleBase + kRing * kSSlot;
    static_assert(kLds <= 160 * 1024, "LDS budget");
    static_assert(128 * kStagePitchF32 <= kLds && 128 * kStagePitch <= kLds, "staging fits");
    // a group's scales are folded one group late, and copied NS - 1 early
    static_assert(kRing > NS, "scale ring");
};

// Own copies older than the last N landed, own LDS reads complete, barrier.
template <int N>
__device__ __forceinline__ void half_sync()
{
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<N>();
    wait_lgkmcnt0();
    wait_lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

template <int NB, int MODE>
__device__ __forceinline__ void issue_half(const BsLoad& L, char* smem, int t, int slot, int wave)
{
    using H = BsHalfCfg<NB>;
    char* dst = smem + slot * H::kSlot + wave * 1024;
    const uint32_t o = (uint32_t)t * 128;
    lds_load16(L.ra, (lds_void*)dst, L.va + uni(o), 0);
    lds_load16(L.ra, (lds_void*)(dst + 8192), L.va + uni(o + L.a_hstep), 0);
#pragma unroll
    for (int c = 0; c < 2 * NB; c++)
        lds_load16(L.rb, (lds_void*)(dst + kHalf + c * 8192), L.vb + uni(o + c * L.b_hstep), 0);
    if constexpr (MODE != PS_TENSOR)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            L.rs,
            (lds_void*)(smem + H::kScaleBase + (t & (H::kRing - 1)) * kSSlot + wave * 256), 4,
            L.vs + uni((uint32_t)t * L.s_kstep), 0, 0, 0);
}

// The chain of a tile of 128 rows and NB * 128 columns, as bs_pp_chain (issue_half).
template <int NB, int MODE, class Load>
__device__ __forceinline__ void bs_half_chain(const Load& L, const BsRead& rb, char* smem,
                                              int nsteps, int wave, int grp, v4f (&acc)[NB][4][2])
{
    using H = BsHalfCfg<NB>;
    constexpr int NS = H::NS;
    constexpr int kC = 2 + 2 * NB + (MODE == PS_TENSOR ? 0 : 1); // copies per wave and group
    v4f p[NB][4][2];
    v8i fa[4], fb[NB][2];
    ScaleVals sv[NB];
    auto scales = [&](int s) { // of group s
        const int ring = s & (H::kRing - 1);
        sv[0] = read_scales<MODE, 0, 0>(rb, ring);
        if constexpr (NB == 2)
            sv[1] = read_scales<MODE, 0, 1>(rb, ring);
    };

    static_for<NS - 1>([&](auto J) {
        constexpr int j = decltype(J)::value;
        issue_half<NB, MODE>(L, smem, j, j, wave);
    });
    half_sync<kC*(NS - 2)>();
    if (grp == 1)
        slot_sync(); // second group runs one barrier behind

    // Group s in slot S = s % NS: copies of group s + NS - 1 into the slot of
    // group s - 1, whose last reads (the second wave group's) ended one barrier
    // ago. Waiting for all but the newest NS - 2 groups' copies after the memory
    // half retires group s + 1's, read two barriers on at the earliest. The
    // scales of group s - 1 are read here and their slot is copied into again
    // at the earliest in group s + 1.
    auto step = [&](int s, auto SC) {
        constexpr int S = decltype(SC)::value;
        issue_half<NB, MODE>(L, smem, s + NS - 1, (S + NS - 1) % NS, wave);
        if (s > 0)
            scales(s - 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; i++)
            fa[i] = lds_frag(rb.a0 + S * H::kSlot + i * 2048, rb.a1 + S * H::kSlot + i * 2048);
#pragma unroll
        for (int q = 0; q < NB; q++)
#pragma unroll
            for (int t = 0; t < 2; t++)
                fb[q][t] = lds_frag(rb.b0 + S * H::kSlot + q * kHalf + t * 2048,
                                    rb.b1 + S * H::kSlot + q * kHalf + t * 2048);
        __builtin_amdgcn_sched_barrier(0);
        if (s > 0)
#pragma unroll
            for (int q = 0; q < NB; q++)
                apply_scales<MODE>(sv[q], acc[q], p[q]);
        half_sync<kC*(NS - 2)>();
#pragma unroll
        for (int q = 0; q < NB; q++)
            mma_quadrant<MODE, false>(acc[q], p[q], fa, fb[q], acc[q], sv[q]);
        half_sync<kC*(NS - 2)>();
    };
    int s = 0;
    for (; s + NS <= nsteps; s += NS)
        static_for<NS>([&](auto J) {
            constexpr int j = decltype(J)::value;
            step(s + j, std::integral_constant<int, j>{});
        });
    static_for<NS - 1>([&](auto J) {
        constexpr int j = decltype(J)::value;
        if (s + j < nsteps)
            step(s + j, std::integral_constant<int, j>{});
    });
    if (grp == 0)
        slot_sync(); // matches the second group's extra barrier
    if constexpr (MODE != PS_TENSOR) {
        scales(nsteps - 1);
#pragma unroll
        for (int q = 0; q < NB; q++)
            apply_scales<MODE>(sv[q], acc[q], p[q]);
    }
    wait_vmcnt<0>(); // copies past K land before the LDS is used again, and before exit
}

} // namespace bspp
} // namespace ga

// ga_bs_decode.hpp -- the pieces that the few-row FP8 GEMMs with fp32 scales share
// (gemm_bs_decode.hip: one matrix; gemm_experts.hip: an expert's rows): the
// ring of a wave in LDS, its chain of 128-K steps, the sum of the K slices.
#pragma once

#include "ga_device.hpp"
#include "ga_pp.hpp"

namespace ga {

enum { BD_GROUP128 = 0, BD_GROUP1 = 1, BD_TENSOR = 2 };

// A wave's operands of one 128-K step in LDS: 16-row blocks of 2 KB, TM of A
// then NG of B, each 16 rows of 128 bytes with 16-byte K chunk c of row r at
// slot c ^ ((r >> 1) & 7); then the step's scales, 64 dwords of SFA (one per
// row) and 64 of SFB. D such steps make the wave's ring.
template <int TM, int NG>
struct BdCfg {
    static constexpr int kScales = (TM + NG) * 2048;
    static constexpr int kStep = kScales + 512;
    static constexpr int kMax = 20480; // 8 waves in 160 KB
    static constexpr int D = kMax / kStep;
    static constexpr int kWave = D * kStep > TM * NG * 1024 ? D * kStep : TM * NG * 1024;
    static_assert(D >= 1 && kWave <= kMax, "LDS budget");
};

__device__ __forceinline__ uint32_t bd_uni(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// The chain of a wave: acc += the products of nsteps steps, which
// load(step, slot) copies into a ring slot (kLoads copy instructions each).
template <int TM, int NG, int MODE, class Load>
__device__ __forceinline__ void bd_chain(char* ring, int lane, int nsteps, const Load& load,
                                         v4f (&acc)[NG][TM])
{
    using Cfg = BdCfg<TM, NG>;
    constexpr int D = Cfg::D;
    constexpr int kLoadsPerStep = 2 * NG + 2 * TM + (MODE == BD_TENSOR ? 0 : 2);
    static_assert(kLoadsPerStep * (D - 1) < 64, "vmcnt range");
    const int r = lane & 15, g = lane >> 4;
    uint32_t o0, o1;
    pp::operand_lane(lane, o0, o1);
    // the step in slot j (its copies have landed): fragments and scales
    // out, then, once every one has been read, the slot's next step `next`
    // in (negative: none), then the products
    auto step = [&](int next, auto J) {
        const char* q = ring + decltype(J)::value * Cfg::kStep;
        v8i fa[TM], fb[NG];
        float sa[TM];
        v4f sb[NG];
#pragma unroll
        for (int c = 0; c < NG; c++)
            fb[c] = pp::lds_frag(q + (TM + c) * 2048 + o0, q + (TM + c) * 2048 + o1);
#pragma unroll
        for (int i = 0; i < TM; i++)
            fa[i] = pp::lds_frag(q + i * 2048 + o0, q + i * 2048 + o1);
        if constexpr (MODE != BD_TENSOR) {
            const float* qs = (const float*)(q + Cfg::kScales);
#pragma unroll
            for (int i = 0; i < TM; i++)
                sa[i] = qs[i * 16 + r];
#pragma unroll
            for (int c = 0; c < NG; c++) {
                if constexpr (MODE == BD_GROUP128)
                    sb[c][0] = qs[64 + c];
                else
                    sb[c] = *(const v4f*)(qs + 64 + c * 16 + g * 4);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        wait_lgkmcnt0();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (next >= 0)
            load(next, ring + decltype(J)::value * Cfg::kStep);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < NG; c++)
#pragma unroll
            for (int i = 0; i < TM; i++) {
                if constexpr (MODE == BD_TENSOR) {
                    acc[c][i] = mfma_mx16<0, 0>(fb[c], fa[i], acc[c][i], 127, 127);
                } else {
                    const v4f p =
                        mfma_mx16<0, 0>(fb[c], fa[i], (v4f){0.f, 0.f, 0.f, 0.f}, 127, 127);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float sc = MODE == BD_GROUP128 ? sa[i] * sb[c][0] : sa[i] * sb[c][e];
                        acc[c][i][e] = __builtin_fmaf(p[e], sc, acc[c][i][e]);
                    }
                }
            }
        __builtin_amdgcn_sched_barrier(0);
    };

    // In the loop every step issues the copies of the step D ahead, so the
    // wait before a step leaves exactly the D - 1 younger steps in flight.
    // In the last whole block some steps have none to issue: the wait
    // counts only the block's own younger steps. What is left waits for
    // everything.
    static_for<D>([&](auto J) {
        if ((int)J < nsteps)
            load((int)J, ring + decltype(J)::value * Cfg::kStep);
        __builtin_amdgcn_sched_barrier(0);
    });
    int s = 0;
    for (; s + 2 * D <= nsteps; s += D)
        static_for<D>([&](auto J) {
            wait_vmcnt<kLoadsPerStep * (D - 1)>();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            step(s + D + (int)J, J);
        });
    if (s + D <= nsteps) {
        static_for<D>([&](auto J) {
            wait_vmcnt<kLoadsPerStep * (D - 1 - decltype(J)::value)>();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            const int next = s + D + (int)J;
            step(next < nsteps ? next : -1, J);
        });
        s += D;
    }
    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    static_for<D>([&](auto J) {
        if ((int)J < nsteps - s)
            step(-1, J);
    });
}

// K slices of a column group summed in slice order, the group's 16x16 tiles
// shared out over its ks waves: wave `slice` sums and stores tiles slice, slice +
// ks, ... by store(column group, row block, sum). Every wave of the workgroup
// comes here; those that are not live store nothing.
template <int TM, int NG, class Store>
__device__ __forceinline__ void bd_join(char* smem, int wave, int lane, int slice, int tl, int ks,
                                        bool live, const v4f (&acc)[NG][TM], const Store& store)
{
    using Cfg = BdCfg<TM, NG>;
    constexpr int NT = NG * TM;
    float* mine = (float*)(smem + wave * Cfg::kWave);
#pragma unroll
    for (int c = 0; c < NG; c++)
#pragma unroll
        for (int i = 0; i < TM; i++)
            *(v4f*)(mine + (i * NG + c) * 256 + lane * 4) = acc[c][i];
    __syncthreads();
    if (!live)
        return;
    const char* part = smem + tl * ks * Cfg::kWave + lane * 16;
    for (int f = slice; f < NT; f += ks) {
        v4f t = *(const v4f*)(part + f * 1024);
        for (int z = 1; z < ks; z++) {
            const v4f u = *(const v4f*)(part + z * Cfg::kWave + f * 1024);
            t = (v4f){t[0] + u[0], t[1] + u[1], t[2] + u[2], t[3] + u[3]};
        }
        store(f % NG, f / NG, t);
    }
}

} // namespace ga

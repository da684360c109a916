// ga_experts.hpp -- which rows a tile of the experts' products has: the counts are on the GPU, so
// every workgroup works out its own from the experts' first rows.
#pragma once

#include "ga_device.hpp"

namespace ga {

// Tiles of `height` rows, an expert's one after the other: at most so many for `rows` rows of
// `experts` experts, since a tile that is not full is its expert's last.
inline long long most_expert_tiles(long long rows, long long experts, int height)
{
    const long long full = (rows + experts * (height - 1)) / height;
    return rows < full ? rows : full;
}

// Rows first .. last - 1 of an expert, which has `tiles` tiles; `before` tiles of experts before it.
struct ExpertTile {
    int expert, first, last;
    int before, tiles;
};

// Over the lanes up to this one; op(x, 0) = x.
template <class Op>
__device__ __forceinline__ int wave_scan(int x, const Op& op)
{
    auto dpp = [](int v, auto ctrl, auto rows) {
        return __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xF,
                                           true);
    };
    using std::integral_constant;
    x = op(x, dpp(x, integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{})); // row_shr 1
    x = op(x, dpp(x, integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{})); // 2
    x = op(x, dpp(x, integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{})); // 4
    x = op(x, dpp(x, integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{})); // 8
    x = op(x, dpp(x, integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{})); // row_bcast 15
    x = op(x, dpp(x, integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{})); // row_bcast 31
    return x;
}

// The tiles of all experts, and the expert of one of them. First rows are taken as the nearest of
// 0 .. rows, and where they decrease as the largest before, so that there are no more tiles than
// most_expert_tiles(). Every lane of a wave calls it: a lane has a run of P experts in registers, a
// scan over the wave gives the tiles before them. pick(total) says which tile (uniform; outside
// 0 .. total - 1: none, and false is returned).
template <int P, class Pick>
__device__ __forceinline__ bool find_expert_run(const int* __restrict__ starts, int experts, int rows,
                                                int height, int lane, const Pick& pick,
                                                ExpertTile& x)
{
    int s[P + 1];
#pragma unroll
    for (int i = 0; i <= P; i++)
        s[i] = starts[min(lane * P + i, experts)];
#pragma unroll
    for (int i = 0; i <= P; i++)
        s[i] = min(max(s[i], 0), rows);
    int largest = s[0]; // of this lane's run, the next one's first left out
#pragma unroll
    for (int i = 1; i < P; i++)
        largest = max(largest, s[i]);
    int before_run = __shfl_up(wave_scan(largest, [](int a, int b) { return max(a, b); }), 1, 64);
    before_run = lane > 0 ? before_run : 0;
    s[0] = max(s[0], before_run);
#pragma unroll
    for (int i = 1; i <= P; i++)
        s[i] = max(s[i], s[i - 1]);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < P; i++)
        mine += (s[i + 1] - s[i] + height - 1) / height;
    const int upto = wave_scan(mine, [](int a, int b) { return a + b; });
    const int total = __builtin_amdgcn_readlane(upto, 63);
    const int t = pick(total);
    if (t < 0 || t >= total)
        return false;
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > t));
    int before = upto - mine;
    ExpertTile o = {0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < P; i++) {
        const int n = (s[i + 1] - s[i] + height - 1) / height;
        if (before <= t && t < before + n)
            o = {lane * P + i, s[i], s[i + 1], before, n};
        before += n;
    }
    x.expert = __builtin_amdgcn_readlane(o.expert, l);
    x.first = __builtin_amdgcn_readlane(o.first, l);
    x.last = __builtin_amdgcn_readlane(o.last, l);
    x.before = __builtin_amdgcn_readlane(o.before, l);
    x.tiles = __builtin_amdgcn_readlane(o.tiles, l);
    return true;
}

template <class Pick>
__device__ __forceinline__ bool find_expert(const int* __restrict__ starts, int experts, int rows,
                                            int height, int lane, const Pick& pick, ExpertTile& x)
{
    static_assert(GA_EXPERTS_MAX <= 64 * 16, "a lane's run");
    if (experts <= 64)
        return find_expert_run<1>(starts, experts, rows, height, lane, pick, x);
    if (experts <= 256)
        return find_expert_run<4>(starts, experts, rows, height, lane, pick, x);
    return find_expert_run<16>(starts, experts, rows, height, lane, pick, x);
}

} // namespace ga

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

// Rows first .. last - 1 of expert e; `index` of this expert's `tiles` tiles, `before` tiles of
// experts before it.
struct ExpertTile {
    int expert, first, last;
    int before, tiles;
};

// The expert that tile t of those of all experts belongs to. First rows are taken as the nearest of
// 0 .. rows, an expert whose end lies before its start has none. total: all tiles. Every lane of a
// wave calls it, and everything it returns is uniform. t >= total: nothing.
// A lane has a run of experts, one scan over the wave gives the tiles before them.
__device__ __forceinline__ ExpertTile find_expert(const int* __restrict__ starts, int experts,
                                                  int rows, int height, int lane, int t, int* total)
{
    const int per = (experts + 63) / 64;
    const int e0 = min(experts, lane * per), e1 = min(experts, e0 + per);
    int mine = 0;
    const int from = min(max(starts[e0], 0), rows);
    int f = from;
    for (int e = e0; e < e1; e++) {
        const int to = min(max(starts[e + 1], 0), rows);
        mine += (max(to - f, 0) + height - 1) / height;
        f = to;
    }
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d, 64);
        upto += lane >= d ? o : 0;
    }
    *total = __builtin_amdgcn_readlane(upto, 63);
    ExpertTile x = {0, 0, 0, 0, 0};
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > t);
    if (past == 0)
        return x;
    const int l = __builtin_ctzll(past);
    // the run of lane l, again, by every lane
    int e = __builtin_amdgcn_readlane(e0, l);
    int before = __builtin_amdgcn_readlane(upto - mine, l);
    f = __builtin_amdgcn_readlane(from, l);
    for (;; e++) {
        const int to = min(max(__builtin_amdgcn_readfirstlane(starts[e + 1]), 0), rows);
        const int n = (max(to - f, 0) + height - 1) / height;
        if (before + n > t) {
            x.expert = e;
            x.first = f;
            x.last = to;
            x.before = before;
            x.tiles = n;
            return x;
        }
        before += n;
        f = to;
    }
}

} // namespace ga

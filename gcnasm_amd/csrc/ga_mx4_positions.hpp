// ga_mx4_positions.hpp -- which tokens of the MXFP4 cache rows see (plain C++, host and device).
//
// Row i of a sequence's n rows over len tokens stands at position len - n + i, which is negative
// where there are more rows than tokens, and sees the tokens t with
//   t <= last_seen(position),  t > before_first(position).
// The window is any int from 0 on (0: none): it is taken off the position only where that leaves
// 32 bits enough, so 2^31 - 1 is a window that hides nothing.
#pragma once

#include "ga_extent.hpp"

namespace ga {

constexpr GA_HOST_DEVICE int last_seen(int pos, int len, bool causal)
{
    return causal && pos < len - 1 ? pos : len - 1;
}

constexpr GA_HOST_DEVICE int before_first(int pos, int window)
{
    const int at = pos > -1 ? pos : -1;
    return window && at - window > -1 ? at - window : -1;
}

// What rows i0 .. i1 see: the least and the greatest of both bounds.
struct Seen {
    int hi_min, hi_max, lo_min, lo_max;
    GA_HOST_DEVICE Seen(int len, int n, int i0, int i1, bool causal, int window)
        : hi_min(last_seen(len - n + i0, len, causal)),
          hi_max(last_seen(len - n + i1, len, causal)),
          lo_min(before_first(len - n + i0, window)), lo_max(before_first(len - n + i1, window))
    {
    }
    // the tokens that some row sees: [begin, end), begin a multiple of 64
    GA_HOST_DEVICE int begin() const { return (lo_min + 1) & ~63; }
    GA_HOST_DEVICE int end() const { return hi_max + 1; }
};

// One of `parts` alike stretches of n tokens, [lo, hi): `rows` times 64, the last time maybe fewer.
struct Stretch {
    int lo, hi, rows;
    GA_HOST_DEVICE Stretch(int n, int part, int parts)
    {
        const int most = (n + 64 * parts - 1) / (64 * parts) * 64;
        lo = part * most < n ? part * most : n;
        hi = n - lo < most ? n : lo + most;
        rows = (hi - lo + 63) / 64;
    }
};

} // namespace ga

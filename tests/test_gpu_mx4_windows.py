"""Windows over the MXFP4 cache so large that they hide nothing, up to and past the largest int, as
"no limit" is written, with fewer tokens than rows among them: what no window gives."""
import sys

import numpy as np
import pytest
import torch

from gcnasm_amd import mx4_cache as mc
from test_gpu_mx4_cache import Setup, host

pytestmark = pytest.mark.gpu

WINDOWS = [1 << 30, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, sys.maxsize]
SHAPES = [([3, 7], [9, 7], 4, 2, 128, 16), ([3, 0, 1], [5, 4, 1], 4, 2, 64, 16),
          ([700, 3, 129], [1, 1, 1], 6, 2, 256, 32), ([300, 20, 5], [250, 60, 70], 4, 2, 128, 64),
          ([130, 40], [129, 100], 2, 1, 64, 16), ([90], [100], 4, 2, 256, 64)]


@pytest.mark.parametrize("lens,rows,hq,h,D,P", SHAPES)
def test_windows_without_an_end(dev, lens, rows, hq, h, D, P):
    s = Setup(dev, lens, rows, hq, h, D, P, seed=31)
    parts = s.expected()
    starts = None if all(r == 1 for r in rows) else s.starts_d
    lse = torch.from_numpy(np.concatenate([p[1] for p in parts]).astype(np.float32)).to(dev)
    for window in WINDOWS:
        print("window", lens, rows, D, window, flush=True)
        s.check(*mc.attention(s.q, s.cache, s.table_d, s.lens_d, starts, window=window), parts)
        got = host(mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d, lse, q_starts=starts,
                                        window=window))
        for b, length in enumerate(lens):
            want = parts[b][2]
            # a term's score in fp32 and its exponential, 2^-14 of each (|score| < 64), and the sum
            tol = want * (2.0 ** -14 + rows[b] * hq * 2.0 ** -23) + 1e-30
            assert (np.abs(got[b, :, :length] - want) <= tol).all()
            assert (got[b, :, length:] == 0).all()


def test_bounds_past_an_int(dev):
    """max_q and max_len only choose the launch, whatever they are."""
    s = Setup(dev, [300, 20], [30, 7], 4, 2, 128, 64, seed=32)
    parts = s.expected()
    for bound in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1):
        s.check(*mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d, bound, bound), parts)


def test_sizes_past_an_int_are_refused(dev):
    s = Setup(dev, [20, 30], [1, 1], 4, 2, 128, 16, seed=33)
    w = torch.zeros((2, 2, 30), device=dev)
    lse = torch.zeros((2, 4), device=dev)
    with pytest.raises(ValueError):
        mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d, lse, width=2 ** 32 + 5)
    with pytest.raises(ValueError):
        mc.evict(s.cache, s.table_d, s.lens_d, w, 2 ** 32 + 5, 1, s.table_d, 128)

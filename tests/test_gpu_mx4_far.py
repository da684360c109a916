"""Sequences of the most tokens that there may be, 2^31 - 4096: the cache is a page of 256 tokens
that the table repeats, the weights are as wide. Positions next to 2^31 have to be those of the
tokens that they name."""
import math

import numpy as np
import pytest
import torch

import mx4_helpers as H
from gcnasm_amd import mx4_cache as mc
from test_gpu_mx4_cache import Setup, host

pytestmark = pytest.mark.gpu

P, MOST = 256, 0x7FFFF000
PAGES = MOST // P


def far(dev, rows, hq, h, D, seed):
    """One page of tokens, a table of it PAGES times and more, a length past the most."""
    s = Setup(dev, [P], [rows], hq, h, D, P, seed=seed)
    table = torch.full((1, PAGES + 40), int(s.table[0, 0]), dtype=torch.int32, device=dev)
    lens = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device=dev)
    return s, table, lens


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,window", [(1, 500), (1, 20000), (3, 300), (60, 777), (200, 1000),
                                         (200, 5)])
def test_windows_at_the_end(dev, rows, window, D):
    print("far", rows, window, D, flush=True)
    s, table, lens = far(dev, rows, 4, 2, D, seed=41)
    out, lse = mc.attention(s.q, s.cache, table, lens, s.starts_d, window=window)
    # the same tokens at the end of a short sequence
    n = -(-(window + rows) // P) * P
    k, v, there = H.tokens(host(s.cache), [int(s.table[0, 0])] * (n // P), P, D, n)
    o, l, w, ot, lt = H.attention(host(s.q.float()).astype(np.float64), k, v, there, n, rows, True,
                                  window, D ** -0.5, 0.0)
    assert (np.abs(host(out.float()) - o) <= ot).all()
    assert (np.abs(host(lse) - l) <= lt).all()
    if rows * 2 > 16:
        return
    got = mc.attention_weights(s.q, s.cache, table, lens, torch.from_numpy(l.astype(np.float32)).to(
        dev), q_starts=s.starts_d, window=window, width=MOST)
    # a term's score in fp32 and its exponential, 2^-14 of each (|score| < 64), and the sum
    tol = w * (2.0 ** -14 + 4 * rows * 2.0 ** -23) + 1e-30
    assert (np.abs(host(got[0, :, MOST - n:]) - w) <= tol).all()
    for i in range(0, MOST - n, 1 << 28):
        assert not got[0, :, i:min(i + (1 << 28), MOST - n)].any()


def test_all_of_them(dev):
    """Every token repeats the page: the page's output, and its lse plus ln PAGES. A lane adds up
    about 2^20 numbers, each sum off by up to 2^-24 of it."""
    s, table, lens = far(dev, 1, 2, 1, 64, seed=42)
    out, lse = mc.attention(s.q, s.cache, table, lens)
    o, l, _, ot, _ = s.expected()[0]
    mass = np.abs(H.tokens(host(s.cache), s.table[0], P, 64, P)[1]).max()
    assert (np.abs(host(out.float()) - o) <= ot + 2.0 ** -3 * mass).all()
    assert np.abs(host(lse) - l - math.log(PAGES)).max() <= 2.0 ** -3

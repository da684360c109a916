"""Prompts over the MXFP4 cache whose probabilities are all rounded alike: many equal scores below,
or above, a running maximum, at distances where bf16 rounds the probability most. What their
roundings have in common must not reach the output: values of one sign, to the oracle's bounds. The
logarithm of the sum is that of the sum that is not rounded."""
import math

import numpy as np
import pytest
import torch

import mx4_helpers as H
from gcnasm_amd import mx4_cache as mc
from test_gpu_mx4_cache import Setup, host

pytestmark = pytest.mark.gpu

# (how many tokens first are of another score, the others' probability beside theirs): 0.5 + a
# little less than half a unit; below a sink; a maximum that lags by 2^7 + about half a unit
FLAT = [(1, 0.50194), (1, 2.0 ** -0.95), (64, 128.502), (1, 0.1263), (64, 1.0039)]


def attend(s, copies, **kw):
    """The rows of the one sequence in `copies` sequences alike: out and lse of the first, which all
    of them have to have, and whether the tokens were split."""
    q = s.q.repeat(copies, 1, 1)
    table, lens = s.table_d.expand(copies, -1), s.lens_d.repeat(copies)
    n = s.q.shape[0]
    starts = torch.arange(copies + 1, dtype=torch.int32, device=q.device) * n
    args = (q, s.cache, table, lens, starts, n, s.lens[0])
    split = mc.attention_workspace_bytes(*args) > 0
    out, lse = mc.attention(*args, **kw)
    assert (out.view((copies,) + s.q.shape) == out[:n]).all()
    assert (lse.view(copies, n, -1) == lse[:n]).all()
    return out[:n], lse[:n], split


def flat(dev, n, rows, hq, h, D, P, first, p):
    s = Setup(dev, [n], [rows], hq, h, D, P, seed=21)
    k = np.zeros((n, h, D), np.float32)
    k[:first, :, 0] = 6.0
    v = np.abs(np.random.default_rng(n).standard_normal((n, h, D))).astype(np.float32) + 0.5
    v[:, 0] = 1.5
    mc.append(s.cache, torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev),
              torch.from_numpy(s.slots).to(dev))
    s.q[:] = 0
    s.q[:, :, 0] = 1.0
    key = H.tokens(host(s.cache), s.table[0], P, D, 1)[0]
    return s, -math.log(p) / float(key[0, 0, 0])


@pytest.mark.parametrize("first,p", FLAT)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,hq,P", [(512, 2, 64), (1501, 4, 32)])
@pytest.mark.parametrize("copies", [1, 256])
def test_equal_scores(dev, n, hq, P, D, first, p, copies):
    print("flat", n, hq, P, D, first, p, copies, flush=True)
    s, scale = flat(dev, n, 100, hq, 2, D, P, first, p)
    out, lse, split = attend(s, copies, scale=scale)
    assert split == (copies == 1)
    s.check(out, lse, s.expected(scale=scale))
    # all values alike: their mean is their value
    assert (out[:, :hq // 2] == 1.5).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("copies", [1, 256])
def test_equal_scores_beside_a_value_past_bf16(dev, D, copies):
    """A token whose values the products leave out (scale byte 253; 1.5 * 2^126 is finite) weighs
    as much as the others do."""
    print("past bf16", D, copies, flush=True)
    P = 64
    s, scale = flat(dev, 512, 100, 2, 2, D, P, 1, 0.50194)
    _, vc, _, vs = H.places(P, D)
    slot = s.slots[300]
    cache = host(s.cache).copy()
    cache[slot // P][:, vs[slot % P]] = 253
    cache[slot // P][:, vc[slot % P]] = 0x33
    s.cache.copy_(torch.from_numpy(cache).to(dev))
    out, lse, _ = attend(s, copies, scale=scale)
    parts = s.expected(scale=scale)
    assert np.isfinite(parts[0][0]).all() and parts[0][0].min() > 1e35
    s.check(out, lse, parts)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_nan_stays_with_the_rows_that_see_it(dev, D):
    """Rows of one wave, some of which see a NaN key: the others' results are theirs."""
    print("nan", D, flush=True)
    P, at = 64, 310
    s = Setup(dev, [352], [96], 2, 2, D, P, seed=24)
    clean = s.expected()
    _, _, ks, _ = H.places(P, D)
    slot = s.slots[at]
    cache = host(s.cache).copy()
    cache[slot // P][:, ks[slot % P]] = 255
    s.cache.copy_(torch.from_numpy(cache).to(dev))
    for copies in (1, 256):
        q = s.q.repeat(copies, 1, 1)
        starts = torch.arange(copies + 1, dtype=torch.int32, device=dev) * 96
        out, lse = mc.attention(q, s.cache, s.table_d.expand(copies, -1), s.lens_d.repeat(copies),
                                starts, 96, 352)
        first = at - (352 - 96)  # the first row that sees it
        for c in (0, copies - 1):
            o, l = host(out.float())[c * 96:(c + 1) * 96], host(lse)[c * 96:(c + 1) * 96]
            assert np.isnan(o[first:]).all() and np.isnan(l[first:]).all()
            assert (np.abs(o - clean[0][0]) <= clean[0][3])[:first].all()
            assert (np.abs(l - clean[0][1]) <= clean[0][4])[:first].all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_error_beside_the_outputs_own_rounding(dev, D):
    """Random scores and values of both signs. The output's own rounding to bf16 is off by up to
    2^-8 of it, evenly spread over a unit. The probabilities' is alike, each independently: their
    sum's is as large again beside sqrt(sum p^2 v^2), which is what a sum of independent values
    comes to. Together sqrt(2) of the output's own, at most 1.6 for the spread of both."""
    s = Setup(dev, [2048], [64], 4, 2, D, 64, seed=23)
    out, _, split = attend(s, 256)
    assert not split
    want = s.expected()[0][0]
    got = host(out.float()).astype(np.float64)
    own = host(torch.from_numpy(want).float().bfloat16().float()).astype(np.float64) - want
    ratio = np.sqrt(((got - want) ** 2).mean() / (own ** 2).mean())
    print("D", D, "error in units of the output's own rounding", ratio, flush=True)
    assert ratio <= 1.6

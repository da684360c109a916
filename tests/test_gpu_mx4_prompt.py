"""Prompts over the MXFP4 cache where the kernel's forms differ: pages of 64 tokens and more and
smaller ones, pages that are not in the cache, values past bf16, windows and chunks that
begin inside a page, many rows and few of the same sequence. Against the oracle in float64, with its
bounds of what the kernels may be off by."""
import numpy as np
import pytest
import torch

import mx4_helpers as H
from gcnasm_amd import mx4_cache as mc
from test_gpu_mx4_cache import Setup, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("P", [32, 64, 128, 256])
def test_pages_outside_the_cache_are_hidden(dev, P, D):
    print("hidden pages", P, D, flush=True)
    s = Setup(dev, [5 * P + 3, 2 * P], [100, 90], 4, 2, D, P, seed=11)
    table = s.table.copy()
    table[0, 1], table[0, 4], table[0, 5], table[1, 0] = -1, 1 << 30, s.cache.shape[0], -(1 << 31)
    out, lse = mc.attention(s.q, s.cache, torch.from_numpy(table).to(dev), s.lens_d, s.starts_d)
    s.check(out, lse, s.expected(table=table))
    # nothing but hidden pages
    table[:] = -5
    out, lse = mc.attention(s.q, s.cache, torch.from_numpy(table).to(dev), s.lens_d, s.starts_d)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("P,window", [(128, 0), (128, 70), (256, 129), (64, 64), (16, 100)])
def test_windows_that_begin_inside_a_page(dev, P, window, D):
    print("window", P, window, D, flush=True)
    s = Setup(dev, [611, 190], [140, 77], 4, 2, D, P, seed=12)
    out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d, window=window)
    s.check(out, lse, s.expected(window=window))


@pytest.mark.parametrize("P", [16, 64, 128])
@pytest.mark.parametrize("length", [65, 127, 128, 129, 191, 192, 193])
def test_lengths_around_the_ends_of_tiles(dev, length, P):
    print("length", length, P, flush=True)
    for D in (64, 128):
        s = Setup(dev, [length], [min(length, 80)], 2, 1, D, P, seed=length)
        s.check(*mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d), s.expected())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("P", [32, 64, 256])
def test_infinite_and_nan_values_reach_who_sees_them(dev, P, D):
    print("infinite", P, D, flush=True)
    n, at = 200, 130
    s = Setup(dev, [n], [n], 4, 2, D, P, seed=13)
    clean = s.expected()
    _, vc, ks, vs = H.places(P, D)
    slot = s.slots[at]
    cache = host(s.cache).copy()
    page = cache[slot // P]
    page[0, vs[slot % P]] = 254  # the first head's values: 6 * 2^127 is past float32
    page[0, vc[slot % P]] = 0xF7  # +6 and -6 in turn
    s.cache.copy_(torch.from_numpy(cache).to(dev))
    out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d)
    assert np.isfinite(host(lse)).all()
    out = host(out.float())
    assert np.isposinf(out[at:, :2, ::2]).all() and np.isneginf(out[at:, :2, 1::2]).all()
    ok = np.abs(out - clean[0][0]) <= clean[0][3]
    assert ok[:at].all() and ok[:, 2:].all()
    page[0, vs[slot % P]] = 255
    s.cache.copy_(torch.from_numpy(cache).to(dev))
    out = host(mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d)[0].float())
    assert np.isnan(out[at:, :2]).all()
    ok = np.abs(out - clean[0][0]) <= clean[0][3]
    assert ok[:at].all() and ok[:, 2:].all()


@pytest.mark.parametrize("D,hq,h", [(64, 8, 2), (128, 8, 2), (256, 4, 2)])
@pytest.mark.parametrize("P", [32, 64])
def test_a_prompt_in_pieces_gives_what_the_whole_gives(dev, D, hq, h, P):
    """Rows one at a time, by eights and all at once are three kernels' paths; each is held to the
    oracle's bounds, so two of them to twice those."""
    print("pieces", D, hq, h, P, flush=True)
    n = 97
    s = Setup(dev, [n], [n], hq, h, D, P, seed=14)
    parts = s.expected()
    whole = mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d)
    s.check(*whole, parts)
    for step in (1, 8):
        outs, lses = [], []
        for r in range(0, n, step):
            m = min(step, n - r)
            starts = None if m == 1 else torch.tensor([0, m], dtype=torch.int32, device=dev)
            o, l = mc.attention(s.q[r:r + m], s.cache, s.table_d,
                                torch.tensor([r + m], dtype=torch.int32, device=dev), starts)
            outs.append(o)
            lses.append(l)
        s.check(torch.cat(outs), torch.cat(lses), parts)


@pytest.mark.parametrize("rows", [33, 100, 300])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights_of_many_rows_over_ragged_sequences(dev, rows, D):
    """Blocks of tokens divide the rows that see them: sequences of many rows beside such with few or
    none, and a window that leaves most rows behind."""
    print("weights", rows, D, flush=True)
    lens, n = [700, 150, 40], [rows, 7, 0]
    s = Setup(dev, lens, n, 4, 2, D, 64, seed=15)
    for window in (0, 50):
        parts = s.expected(window=window)
        lse = np.concatenate([p[1] for p in parts]).astype(np.float32)
        got = host(mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d,
                                        torch.from_numpy(lse).to(dev), q_starts=s.starts_d,
                                        max_q=rows, max_len=700, window=window))
        for b, length in enumerate(lens):
            want = parts[b][2]
            # a term's score in fp32 and its exponential, 2^-14 of each (|score| < 64), and the sum
            tol = want * (2.0 ** -14 + n[b] * 2 * 2.0 ** -23) + 1e-30
            assert (np.abs(got[b, :, :length] - want) <= tol).all()
            assert (got[b, :, length:] == 0).all()


@pytest.mark.parametrize("D,hq,h,length", [(64, 2, 1, 20011), (128, 1, 1, 9001), (256, 2, 1, 17000)])
def test_many_splits_of_one_row(dev, D, hq, h, length):
    print("splits", D, hq, h, length, flush=True)
    s = Setup(dev, [length, 1], [1, 1], hq, h, D, 64, seed=16)
    parts = s.expected()
    for lens, b in ((s.lens_d[:1], 0), (s.lens_d[1:], 1)):  # alone, so that it is cut the most
        s1 = mc.attention(s.q[b:b + 1], s.cache, s.table_d[b:b + 1], lens, max_len=length)
        o, l, _, ot, lt = parts[b]
        assert (np.abs(host(s1[0].float()) - o) <= ot).all()
        assert (np.abs(host(s1[1]) - l) <= lt).all()


@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("window", [1, 6, 128, 700, 5000])
def test_weights_of_few_rows_with_a_window(dev, rows, window):
    print("weights with a window", rows, window, flush=True)
    lens, n = [3001, 640, 130, 5, 0], [rows, rows, 0, rows, rows]
    s = Setup(dev, lens, n, 4, 2, 128, 32, seed=17)
    parts = s.expected(window=window)
    lse = torch.from_numpy(np.concatenate([p[1] for p in parts]).astype(np.float32)).to(dev)
    width = 3020
    before = torch.rand((5, 2, width), device=dev)
    old = host(before).astype(np.float64)
    kw = dict(q_starts=s.starts_d, max_q=rows, max_len=3001, window=window)
    args = (s.q, s.cache, s.table_d, s.lens_d, lse)
    got = mc.attention_weights(*args, before, **kw)
    for b, length in enumerate(lens):
        want = parts[b][2] + old[b, :, :length]
        # as of many rows, and the sum's rounding to fp32
        tol = parts[b][2] * (2.0 ** -14 + 2 * rows * 2.0 ** -23) + want * 2.0 ** -22 + 1e-30
        assert (np.abs(host(got)[b, :, :length] - want) <= tol).all()
        assert (host(got)[b, :, length:] == 0).all()
    base = mc.attention_weights(*args, None, width=width, **kw)
    for b, length in enumerate(lens):
        want = parts[b][2]
        tol = want * (2.0 ** -14 + 2 * rows * 2.0 ** -23) + 1e-30
        assert (np.abs(host(base)[b, :, :length] - want) <= tol).all()
    place = before.clone()
    assert mc.attention_weights(*args, place, out=place, **kw) is place
    assert torch.equal(place, got)

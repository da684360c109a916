"""The MXFP4 key/value cache on the GPU against its definition in numpy and
float64 (mx4_helpers): bytes and whole numbers equal, computed numbers within
bounds that follow from the widths the kernels compute in."""
import itertools

import numpy as np
import pytest
import torch

import mx4_helpers as H
import oracle
from gcnasm_amd import GaError, _lib, mx4_cache as mc

pytestmark = pytest.mark.gpu


def bf16(x):
    """float64 array rounded to bf16 (through fp32; exactly representable inputs here)."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16)


def host(x):
    return x.detach().cpu().numpy()


class Setup:
    """A cache whose pages lie in no order, filled by append(); what no token uses is 0xFF (codes
    -6, scales NaN)."""

    def __init__(self, dev, lens, rows, hq, h, D, P=16, seed=0, spare=3, extra_pages=2):
        rng = np.random.default_rng(seed)
        self.lens, self.rows, self.D, self.P, self.h, self.hq = lens, rows, D, P, h, hq
        n = len(lens)
        per = max(1, max(-(-x // P) for x in lens) + extra_pages)
        total = n * per + spare
        order = rng.permutation(total)[:n * per].reshape(n, per).astype(np.int32)
        self.table = order.copy()
        self.cache = mc.new_cache(total, h, D, P, dev)
        self.cache.fill_(0xFF)
        slots, ks, vs = [], [], []
        for b, length in enumerate(lens):
            t = np.arange(length)
            slots.append(order[b][t // P].astype(np.int64) * P + t % P)
            self.table[b, -(-length // P):] = -1  # never looked at
            ks.append(rng.standard_normal((length, h, D)) * np.exp(rng.standard_normal(D) / 2))
            vs.append(rng.standard_normal((length, h, D)))
        self.slots = np.concatenate(slots) if slots else np.zeros(0, np.int64)
        self.k = np.concatenate(ks).astype(np.float32)
        self.v = np.concatenate(vs).astype(np.float32)
        if len(self.slots):
            mc.append(self.cache, torch.from_numpy(self.k).to(dev), torch.from_numpy(self.v).to(dev),
                      torch.from_numpy(self.slots).to(dev))
        self.q = bf16(rng.standard_normal((sum(rows), hq, D))).to(dev)
        self.table_d = torch.from_numpy(self.table).to(dev)
        self.lens_d = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.starts_d = torch.from_numpy(self.starts).to(dev)

    def expected(self, causal=True, window=0, scale=None, softcap=0.0, table=None, cache=None):
        cache = host(self.cache) if cache is None else cache
        table = self.table if table is None else table
        q = host(self.q.float()).astype(np.float64)
        scale = self.D ** -0.5 if scale is None else scale
        parts = []
        for b, (length, n) in enumerate(zip(self.lens, self.rows)):
            k, v, there = H.tokens(cache, table[b], self.P, self.D, length)
            parts.append(H.attention(q[self.starts[b]:self.starts[b + 1]], k, v, there, length, n,
                                     causal, window, scale, softcap))
        return parts

    def check(self, out, lse, parts):
        out, lse = host(out.float()).astype(np.float64), host(lse).astype(np.float64)
        for b, (o, l, _, ot, lt) in enumerate(parts):
            at = slice(self.starts[b], self.starts[b + 1])
            empty = np.isinf(l)
            assert np.array_equal(np.isneginf(lse[at]), empty), "empty rows of sequence %d" % b
            assert (out[at][empty] == 0).all()
            d = np.abs(out[at] - o)
            assert (d <= ot).all(), (b, float((d - ot).max()), float(d.max()))
            d = np.abs(lse[at][~empty] - l[~empty])
            assert (d <= lt[~empty]).all(), (b, float(d.max()))


# ---- append and read ------------------------------------------------------------------


@pytest.mark.parametrize("D,P", [(64, 16), (64, 128), (128, 16), (128, 64), (256, 32), (256, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rule", [0, 1, 2])
def test_append_writes_the_quantisers_bytes(dev, D, P, dtype, rule):
    print("append D=%d P=%d %s rule %d" % (D, P, dtype, rule), flush=True)
    h, pages, n = 3, 5, 37
    rng = np.random.default_rng(D + P + rule)
    x = rng.standard_normal((2, n, h, D)).astype(np.float32) * 3
    x[0, 0] = 0
    x[1, 1, 0, :32] = 1e-40
    x[0, 2, 1, 5] = np.nan
    x[1, 3, 2, 7] = np.inf
    x[1, 3, 2, 9] = -np.inf
    x[0, 4, 0] *= 1e30
    x[0, 5, 0, ::2] = -0.0
    t = torch.from_numpy(x).to(dtype)
    x = host(t.float())
    slots = rng.permutation(pages * P)[:n].astype(np.int64)
    dropped = {1: -1, 7: pages * P, 8: 1 << 40, 9: -(1 << 40)}
    for i, s in dropped.items():
        slots[i] = s
    cache = mc.new_cache(pages, h, D, P, dev)
    cache.fill_(0xA5)
    t = t.to(dev)
    mc.append(cache, t[0], t[1], torch.from_numpy(slots).to(dev), scale_rule=rule)
    want = np.full((pages, h, mc.page_bytes(P, D)), 0xA5, np.uint8)
    places = H.places(P, D)
    for which in range(2):
        q, s = oracle.quant_mxfp4(x[which].reshape(n * h, D), rule)
        q, s = q.reshape(n, h, D // 2), s.reshape(n, h, D // 32)
        for i in range(n):
            if i in dropped:
                continue
            page, at = divmod(int(slots[i]), P)
            want[page][:, places[which][at]] = q[i]
            want[page][:, places[2 + which][at]] = s[i]
    np.testing.assert_array_equal(host(cache), want)
    # and what the slots then stand for
    for kind in (torch.float32, torch.bfloat16):
        k, v = mc.read(cache, torch.from_numpy(slots).to(dev), D, kind)
        for which, got in enumerate((k, v)):
            got = host(got.float())
            for i in range(n):
                if i in dropped:
                    assert (got[i] == 0).all()
                    continue
                page, at = divmod(int(slots[i]), P)
                with np.errstate(over="ignore"):
                    exp = H.values(want[page][:, places[which][at]],
                                   want[page][:, places[2 + which][at]]).astype(np.float32)
                np.testing.assert_array_equal(got[i], exp)


@pytest.mark.parametrize("scale", [0, 1, 2, 126, 127, 252, 253, 254, 255])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_read_every_code_at_extreme_scales(dev, D, scale):
    P = 16
    cache = mc.new_cache(2, 1, D, P, dev)
    page = np.arange(mc.page_bytes(P, D), dtype=np.uint32).astype(np.uint8) * 37
    kc, vc, ks, vs = H.places(P, D)
    page[ks] = page[vs] = scale
    cache[1, 0] = torch.from_numpy(page).to(dev)
    slots = torch.arange(P, 2 * P, device=dev)
    k, v = mc.read(cache, slots, D, torch.float32)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(host(k)[:, 0],
                                      H.values(page[kc], page[ks]).astype(np.float32))
        np.testing.assert_array_equal(host(v)[:, 0],
                                      H.values(page[vc], page[vs]).astype(np.float32))


@pytest.mark.parametrize("dtype,step", [(torch.float32, 4), (torch.bfloat16, 8), (torch.bfloat16, 4)])
def test_append_takes_strided_rows(dev, dtype, step):
    """Heads and rows apart by more than they hold, k and v parts of one tensor; bf16 rows that
    allow only 8-byte loads."""
    h, D, P, n = 2, 128, 32, 21
    big = torch.randn((n, 2 * h * (D + step) + step), device=dev).to(dtype)
    parts = big[:, step:].unflatten(1, (2, h, D + step))[..., :D]
    k, v = parts[:, 0], parts[:, 1]
    slots = torch.arange(n, device=dev) + 5
    a, b = mc.new_cache(2, h, D, P, dev), mc.new_cache(2, h, D, P, dev)
    mc.append(a, k, v, slots)
    mc.append(b, k.contiguous(), v.contiguous(), slots)
    assert torch.equal(a, b) and a.any()
    empty = torch.empty((0, h, D), device=dev, dtype=dtype)
    mc.append(a, empty, empty, slots[:0])
    assert torch.equal(a, b)
    assert mc.read(a, slots[:0], D)[0].shape == (0, h, D)


# ---- attention ----------------------------------------------------------------------------


SHAPES = [
    # lens, rows, heads, kv heads, D, P
    ([1], [1], 1, 1, 128, 16),
    ([513], [1], 32, 8, 128, 64),
    ([0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129], [1] * 14, 8, 2, 128, 16),
    ([700, 3, 0, 129], [1, 1, 1, 1], 6, 2, 64, 32),
    ([700, 3, 0, 129], [1, 1, 1, 1], 10, 2, 256, 256),
    ([300, 77], [1, 1], 40, 1, 128, 128),          # 40 rows of one kv head: 3 blocks of 16
    ([64, 200, 5, 90], [64, 33, 5, 0], 8, 4, 128, 16),
    ([131, 260], [131, 17], 8, 1, 64, 64),
    ([100, 40], [70, 40], 4, 4, 256, 32),
    ([3, 7], [9, 7], 4, 2, 128, 16),               # more rows than tokens: the first see none
    ([420, 333], [300, 333], 6, 2, 128, 64),
]


@pytest.mark.parametrize("lens,rows,hq,h,D,P", SHAPES)
@pytest.mark.parametrize("window,softcap,causal", [(0, 0.0, True), (40, 0.0, True), (1, 20.0, True),
                                                   (0, 5.0, False)])
def test_attention(dev, lens, rows, hq, h, D, P, window, softcap, causal):
    print("attention", lens, rows, hq, h, D, P, window, softcap, causal, flush=True)
    s = Setup(dev, lens, rows, hq, h, D, P, seed=len(lens) * 100 + D)
    starts = None if all(r == 1 for r in rows) else s.starts_d
    kw = dict(causal=causal, window=window, softcap=softcap)
    parts = s.expected(**kw)
    out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d, starts, max(rows), max(lens), **kw)
    s.check(out, lse, parts)
    # the same bits again, and without the host's bounds the same rows
    again = mc.attention(s.q, s.cache, s.table_d, s.lens_d, starts, max(rows), max(lens), **kw)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    s.check(*mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d, **kw), parts)


@pytest.mark.parametrize("lens,rows,hq,h,D,P", [SHAPES[1], SHAPES[6], SHAPES[10]])
def test_attention_bounds_that_are_too_small(dev, lens, rows, hq, h, D, P):
    """max_q and max_len choose the launch only."""
    s = Setup(dev, lens, rows, hq, h, D, P, seed=3)
    out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d, 1, 1)
    s.check(out, lse, s.expected())


@pytest.mark.parametrize("scale", [0.0, 3.0, -0.5])
def test_attention_scales(dev, scale):
    s = Setup(dev, [150, 40], [5, 40], 4, 2, 128, 16, seed=4)
    s.check(*mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d, scale=scale),
            s.expected(scale=scale))


def test_attention_strides_and_given_results(dev):
    s = Setup(dev, [90, 33, 257], [7, 33, 1], 6, 3, 128, 32, seed=5)
    n = s.q.shape[0]
    wide = torch.zeros((n, 8, 160), dtype=torch.bfloat16, device=dev)
    wide[:, 1:7, 8:136] = s.q
    q = wide[:, 1:7, 8:136]
    out = torch.full((6, n, 136), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((n, 9), 7.0, device=dev)
    view = out[:, :, :128].transpose(0, 1)
    pool = torch.zeros((s.cache.shape[0], 2) + tuple(s.cache.shape[1:]), dtype=torch.uint8,
                       device=dev)
    pool[:, 1] = s.cache  # one layer of a pool that interleaves two
    table = torch.full((3, s.table.shape[1] + 5), -7, dtype=torch.int32, device=dev)
    table[:, :-5] = s.table_d
    need = mc.attention_workspace_bytes(q, pool[:, 1], table[:, :-5], s.lens_d, s.starts_d)
    ws = torch.empty(need + 64, dtype=torch.uint8, device=dev)
    got = mc.attention(q, pool[:, 1], table[:, :-5], s.lens_d, s.starts_d, out=view, lse=lse[:, :6],
                       workspace=ws)
    assert got[0].data_ptr() == out.data_ptr()
    s.check(view, lse[:, :6], s.expected())
    assert (out[:, :, 128:] == 7).all() and (lse[:, 6:] == 7).all()
    if need:
        with pytest.raises(GaError) as e:
            mc.attention(q, pool[:, 1], table[:, :-5], s.lens_d, s.starts_d, workspace=ws[:need - 16])
        assert e.value.status == _lib.GA_ERR_WORKSPACE


@pytest.mark.parametrize("rows", [[1, 1], [30, 120]])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_pages_outside_the_cache_are_hidden(dev, rows, D):
    s = Setup(dev, [150, 130], rows, 4, 2, D, 16, seed=6)
    table = s.table.copy()
    table[0, 3], table[0, 8], table[1, 0], table[1, 5] = -1, 1 << 30, -(1 << 31), s.cache.shape[0]
    got = mc.attention(s.q, s.cache, torch.from_numpy(table).to(dev), s.lens_d, s.starts_d)
    s.check(*got, s.expected(table=table))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hq", [2, 6])
def test_what_a_row_does_not_see_does_not_reach_it(dev, D, hq):
    """Infinite and NaN keys and values of later tokens: rows before them have finite results, those
    that see an infinite value have it."""
    P, n = 16, 120
    s = Setup(dev, [n], [n], hq, 2, D, P, seed=7)
    clean = s.expected()
    kc, vc, ks, vs = H.places(P, D)
    at = 75
    slot = s.slots[at]
    cache = host(s.cache).copy()
    page = cache[slot // P]
    page[:, vs[slot % P]] = 254              # values of up to 6 * 2^127
    page[:, vc[slot % P]] = 0x77             # all +6
    s.cache.copy_(torch.from_numpy(cache).to(dev))
    out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d)
    out = host(out.float())
    assert np.isposinf(out[at:]).all()
    assert (np.abs(out[:at] - clean[0][0][:at]) <= clean[0][3][:at]).all()
    assert np.isfinite(host(lse)).all()
    page[:, vs[slot % P]] = 255              # NaN
    page[:, ks[slot % P]] = 255
    s.cache.copy_(torch.from_numpy(cache).to(dev))
    out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d, s.starts_d)
    out, lse = host(out.float()), host(lse)
    assert np.isnan(out[at:]).all() and np.isnan(lse[at:]).all()
    assert (np.abs(out[:at] - clean[0][0][:at]) <= clean[0][3][:at]).all()
    w = host(mc.attention_weights(s.q[:at], s.cache, s.table_d, s.lens_d, torch.from_numpy(
        lse[:at].copy()).to(dev), q_starts=torch.tensor([0, 0], dtype=torch.int32, device=dev)))
    assert (w == 0).all()  # no rows: nothing is given
    # one row at the end of a window that leaves the token behind
    got = mc.attention(s.q[-1:], s.cache, s.table_d, s.lens_d, window=n - 1 - at)
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()


def test_attention_of_equal_scores_is_the_mean(dev):
    """Scale 0: every visible token alike, at lengths over several splits."""
    for n in (1, 129, 5000):
        s = Setup(dev, [n], [1], 8, 2, 128, 64, seed=n)
        out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d, scale=0.0)
        _, v, _ = H.tokens(host(s.cache), s.table[0], 64, 128, n)
        mean = v.mean(0).repeat(4, 0)
        tol = (2.0 ** -9 + n * 2.0 ** -23) * np.abs(v).mean(0).repeat(4, 0) + 2.0 ** -8.9 * np.abs(mean)
        assert (np.abs(host(out.float())[0] - mean) <= tol).all()
        assert np.abs(host(lse)[0] - np.log(n)).max() <= 2.0 ** -20 * (1 + np.log(n))


def test_scores_that_rise_along_the_tokens(dev):
    """A maximum that moves on at every tile, by little and by much."""
    D, P, n, h = 128, 16, 700, 1
    for step in (0.05, 0.3, 6.0):
        s = Setup(dev, [n], [1], 4, h, D, P, seed=8)
        k = np.zeros((n, h, D), np.float32)
        k[:, 0, 0] = 1.0
        k[:, 0, 32] = np.arange(n) % 7  # exact codes 0 .. 6 without 5
        k[:, 0, 64] = 2.0 ** np.floor(np.arange(n) / 100)
        mc.append(s.cache, torch.from_numpy(k).to(dev), torch.from_numpy(s.v).to(dev),
                  torch.from_numpy(s.slots).to(dev))
        s.q[:] = 0
        s.q[:, :, 0], s.q[:, :, 32], s.q[:, :, 64] = 1.0, 0.5, step
        s.check(*mc.attention(s.q, s.cache, s.table_d, s.lens_d, scale=1.0), s.expected(scale=1.0))


def test_no_sequences_and_no_rows(dev):
    s = Setup(dev, [20, 30], [1, 1], 4, 2, 128, 16)
    none = torch.empty((0, 4, 128), dtype=torch.bfloat16, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    out, lse = mc.attention(none, s.cache, torch.empty((0, 3), **i32), torch.empty((0,), **i32))
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    out, _ = mc.attention(none, s.cache, s.table_d, s.lens_d, torch.zeros(3, **i32))
    assert out.shape == (0, 4, 128)
    # a table without pages: every sequence is empty, whatever its length says
    out, lse = mc.attention(s.q, s.cache, torch.empty((2, 0), **i32), s.lens_d)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_a_cache_past_four_gib(dev):
    """Pages whose byte offsets pass 32 bits, read by every kernel."""
    h, D, P = 8, 128, 256
    size = mc.page_bytes(P, D) * h
    total = (9 << 30) // 2 // size + 8
    cache = mc.new_cache(total, h, D, P, dev)
    rng = np.random.default_rng(11)
    n = 300
    k = rng.standard_normal((n, h, D)).astype(np.float32)
    v = rng.standard_normal((n, h, D)).astype(np.float32)
    small = mc.new_cache(4, h, D, P, dev)
    far = [total - 1, total - 5]
    near = [2, 0]
    q = bf16(rng.standard_normal((40, 16, D))).to(dev)
    results = []
    for c, pages in ((cache, far), (small, near)):
        t = np.arange(n)
        slots = torch.from_numpy(np.array(pages)[t // P].astype(np.int64) * P + t % P).to(dev)
        mc.append(c, torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), slots)
        table = torch.tensor([pages], dtype=torch.int32, device=dev)
        dst = torch.tensor([[pages[0] - 1, pages[1] + 3 if pages is near else pages[1] - 1]],
                           dtype=torch.int32, device=dev)
        lens = torch.tensor([n], dtype=torch.int32, device=dev)
        starts = torch.tensor([0, 40], dtype=torch.int32, device=dev)
        out, lse = mc.attention(q, c, table, lens, starts)
        w = mc.attention_weights(q, c, table, lens, lse, q_starts=starts)
        kept, nl, nw = mc.evict(c, table, lens, w, 270, 20, dst, D)
        j = torch.arange(270, device=dev)
        dslots = dst[0].long()[j // P] * P + j % P
        results.append((out, lse, w, kept, nl, nw) + mc.read(c, slots, D) + mc.read(c, dslots, D) +
                       mc.attention(q[:1], c, dst, nl))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    del cache


# ---- weights ----------------------------------------------------------------------------------


@pytest.mark.parametrize("lens,rows,hq,h,D,P", SHAPES)
@pytest.mark.parametrize("window,softcap,causal", [(0, 0.0, True), (40, 20.0, True), (0, 0.0, False)])
def test_attention_weights(dev, lens, rows, hq, h, D, P, window, softcap, causal):
    print("weights", lens, rows, hq, h, D, P, window, softcap, causal, flush=True)
    s = Setup(dev, lens, rows, hq, h, D, P, seed=len(lens) * 10 + D)
    starts = None if all(r == 1 for r in rows) else s.starts_d
    kw = dict(causal=causal, window=window, softcap=softcap)
    parts = s.expected(**kw)
    # the kernel's input is an lse in fp32: the definition's, rounded
    lse = np.concatenate([p[1] for p in parts]).astype(np.float32)
    lse_d = torch.from_numpy(lse).to(dev)
    width = max(lens) + 9
    before = torch.rand((len(lens), h, width + 3), device=dev)[:, :, :width]
    out = mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d, lse_d, before, starts, max(rows),
                               max(lens), **kw)
    got, old = host(out).astype(np.float64), host(before).astype(np.float64)
    for b, (_, l, w, _, lt) in enumerate(parts):
        # each probability as far off as its score and lse are, the sum in fp32
        err = (2 * lt.max(initial=0) + 2.0 ** -20) if lt.size else 0.0
        want = old[b, :, :lens[b]] + w
        tol = w * err + 2.0 ** -22 * (want + 1) * (1 + rows[b] * hq * 2.0 ** -6)
        d = np.abs(got[b, :, :lens[b]] - want)
        assert (d <= tol).all(), (b, float((d - tol).max()))
        assert (got[b, :, lens[b]:] == 0).all()
    # in place, and from nothing
    base = mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d, lse_d, None, starts, width=width,
                                **kw)
    inplace = torch.zeros((len(lens), h, width), device=dev)
    assert mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d, lse_d, inplace, starts,
                                out=inplace, **kw) is inplace
    assert torch.equal(base, inplace)
    # fewer tokens than there are
    few = mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d, lse_d, None, starts, width=5, **kw)
    assert torch.equal(few, base[:, :, :5])


@pytest.mark.parametrize("D", [64, 128])
def test_weights_of_garbage_behind_the_length(dev, D):
    """NaN scales in the last tile's unused tokens and in a hidden page give nothing."""
    s = Setup(dev, [49, 17], [3, 17], 4, 2, D, 16, seed=12)
    table = s.table.copy()
    table[0, 1] = -5
    parts = s.expected(table=table)
    lse = torch.from_numpy(np.concatenate([p[1] for p in parts]).astype(np.float32)).to(dev)
    w = host(mc.attention_weights(s.q, s.cache, torch.from_numpy(table).to(dev), s.lens_d, lse,
                                  q_starts=s.starts_d, width=64))
    assert np.isfinite(w).all()
    for b, p in enumerate(parts):
        assert np.abs(w[b, :, :s.lens[b]] - p[2]).max() <= 1e-3
    assert (w[0, :, 16:32] == 0).all()


# ---- eviction ------------------------------------------------------------------------------------


def evict_case(dev, s, weights, keep, recent, new_width=None):
    n, h, D, P = len(s.lens), s.h, s.D, s.P
    used = set(s.table.ravel().tolist())
    need = -(-keep // P)
    size = s.cache.shape[0]
    pool = torch.cat([s.cache, torch.full((n * need,) + tuple(s.cache.shape[1:]), 0x5A,
                                          dtype=torch.uint8, device=dev)])
    dst = np.random.default_rng(1).permutation(n * need).reshape(n, need).astype(np.int32) + size
    assert not used & set(dst.ravel().tolist())
    before = host(pool).copy()
    w = torch.from_numpy(weights).to(dev)
    new = None if new_width is None else torch.full((n, h, new_width), 9.0, device=dev)
    kept, lens, nw = mc.evict(pool, s.table_d, s.lens_d, w, keep, recent,
                              torch.from_numpy(dst).to(dev), D, new_weights=new)
    kept, lens, nw, after = host(kept), host(lens), host(nw), host(pool)
    places = H.places(P, D)
    np.testing.assert_array_equal(after[:size], before[:size])
    for b in range(n):
        assert lens[b] == min(s.lens[b], keep)
        for head in range(h):
            want = H.evict(weights[b, head], s.lens[b], keep, recent)
            m = len(want)
            assert m == lens[b]
            np.testing.assert_array_equal(kept[b, head, :m], want)
            assert (kept[b, head, m:] == -1).all()
            np.testing.assert_array_equal(nw[b, head, :m], weights[b, head][want])
            assert (nw[b, head, m:] == 0).all()
            j = np.arange(m)
            for p in places:
                src = before[s.table[b][want // P], head][j[:, None], p[want % P]]
                got = after[dst[b][j // P], head][j[:, None], p[j % P]]
                np.testing.assert_array_equal(got, src)
    return kept


@pytest.mark.parametrize("D,P", [(64, 16), (128, 32), (256, 64), (128, 256)])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (65, 64), (100, 10), (130, 0), (400, 17)])
def test_evict(dev, D, P, keep, recent):
    print("evict", D, P, keep, recent, flush=True)
    s = Setup(dev, [333, 100, 0, 101, 130], [1] * 5, 4, 2, D, P, seed=keep)
    rng = np.random.default_rng(keep + recent)
    w = np.exp(3 * rng.standard_normal((5, 2, 340))).astype(np.float32)
    evict_case(dev, s, w, keep, recent)
    evict_case(dev, s, w, keep, recent, new_width=keep + 11)


@pytest.mark.parametrize("what", ["equal", "few values", "zeros of both signs", "nan", "huge",
                                  "subnormal", "negative"])
def test_evict_orders(dev, what):
    """Ties go to the lowest index; NaN counts as largest; both zeros alike."""
    lens = [2500, 1027]
    s = Setup(dev, lens, [1, 1], 2, 2, 64, 64, seed=13)
    rng = np.random.default_rng(14)
    w = rng.standard_normal((2, 2, 2500)).astype(np.float32)
    if what == "equal":
        w[:] = 0.25
    elif what == "few values":
        w = rng.integers(0, 3, w.shape).astype(np.float32)
    elif what == "zeros of both signs":
        w = np.where(rng.random(w.shape) < 0.5, np.float32(0.0), np.float32(-0.0))
    elif what == "nan":
        w[rng.random(w.shape) < 0.01] = np.nan
    elif what == "huge":
        w[rng.random(w.shape) < 0.1] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
    elif what == "subnormal":
        w = (w * 1e-40).astype(np.float32)
    else:
        w = -np.abs(w)
    evict_case(dev, s, w, 1000, 30)
    if what != "nan":
        evict_case(dev, s, w, 41, 0)


def test_evict_what_attention_then_sees(dev):
    """The kept tokens, attended to at their new places, as those tokens alone."""
    s = Setup(dev, [400], [1], 4, 2, 128, 32, seed=15)
    w = np.random.default_rng(16).random((1, 2, 400)).astype(np.float32)
    dst = torch.arange(s.cache.shape[0], s.cache.shape[0] + 4, dtype=torch.int32, device=dev)[None]
    pool = torch.cat([s.cache, torch.full((4,) + tuple(s.cache.shape[1:]), 0xFF, dtype=torch.uint8,
                                          device=dev)])
    kept, lens, _ = mc.evict(pool, s.table_d, s.lens_d, torch.from_numpy(w).to(dev), 100, 10, dst, 128)
    out, lse = mc.attention(s.q, pool, dst, lens)
    k, v, there = H.tokens(host(s.cache), s.table[0], 32, 128, 400)
    q = host(s.q.float()).astype(np.float64)
    for head in range(2):
        at = host(kept)[0, head]
        o, l, _, ot, lt = H.attention(q[:, 2 * head:2 * head + 2], k[at][:, head:head + 1],
                                      v[at][:, head:head + 1], there[at], 100, 1, True, 0,
                                      128 ** -0.5, 0.0)
        assert (np.abs(host(out.float())[:, 2 * head:2 * head + 2] - o) <= ot).all()
        assert (np.abs(host(lse)[:, 2 * head:2 * head + 2] - l) <= lt).all()


# ---- streams and graphs -----------------------------------------------------------------------------


@pytest.mark.parametrize("raw", [False, True])
def test_a_stream_of_ones_own(dev, raw):
    """Inputs made on a side stream and the calls given that stream, as an object or a handle, while
    the current one is another."""
    s = Setup(dev, [600, 90], [1, 1], 8, 2, 128, 64, seed=17)
    w = torch.rand((2, 2, 600), device=dev)
    dst = torch.arange(s.cache.shape[0] - 1, s.cache.shape[0] - 3, -1, dtype=torch.int32,
                       device=dev)[:, None]
    pool = torch.cat([s.cache] * 2)
    dst += len(s.cache)
    slots_here = torch.from_numpy(s.slots[:50]).to(dev)

    def passes(q, stream):
        out, lse = mc.attention(q, pool, s.table_d, s.lens_d, stream=stream)
        nw = mc.attention_weights(q, pool, s.table_d, s.lens_d, lse, w, stream=stream)
        kept, lens, w2 = mc.evict(pool, s.table_d, s.lens_d, nw, 50, 5, dst, 128, stream=stream)
        slots = slots_here if stream is None else slots_side
        return [out, lse, nw, kept, lens, w2] + list(mc.read(pool, slots, 128, stream=stream))

    want = passes(s.q, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        slots_side = slots_here * 1
        busy = torch.randn((2048, 2048), device=dev)
        for _ in range(20):
            busy = busy @ busy * 1e-3
        q = s.q * 1  # behind the products on the side stream
    got = passes(q, side.cuda_stream if raw else side)
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_a_captured_step_replays(dev):
    """Append, attention and weights captured once; replays follow the inputs and equal eager
    calls, with eager work between."""
    s = Setup(dev, [1200, 77, 300], [1, 1, 1], 8, 2, 128, 64, seed=18)
    k = torch.randn((3, 2, 128), device=dev)
    v = torch.randn((3, 2, 128), device=dev)
    slots = torch.tensor([int(s.table[b, (n - 1) // 64]) * 64 + (n - 1) % 64
                          for b, n in enumerate(s.lens)], device=dev)
    weights = torch.zeros((3, 2, 1200), device=dev)

    def step():
        mc.append(s.cache, k, v, slots)
        out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d, max_len=1200)
        return out, lse, mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d, lse, weights)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        k.normal_()
        v.normal_()
        s.q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        want = step()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ---- refusals ---------------------------------------------------------------------------------------


def test_refusals(dev):
    s = Setup(dev, [20, 30], [1, 1], 4, 2, 128, 16)
    q, c, t, n = s.q, s.cache, s.table_d, s.lens_d
    k = torch.zeros((3, 2, 128), device=dev)
    slots = torch.arange(3, device=dev)
    w = torch.zeros((2, 2, 30), device=dev)
    lse = torch.zeros((2, 4), device=dev)
    bad = [
        lambda: mc.new_cache(2, 2, 96, 16, dev),
        lambda: mc.new_cache(2, 2, 128, 24, dev),
        lambda: mc.append(c, k, k[:2], slots),
        lambda: mc.append(c, k.half(), k.half(), slots),
        lambda: mc.append(c, k[:, :1], k[:, :1], slots),
        lambda: mc.append(c, k, k, slots.int()),
        lambda: mc.append(c, k, k, slots[:2]),
        lambda: mc.append(c, k.cpu(), k, slots),
        lambda: mc.append(c.float(), k, k, slots),
        lambda: mc.append(c, k, k, slots, scale_rule=3),
        lambda: mc.append(c, torch.zeros((3, 2, 129), device=dev)[..., 1:], k, slots),
        lambda: mc.append(c.transpose(0, 1), k, k, slots),
        lambda: mc.read(c, slots, 96),
        lambda: mc.read(c, slots, 128, torch.float16),
        lambda: mc.attention(q.float(), c, t, n),
        lambda: mc.attention(q[:, :3], c, t, n),
        lambda: mc.attention(q, c, t.long(), n),
        lambda: mc.attention(q, c, t[:1], n),
        lambda: mc.attention(q, c, t, n.long()),
        lambda: mc.attention(q[:1], c, t, n),
        lambda: mc.attention(q, c, t, n, torch.zeros(2, dtype=torch.int32, device=dev)),
        lambda: mc.attention(q, c, t, n, window=-1),
        lambda: mc.attention(q, c, t, n, window=5, causal=False),
        lambda: mc.attention(q, c, t, n, softcap=-1.0),
        lambda: mc.attention(q, c, t, n, softcap=float("nan")),
        lambda: mc.attention(q, c, t, n, out=torch.zeros_like(q).float()),
        lambda: mc.attention(q, c, t, n, lse=lse[:1]),
        lambda: mc.attention(torch.zeros((2, 4, 132), dtype=torch.bfloat16, device=dev)[..., 4:], c,
                             t, n),
        lambda: mc.attention(q.transpose(0, 2).contiguous().transpose(0, 2), c, t, n),
        lambda: mc.attention_weights(q, c, t, n, lse[:, :3]),
        lambda: mc.attention_weights(q, c, t, n, lse, w[:, :1]),
        lambda: mc.attention_weights(q, c, t, n, lse, w, width=31),
        lambda: mc.attention_weights(q, c, t, n, lse, w.double()),
        lambda: mc.evict(c, t, n, w, 0, 0, t, 128),
        lambda: mc.evict(c, t, n, w, 8, 9, t, 128),
        lambda: mc.evict(c, t, n, w, 17, 1, t[:, :1], 128),
        lambda: mc.evict(c, t, n, w, 8, 1, t, 128, new_weights=torch.zeros((2, 2, 7), device=dev)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((GaError, ValueError, TypeError)):
            f()
            print("not refused: item", i, flush=True)
    torch.cuda.synchronize()

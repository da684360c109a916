"""Layers of experts on the GPU against their definitions in numpy and float64
(experts_helpers): whole numbers equal, computed numbers within bounds that follow from the widths
the kernels compute in; the products against the oracle's model of the matrix instruction."""
import itertools

import numpy as np
import pytest
import torch

import experts_helpers as H
import oracle
from gcnasm_amd import GaError, _lib, experts as ex, ops
from helpers import assert_parity, bf16_compare

pytestmark = pytest.mark.gpu


def host(x):
    return x.detach().cpu().numpy()


def on(x, dev):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dev)


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x, np.float32))).to(torch.bfloat16)


# ---- route -----------------------------------------------------------------------------

def check_route(dev, logits, top, dtype, bias=None, **kw):
    x = torch.from_numpy(np.asarray(logits, np.float32)).to(dtype)
    b = None if bias is None else np.asarray(bias, np.float32)
    names = dict(kw)
    want, w = H.route(host(x.float()), top, b, names.pop("scores", "softmax"),
                      most=torch.finfo(dtype).max, **names)
    ids, weights = ex.route(x.to(dev), top, None if b is None else on(b, dev), **kw)
    assert ids.dtype == torch.int32 and weights.dtype == torch.float32
    assert np.array_equal(host(ids), want)
    # in fp32: an exponential off by 2^-22 and its argument by 2^-24 of itself, the sum by what its
    # terms are (2^-24 of the chosen logits' spread) and a rounding a step, the quotient
    z = np.take_along_axis(host(x.double()), np.maximum(want, 0), 1)
    z = np.where((want >= 0) & np.isfinite(z), z, 0)
    tol = (np.minimum(z.max(1) - z.min(1), 200) + 32)[:, None] * 2.0 ** -24
    if not kw.get("renormalise", True):
        # a softmax's sum over all: up to 16 terms of a lane and 6 steps between them, the terms off
        # by 2^-22.6 of their arguments, 7 of which are e of 1024
        tol = 2.0 ** -18
    assert (np.abs(host(weights) - w) <= tol * np.abs(w) + 2.0 ** -126).all()


@pytest.mark.parametrize("experts,top,groups,top_groups", [
    (1, 1, 1, 1), (7, 7, 1, 1), (7, 2, 7, 2), (60, 4, 1, 1), (60, 4, 3, 2), (64, 6, 1, 1),
    (65, 8, 5, 3), (128, 8, 64, 5), (192, 6, 8, 3), (256, 1, 2, 1), (320, 10, 1, 1),
    (1000, 13, 10, 4), (1024, 64, 16, 1), (1024, 5, 64, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route(dev, experts, top, groups, top_groups, dtype):
    rng = np.random.default_rng(experts * 7 + top)
    for i, (scores, rank, bias, renorm) in enumerate(itertools.product(
            ("softmax", "sigmoid"), (1, 2), (False, True), (True, False))):
        tokens = (1, 5, 33)[i % 3]
        check_route(dev, 2 * rng.standard_normal((tokens, experts)), top, dtype,
                    0.3 * rng.standard_normal(experts) if bias else None, scores=scores,
                    groups=groups, top_groups=top_groups, group_rank=rank, renormalise=renorm,
                    scale=(1.0, 2.5)[i % 2])


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_route_of_equal_and_missing_experts(dev, scores, bias):
    rng = np.random.default_rng(3)
    inf, nan = np.inf, np.nan
    for E, top, groups, kept, rank in ((12, 5, 4, 2, 2), (200, 9, 1, 1, 1), (96, 8, 6, 3, 1)):
        x = rng.integers(-2, 3, (40, E)).astype(np.float32)  # equal ones among them, both zeros
        x[x == 0] *= rng.choice([-1, 1], (x == 0).sum())
        x[1] = -inf
        x[2] = nan
        x[3, 1:] = -inf
        x[4, ::2] = nan
        x[5, 3] = inf
        x[6, :E // 2] = inf
        x[7] = 3e38
        x[8, :] = -3e38
        x[9] = -200.0  # scores that vanish in 32 bits
        x[10] = -800.0  # and in 64
        x[11, :-2] = -inf
        b = rng.integers(-1, 2, E).astype(np.float32)
        b[:3] = (-inf, nan, inf)
        for renorm in (True, False):
            check_route(dev, x, top, torch.float32, b if bias else None, scores=scores,
                        groups=groups, top_groups=kept, group_rank=rank, renormalise=renorm)


@pytest.mark.parametrize("experts,groups", [(48, 1), (250, 5), (256, 16), (600, 20), (1024, 1)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_by_keys_that_32_bits_do_not_tell_apart(dev, experts, groups, scores):
    """Biases that leave of the scores what their rounding to fp32 does: keys of 2^-25 of them, in an
    order that only 64 bits have. (Two keys of 64 bits are that near each other with a chance of
    2^-20 here.)"""
    rng = np.random.default_rng(experts)
    x = np.tile(rng.standard_normal(experts).astype(np.float32), (7, 1))
    bias = -H.scores(x[:1], scores, np.inf)[2][0].astype(np.float32)
    for rank in (1, 2):
        check_route(dev, x, 5, torch.float32, bias, scores=scores, groups=groups,
                    top_groups=max(1, groups // 2), group_rank=rank)
    # far from zero, where fp32 has steps of 2^-10, 1024 and more
    for far in (2.0 ** 13, -2.0 ** 33, 1e30):
        check_route(dev, rng.standard_normal((9, experts)), 4, torch.float32,
                    far + rng.integers(0, 3, experts) * abs(far) * 2.0 ** -23, scores=scores)


def few_scores(scores, most):
    """Logits of several experts that differ while their scores in 64 bits do not, by ranges: `most`
    is 900 or less where their type has too few bits."""
    if scores == "sigmoid":
        return [(35.0, 90.0), (-most, -746.0), (-1e-20, 1e-20)]
    return [(-most, -746.0), (0.0, 1e-20)]  # beside an expert of logit 0 or 1


# experts 512 and up, and more than 16 choices: a token a wave
@pytest.mark.parametrize("experts,groups,kept,top", [
    (12, 3, 1, 2), (12, 4, 2, 3), (64, 8, 3, 6), (60, 10, 7, 9), (256, 16, 5, 16), (192, 8, 3, 20),
    (320, 20, 4, 8), (512, 8, 4, 10), (1024, 64, 9, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_groups_by_their_largest_logit(dev, experts, groups, kept, top, dtype, scores):
    """Without a bias, groups by their largest expert go by its logit, also where 64 bits do not tell the
    scores apart."""
    rng = np.random.default_rng(experts + top)
    size = experts // groups
    for lo, hi in few_scores(scores, 900.0):
        for equal in (False, True):
            x = rng.uniform(lo, hi, (24, experts))
            if equal:  # as many again as another one of their token
                at = rng.integers(0, experts, x.shape)
                x = np.where(rng.random(x.shape) < 0.5, x, np.take_along_axis(x, at, 1))
            if scores == "softmax":
                first = rng.integers(0, groups, 24) * size  # in any group
                x[np.arange(24), first] = 0.0 if lo < 0 else 1.0
            x[:4, rng.random(experts) < 0.3] = -np.inf
            for renormalise in (True, False):
                check_route(dev, x, top, dtype, scores=scores, groups=groups, top_groups=kept,
                            group_rank=1, renormalise=renormalise)


@pytest.mark.parametrize("experts", [12, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_groups_of_saturated_sigmoids(dev, experts, dtype):
    """Three groups, two of them kept, logits whose sigmoid is 1 in 64 bits: far apart, and, of two equal
    ones, near each other."""
    size = experts // 3
    x = np.full((2, experts), -1.0, np.float32)
    x[0, [0, size, 2 * size]] = 40, 41, 60
    x[1, [0, size, size + 1, 2 * size]] = 40, 44, 44, 48
    ids, _ = ex.route(torch.from_numpy(x).to(dtype).to(dev), 3, scores="sigmoid", groups=3,
                      top_groups=2)
    assert host(ids).tolist() == [[2 * size, size, size + 1], [2 * size, size, size + 1]]


@pytest.mark.parametrize("experts,groups,kept,top", [
    (6, 3, 2, 2), (8, 4, 3, 5), (48, 16, 9, 16), (256, 16, 12, 7), (60, 20, 11, 9), (128, 8, 5, 20),
    (600, 60, 41, 64)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_of_biases_next_to_the_lowest_number(dev, experts, groups, kept, top, scores):
    """Finite biases of which two have a sum below the least number of 32 bits, as masks put them in: groups
    that have none but such experts left are still there."""
    rng = np.random.default_rng(experts)
    most = float(np.finfo(np.float32).max)
    size = experts // groups
    for masked, missing in itertools.product((0.3, 0.9, 1.0), (0.0, 0.5, 0.9)):
        b = 0.1 * rng.standard_normal(experts)
        whole = np.repeat(rng.random(groups) < masked, size)  # groups at a time
        b[whole] = rng.choice([-most, -3e38, -2e38], whole.sum())
        x = rng.standard_normal((40, experts))
        x[rng.random(x.shape) < missing] = -np.inf
        x[0] = np.where(np.arange(experts) == 0, 1.0, np.where(whole, x[0], -np.inf))
        for dtype, rank in itertools.product((torch.float32, torch.bfloat16), (1, 2)):
            check_route(dev, x, top, dtype, b, scores=scores, groups=groups, top_groups=kept,
                        group_rank=rank)


def test_route_of_the_largest_logits(dev):
    """Of bf16 its own largest value is what an infinity counts as."""
    x = np.zeros((3, 70), np.float32)
    x[:, 40], x[:, 20], x[1, 3] = np.inf, 3.3895313892515355e38, np.inf
    for dtype in (torch.float32, torch.bfloat16):
        for E in (33, 70):
            check_route(dev, np.roll(x, -9, 1)[:, :E], 3, dtype)


def test_route_takes_rows_of_a_wider_matrix_and_given_results(dev):
    rng = np.random.default_rng(5)
    wide = on(rng.standard_normal((9, 100)).astype(np.float32), dev)
    x = wide[:, 17:17 + 48]
    ids = torch.full((9, 4), 77, dtype=torch.int32, device=dev)
    w = torch.zeros((9, 4), device=dev)
    got = ex.route(x, 4, ids=ids, weights=w)
    assert got[0] is ids and got[1] is w
    want, ww = H.route(host(x), 4)
    assert np.array_equal(host(ids), want) and np.allclose(host(w), ww, rtol=2.0 ** -22)
    assert ex.route(x[:0], 4)[0].shape == (0, 4)


# ---- arrange ---------------------------------------------------------------------------

def check_arrange(dev, ids, experts, first=0):
    got = ex.arrange(on(np.asarray(ids, np.int32), dev), experts, first)
    for x, y, what in zip(got, H.arrange(ids, experts, first), ("starts", "tokens", "place")):
        assert np.array_equal(host(x), y), what


@pytest.mark.parametrize("tokens,top,experts,first", [
    (0, 3, 5, 0), (1, 1, 1, 0), (1, 8, 128, 0), (5, 3, 7, 2), (63, 1, 9, 0), (64, 1, 9, 0),
    (65, 1, 9, 1), (700, 6, 60, 30), (1025, 4, 1024, 0), (4096, 1, 3, 0), (4097, 1, 3, 1),
    (5003, 7, 192, 0), (16384, 6, 192, 0)])
def test_arrange(dev, tokens, top, experts, first):
    rng = np.random.default_rng(tokens + top)
    ids = rng.integers(-1, first + experts + 3, (tokens, top))
    check_arrange(dev, ids, experts, first)
    check_arrange(dev, np.full_like(ids, first + experts - 1), experts, first)  # all the same one
    check_arrange(dev, np.full_like(ids, -1), experts, first)  # nobody's
    ids[::3] = np.int32(-2 ** 31)
    ids[1::3] = 2 ** 31 - 1
    check_arrange(dev, ids, experts, first)


def test_arrange_more_pairs_than_the_bits_of_one_pass(dev):
    rng = np.random.default_rng(8)
    check_arrange(dev, rng.integers(-1, 9, (100003, 6)), 8)
    check_arrange(dev, np.full((262145, 1), 2), 4)


# ---- product ---------------------------------------------------------------------------

def operands(rows, experts, n, k, seed):
    a, sfa = oracle.quant_fp8_1x128(oracle.randn(rows * k, seed).reshape(rows, k))
    b = np.empty((experts, n, k), np.uint8)
    sfb = np.empty((experts, (n + 127) // 128, k // 128), np.float32)
    for e in range(experts):
        b[e], sfb[e] = oracle.quant_fp8_128x128(oracle.randn(n * k, seed + 1 + e).reshape(n, k))
    return a, sfa, b, sfb


def check_product(dev, a, sfa, b, sfb, starts, rows=None, label="", cuts=(0,)):
    total = a.shape[0] if rows is None else len(rows)
    want, mass, written = H.product(a, sfa, b, sfb, starts, rows)
    args = [on(a, dev), on(sfa, dev), on(b, dev), on(sfb, dev), on(np.asarray(starts, np.int32), dev),
            None if rows is None else on(np.asarray(rows, np.int32), dev)]
    for cut in cuts:
        out = torch.full((total, b.shape[1]), 77.0, dtype=torch.bfloat16, device=dev)
        got = ex.product(*args, out=out, cut=cut)
        assert got is out
        bits = host(out.view(torch.int16)).view(np.uint16)
        assert (bits[~written] == 0x429A).all(), "rows that are nobody's have been written"
        _, st = bf16_compare(bits[written], want[written], mass[written])
        assert_parity(st, "product %s cut %d" % (label, cut))


CUTS = range(_lib.GA_EXPERTS_CUTS + 1)  # 0: what the sizes choose
COUNTS = {  # rows of each expert
    "one": [1], "single": [0, 1, 0, 0, 1, 1, 0], "few": [3, 0, 16, 17, 1, 15], "wave": [33, 64, 0, 65],
    "tile": [128, 1, 129, 127, 0], "large": [300, 0, 513, 256, 255], "skewed": [1, 700, 2, 0, 0, 3]}


@pytest.mark.parametrize("counts", sorted(COUNTS))
@pytest.mark.parametrize("n,k", [(16, 128), (200, 256), (130, 1152), (513, 640), (256, 1024)])
@pytest.mark.parametrize("gathered", [False, True])
def test_product(dev, counts, n, k, gathered):
    c = COUNTS[counts]
    starts = np.concatenate([[0], np.cumsum(c)])
    total = int(starts[-1]) + 5  # rows behind the last expert's
    rng = np.random.default_rng(n + k)
    m = max(1, total // 3) if gathered else total
    a, sfa, b, sfb = operands(m, len(c), n, k, seed=n * 3 + k)
    rows = None
    if gathered:
        rows = rng.integers(0, m, total)
        rows[rng.random(total) < 0.1] = -1
        rows[rng.random(total) < 0.05] = m
        rows[rng.random(total) < 0.02] = 2 ** 31 - 1
        rows[rng.random(total) < 0.02] = -2 ** 31
    check_product(dev, a, sfa, b, sfb, starts, rows, "%s %dx%d" % (counts, n, k), CUTS)


@pytest.mark.parametrize("experts", [63, 64, 65, 130, 1024])
def test_product_of_many_experts(dev, experts):
    rng = np.random.default_rng(experts)
    c = rng.integers(0, 4, experts)
    starts = np.concatenate([[0], np.cumsum(c)])
    a, sfa, b, sfb = operands(int(starts[-1]), experts, 32, 256, seed=experts)
    check_product(dev, a, sfa, b, sfb, starts, None, "%d experts" % experts, CUTS)


@pytest.mark.parametrize("starts", [[-5, 3, 3, 9, 40], [0, 0, 0, 0, 0], [7, 7, 12, 12, 2 ** 31 - 1],
                                    [-2 ** 31, -1, 4, 4, 20], [20, 20, 21, 22, 23],
                                    [-5, 3, 2, 9, 40], [7, 7, 30, 11, 20], [100, 200, 5, -1, 8],
                                    [2 ** 31 - 1, 0, -2 ** 31, 1, 2 ** 31 - 1], [9, 3, 12, 1, 17]])
def test_product_keeps_first_rows_inside(dev, starts):
    """First rows that pass the rows or decrease: taken as documented, nothing written elsewhere."""
    a, sfa, b, sfb = operands(20, 4, 48, 256, seed=4)
    check_product(dev, a, sfa, b, sfb, starts, None, str(starts), CUTS)
    guarded = torch.full((60, 48), 77.0, dtype=torch.bfloat16, device=dev)
    args = [on(a, dev), on(sfa, dev), on(b, dev), on(sfb, dev), on(np.array(starts, np.int32), dev)]
    for cut in CUTS:
        ex.product(*args, out=guarded[20:40], cut=cut)
        assert (guarded[:20] == 77).all() and (guarded[40:] == 77).all()


@pytest.mark.parametrize("experts", [70, 300, 1024])
def test_product_of_many_first_rows_that_decrease(dev, experts):
    rng = np.random.default_rng(experts)
    starts = rng.integers(-3, 60, experts + 1)
    a, sfa, b, sfb = operands(50, experts, 16, 128, seed=6)
    check_product(dev, a, sfa, b, sfb, starts, None, "%d" % experts, CUTS)


@pytest.mark.parametrize("k", [128, 384])
def test_product_of_one_row_gathered_many_times(dev, k):
    """Copies ahead of the last step, and of rows that are nowhere, from a matrix of one row."""
    a, sfa, b, sfb = operands(1, 2, 257, k, seed=k)
    rows = np.zeros(430, np.int32)
    rows[::7], rows[3::50] = -1, 1
    check_product(dev, a, sfa, b, sfb, np.array([0, 250, 430]), rows, "one row, K %d" % k, CUTS)


@pytest.mark.parametrize("counts", ["single", "few", "wave", "skewed"])
@pytest.mark.parametrize("n,k", [(144, 2816), (33, 3456), (72, 4224)])
@pytest.mark.parametrize("gathered", [False, True])
def test_product_of_long_k(dev, counts, n, k, gathered):
    """22, 27 and 33 steps: a wave's ring of few rows comes round more than once in each of two and
    four pieces of K, the last of them shorter."""
    c = COUNTS[counts]
    starts = np.concatenate([[0], np.cumsum(c)])
    total = int(starts[-1]) + 3
    rng = np.random.default_rng(n + k)
    m = max(1, total // 2) if gathered else total
    a, sfa, b, sfb = operands(m, len(c), n, k, seed=n + k)
    rows = None
    if gathered:
        rows = rng.integers(0, m, total)
        rows[rng.random(total) < 0.1] = -1
    check_product(dev, a, sfa, b, sfb, starts, rows, "%s %dx%d" % (counts, n, k), CUTS)


def strided(x, strides):
    """x in memory of its own with these strides (elements)."""
    size = 1 + sum((n - 1) * s for n, s in zip(x.shape, strides))
    view = torch.empty(size, dtype=x.dtype, device=x.device).as_strided(x.shape, strides)
    view.copy_(x)
    return view


@pytest.mark.parametrize("far", ["b", "out", "a", "gathered", "scales"])
def test_product_past_4_gib(dev, far):
    """Operands of which the last expert's weights, the last rows or their scales lie past 2^32 bytes, and
    gathered rows up to the last offset that a call takes (256 of 0xE00000 bytes)."""
    c, n, k = [3, 0, 140, 113, 64], 80, 384
    starts = np.concatenate([[0], np.cumsum(c)])
    total = int(starts[-1])
    rng = np.random.default_rng(7)
    rows = rng.permutation(np.arange(total) % 256) if far == "gathered" else None
    a, sfa, b, sfb = operands(total if rows is None else 256, len(c), n, k, seed=5)
    want, mass, _ = H.product(a, sfa, b, sfb, starts, rows)
    A, S, B, T = on(a, dev), on(sfa, dev), on(b, dev), on(sfb, dev)
    out = torch.empty((total, n), dtype=torch.bfloat16, device=dev)
    if far == "b":
        B = strided(B, (3 << 29, 1 << 20, 1))
    elif far == "out":
        out = strided(out, ((1 << 23) + 3, 1))
    elif far in ("a", "gathered"):
        A = strided(A, (0xE00000, 1))
    else:
        S, T = strided(S, ((1 << 28) + 8, 1)), strided(T, (3 << 28, 1 << 22, 1))
    args = [A, S, B, T, on(starts.astype(np.int32), dev),
            None if rows is None else on(rows.astype(np.int32), dev)]
    for cut in CUTS:
        out.fill_(5.0)
        ex.product(*args, out=out, cut=cut)
        bits = host(out.contiguous().view(torch.int16)).view(np.uint16)
        _, st = bf16_compare(bits, want, mass)
        assert_parity(st, "far %s cut %d" % (far, cut))


def test_product_of_strided_operands(dev):
    c = [40, 0, 9]
    starts = on(np.array([0, 40, 40, 49], np.int32), dev)
    a, sfa, b, sfb = operands(49, 3, 136, 384, seed=9)
    want, mass, _ = H.product(a, sfa, b, sfb, [0, 40, 40, 49])
    A = torch.zeros((49, 400), dtype=torch.uint8, device=dev)
    A[:, :384] = on(a, dev)
    S = torch.zeros((3, 64), device=dev)
    S[:, :49] = on(sfa, dev)
    B = torch.zeros((3, 140, 416), dtype=torch.uint8, device=dev)
    B[:, :136, :384] = on(b, dev)
    T = torch.zeros((3, 4, 7), device=dev)
    T[:, :2, :3] = on(sfb, dev)
    for (width, first), cut in itertools.product(((144, 0), (140, 0), (143, 1)), CUTS):
        O = torch.full((49, width), 5.0, dtype=torch.bfloat16, device=dev)
        out = O[:, first:first + 136]
        ex.product(A[:, :384], S[:, :49], B[:, :136, :384], T[:, :2, :3], starts, out=out, cut=cut)
        bits = host(out.contiguous().view(torch.int16)).view(np.uint16)
        _, st = bf16_compare(bits, want, mass)
        assert_parity(st, "strided")
        O[:, first:first + 136] = 5.0
        assert (O == 5.0).all()  # nothing beside


@pytest.mark.parametrize("n", [64, 255])
def test_product_rounds_to_the_nearest_bfloat16(dev, n):
    """Rows with one element, so that a result is a product in fp32: its rounding, ties, denormal
    numbers, what passes the largest, NaN."""
    rng = np.random.default_rng(n)
    rows, k, starts = 300, 256, np.array([0, 7, 7, 140, 300], np.int32)
    codes = np.setdiff1d(np.arange(256), [0x00, 0x80, 0x7F, 0xFF])
    a = np.zeros((rows, k), np.uint8)
    a[:, 3] = rng.choice(codes, rows)
    a[5, 3] = 0x7F
    b = rng.choice(codes, (4, n, k)).astype(np.uint8)
    power = rng.integers(-140, 118, rows)
    power[100:200] = rng.integers(-3, 3, 100)
    s = rng.choice([1.0, 1.5, 1.25, 1.75, 1 + 2.0 ** -9, 1 + 2.0 ** -23, 1.3], rows)
    sfa = np.ones((2, rows), np.float32)
    sfa[0] = np.ldexp(s, power)
    sfb = np.ones((4, (n + 127) // 128, 2), np.float32)
    table = oracle.e4m3_decode_table().astype(np.float32)
    expert = np.searchsorted(starts, np.arange(rows), side="right") - 1
    with np.errstate(all="ignore"):
        want = bf16(table[a[:, 3]][:, None] * table[b[expert, :, 3]] * sfa[0][:, None]).float()
    assert (want.abs() == np.inf).any() and (want[5] != want[5]).all()
    assert ((want != 0) & (want.abs() < 2.0 ** -126)).any()
    for cut in CUTS:
        out = ex.product(on(a, dev), on(sfa, dev), on(b, dev), on(sfb, dev), on(starts, dev), cut=cut)
        assert torch.equal(out.float().cpu().nan_to_num(nan=7e37), want.nan_to_num(nan=7e37))


def test_product_scales_with_infinity_stay_in_their_rows(dev):
    """An infinite or NaN scale of one row leaves the others, also those that are nowhere."""
    a, sfa, b, sfb = operands(6, 2, 32, 256, seed=11)
    sfa = sfa.copy()
    sfa[0, 0], sfa[1, 1] = np.inf, np.nan
    rows = np.array([2, -1, 0, 3, 1, 99, 4, 5], np.int32)
    for cut in CUTS:
        out = host(ex.product(on(a, dev), on(sfa, dev), on(b, dev), on(sfb, dev),
                              on(np.array([0, 5, 8], np.int32), dev), on(rows, dev), cut=cut).float())
        clean = np.array([0, 1, 3, 5, 6, 7])
        assert np.isfinite(out[clean]).all() and not np.isfinite(out[[2, 4]]).any()
        assert (out[[1, 5]] == 0).all()


# ---- activate --------------------------------------------------------------------------

def check_activate(x, q, s, live=None):
    live = len(x) if live is None else live
    y, want = H.activate(x[:live])
    q, s = host(q)[:live], host(s)[:, :live]
    # an element: 2^-23 of the exponential and six roundings to fp32; a scale: one of its elements,
    # and its division
    assert (np.abs(s - want) <= 2.0 ** -20.5 * want).all()
    v = oracle.e4m3_decode_table()[q].astype(np.float64)
    r = y / np.repeat(s.T.astype(np.float64), 128, 1)
    # the nearest code: half a step of its binade (2^-4 of a value, 2^-10 below 2^-6), and r's error
    assert (np.abs(v - r) <= np.maximum(np.abs(r) * 2.0 ** -4, 2.0 ** -10) + np.abs(r) * 2.0 ** -20).all()


@pytest.mark.parametrize("rows,inner", [(1, 128), (5, 256), (31, 128), (32, 384), (33, 1408),
                                        (200, 640), (1000, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_activate(dev, rows, inner, dtype):
    rng = np.random.default_rng(rows + inner)
    x = rng.standard_normal((rows, 2 * inner)) * np.exp(rng.standard_normal(2 * inner))
    x[0, :7] = (0.0, -0.0, 88.0, -88.0, 200.0, -200.0, 1e-30)
    x[-1, inner:inner + 128] = 0.0  # a block of zeros: scale 1
    x = torch.from_numpy(x.astype(np.float32)).to(dtype)
    q, s = ex.activate(x.to(dev))
    check_activate(host(x.double()), q, s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_activate_of_gates_far_below_zero(dev, dtype):
    """Gates down to -91.5, to which g / (1 + exp(-g)) is a normal number (2^-126) though exp(g) or exp(-g)
    is none: blocks of such gates alone, and beside others."""
    rng = np.random.default_rng(9)
    x = np.empty((50, 768), np.float32)
    x[:, :384] = rng.uniform(-91.5, -86.5, (50, 384))
    x[25:, :384:3] = rng.standard_normal((25, 128))
    x[:, 384:] = 1e6 * rng.standard_normal((50, 384))  # so that scales are normal numbers too
    x[40:, 128:256] = -89.0
    x = torch.from_numpy(x).to(dtype)
    q, s = ex.activate(x.to(dev))
    check_activate(host(x.double()), q, s)
    assert (host(s) < 2.0 ** -99)[:, :25].all() and (host(q)[:25] & 0x7F).max() == 0x7E
    # further on: denormal numbers, and zero
    x[:, :384] = -120.0
    q, s = ex.activate(x.to(dev))
    assert (s == 1).all() and (q & 0x7F == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_activate_of_strided_and_unaligned_rows(dev, dtype):
    rng = np.random.default_rng(2)
    for width, first in ((520, 8), (515, 3), (513, 1)):
        x = torch.from_numpy(rng.standard_normal((37, width)).astype(np.float32)).to(dtype)
        q, s = ex.activate(x.to(dev)[:, first:first + 512])
        check_activate(host(x.double())[:, first:first + 512], q, s)


@pytest.mark.parametrize("live", [0, 1, 31, 32, 33, 70, 100, -4])
def test_activate_up_to_the_last_row(dev, live):
    x = torch.randn((70, 256), device=dev)
    starts = torch.tensor([0, 3, live], dtype=torch.int32, device=dev)
    q0, s0 = ex.activate(x)
    q = torch.full((70, 128), 200, dtype=torch.uint8, device=dev)
    s = torch.full((1, 70), -3.0, device=dev)
    _lib.check(_lib.lib().ga_experts_activate(x.data_ptr(), 0, 70, 128, 256, q.data_ptr(), 128,
                                              s.data_ptr(), 70, starts.data_ptr() + 8, None))
    n = max(0, min(70, live))
    assert torch.equal(q[:n], q0[:n]) and torch.equal(s[:, :n], s0[:, :n])
    assert (q[n:] == 200).all() and (s[:, n:] == -3.0).all()
    got = ex.activate(x, starts)
    assert torch.equal(got[0][:n], q0[:n]) and torch.equal(got[1][:, :n], s0[:, :n])


def test_activate_quantises_as_the_quantiser(dev):
    """Infinities and NaN: the codes and scales that ops.quant_fp8_1x128 gives for the products."""
    x = torch.zeros((4, 512), device=dev)
    x[:, :256] = 20.0  # 1 / (1 + exp(-20)) = 1 - 2^-28.9: rounds to 1 in fp32, so y = 20 u
    x[:, 256:] = torch.randn((4, 256), device=dev)
    x[0, 300] = float("nan")
    x[3, 5] = float("inf")  # the gate itself: inf u
    x[1, 256] = float("inf")
    x[2, 257], x[2, 300] = -float("inf"), float("nan")
    q, s = ex.activate(x)
    q0, s0 = ops.quant_fp8_1x128(x[:, :256] * x[:, 256:])
    assert torch.equal(q, q0) and torch.equal(s, s0)
    x[2, 7] = -float("inf")  # NaN
    q, s = ex.activate(x)
    y = x[:, :256] * x[:, 256:]
    y[2, 7] = float("nan")
    q0, s0 = ops.quant_fp8_1x128(y)
    assert torch.equal(q, q0) and torch.equal(s, s0)


# ---- combine ---------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,top,n", [(1, 1, 8), (1, 8, 4096), (3, 8, 2056), (17, 6, 100),
                                          (50, 13, 129), (9, 64, 64), (200, 2, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_combine(dev, tokens, top, n, dtype):
    rng = np.random.default_rng(tokens * top + n)
    rows = max(1, tokens * top // 2)
    y = bf16(rng.standard_normal((rows, n)))
    place = rng.integers(-2, rows + 2, (tokens, top)).astype(np.int32)
    place[rng.random(place.shape) < 0.05] = 2 ** 31 - 1
    place[rng.random(place.shape) < 0.05] = -2 ** 31
    place[0] = -1  # a token without rows: zeros
    w = rng.standard_normal((tokens, top)).astype(np.float32)
    got = ex.combine(y.to(dev), on(place, dev), on(w, dev), dtype=dtype)
    want, mass = H.combine(host(y.float()), place, w)
    # `top` fused steps, half a step of the result's type each
    tol = top * 2.0 ** -24 * mass
    tol += (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) * (np.abs(want) + tol)
    assert (np.abs(host(got.double()) - want) <= tol).all()
    assert (host(got.float())[0] == 0).all()


def test_combine_leaves_what_is_not_there(dev):
    """Rows that no place names may hold anything, also the first one."""
    y = torch.full((5, 256), float("nan"), dtype=torch.bfloat16, device=dev)
    y[3] = 2.0
    place = torch.tensor([[3, -1], [-1, 3], [-7, 5]], dtype=torch.int32, device=dev)
    w = torch.tensor([[0.5, float("inf")], [float("nan"), 1.0], [1.0, 1.0]], device=dev)
    out = ex.combine(y, place, w)
    assert (out[0] == 1.0).all() and (out[1] == 2.0).all() and (out[2] == 0).all()
    none = ex.combine(y[:0], place, w, dtype=torch.float32)
    assert none.shape == (3, 256) and (none == 0).all()


def test_combine_of_strided_rows(dev):
    rng = np.random.default_rng(6)
    Y = bf16(rng.standard_normal((20, 300))).to(dev)
    place = on(rng.integers(0, 20, (7, 3)).astype(np.int32), dev)
    w = on(rng.standard_normal((7, 3)).astype(np.float32), dev)
    for first, width in ((0, 296), (1, 256), (8, 256)):
        O = torch.full((7, 299), 9.0, device=dev)
        out = O[:, first:first + width]
        ex.combine(Y[:, first:first + width], place, w, out=out)
        want, mass = H.combine(host(Y[:, first:first + width].float()), host(place), host(w))
        assert (np.abs(host(out) - want) <= 2.0 ** -21 * mass).all()
        out.fill_(9.0)
        assert (O == 9.0).all()


def test_rows_past_4_gib(dev):
    """Activation and sum of rows of which the last lie past 2^32 bytes."""
    rng = np.random.default_rng(4)
    x = torch.from_numpy(rng.standard_normal((20, 512)).astype(np.float32)).to(dev)
    q, s = ex.activate(strided(x, ((3 << 25) + 1, 1)))
    assert all(torch.equal(u, v) for u, v in zip((q, s), ex.activate(x)))
    y, place = x.bfloat16(), on(rng.integers(0, 20, (30, 3)).astype(np.int32), dev)
    w = on(rng.standard_normal((30, 3)).astype(np.float32), dev)
    out = strided(torch.zeros((30, 512), device=dev), ((3 << 24) + 5, 1))
    ex.combine(strided(y, ((3 << 26) + 3, 1)), place, w, out=out)
    assert torch.equal(out.contiguous(), ex.combine(y, place, w, dtype=torch.float32))


# ---- together --------------------------------------------------------------------------

class Layer:
    """A layer with experts first .. first + mine - 1 of `experts`."""

    def __init__(self, dev, hidden, inner, experts, top, first=0, mine=None, seed=0):
        mine = experts if mine is None else mine
        self.first, self.top, self.mine = first, top, mine
        g = torch.Generator(device=dev).manual_seed(seed)
        self.gate = torch.randn((experts, hidden), generator=g, device=dev) / hidden ** 0.5
        w1 = torch.randn((experts, 2 * inner, hidden), generator=g, device=dev) / hidden ** 0.5
        w2 = torch.randn((experts, hidden, inner), generator=g, device=dev) / inner ** 0.5
        both = [[ops.quant_fp8_128x128(w[e]) for e in range(first, first + mine)] for w in (w1, w2)]
        (self.w1, self.s1), (self.w2, self.s2) = (
            [torch.stack([p[i] for p in pairs]) for i in (0, 1)] for pairs in both)

    def __call__(self, x, stream=None):
        with torch.cuda.stream(stream) if stream is not None else torch.no_grad():
            logits = x.float() @ self.gate.t()
        ids, w = ex.route(logits, self.top, stream=stream)
        starts, tokens, place = ex.arrange(ids, self.mine, self.first, stream=stream)
        q, s = ops.quant_fp8_1x128(x, stream=stream)
        h = ex.product(q, s, self.w1, self.s1, starts, tokens, stream=stream)
        q, s = ex.activate(h, starts, stream=stream)
        y = ex.product(q, s, self.w2, self.s2, starts, stream=stream)
        return ex.combine(y, place, w, stream=stream)

    def plain(self, x):
        """The same from dequantised weights in float64, token by token."""
        def weights(q, s):
            v = q.view(torch.float8_e4m3fn).double()
            return v * s.double().repeat_interleave(128, 1)[:, :q.shape[1]].repeat_interleave(128, 2)

        w1, w2 = weights(self.w1, self.s1), weights(self.w2, self.s2)
        ids, w = ex.route(x.float() @ self.gate.t(), self.top)
        out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        for t, j in itertools.product(range(len(x)), range(self.top)):
            e = int(ids[t, j]) - self.first
            if 0 <= e < self.mine:
                g, u = (w1[e] @ x[t].double()).chunk(2)
                out[t] += w[t, j].double() * (w2[e] @ (u * g * torch.sigmoid(g)))
        return out


@pytest.mark.parametrize("tokens,first,mine", [(1, 0, None), (7, 0, None), (60, 0, None), (60, 3, 4)])
def test_layer(dev, tokens, first, mine):
    """A layer from logits to its sum against float64. What e4m3 leaves of the activations is an
    error of up to 2^-4 of an element, uniform within it: 2^-4 / sqrt(3) of its root mean square at
    the most; two such operands' errors add up to 0.052 of the output's, and twice that is the
    bound of a norm over many elements."""
    layer = Layer(dev, 256, 384, 10, 3, first, mine, seed=tokens)
    x = torch.randn((tokens, 256), device=dev).to(torch.bfloat16)
    got, want = layer(x).double(), layer.plain(x)
    assert (got - want).norm() <= 0.104 * want.norm()
    idle = want.abs().sum(1) == 0  # tokens none of whose experts are here
    assert (got[idle] == 0).all()


class Shard(Layer):
    """A layer by one cut of its products."""

    def rows(self, x, cut):
        """The layer's rows before their sum, their first rows, places and weights."""
        ids, w = ex.route(x.float() @ self.gate.t(), self.top)
        starts, tokens, place = ex.arrange(ids, self.mine, self.first)
        h = ex.product(*ops.quant_fp8_1x128(x), self.w1, self.s1, starts, tokens, cut=cut)
        q, s = ex.activate(h, starts)
        return ex.product(q, s, self.w2, self.s2, starts, cut=cut), starts, place, w


@pytest.mark.parametrize("cut", CUTS[1:])
def test_shards_by_the_same_cut_have_the_same_rows(dev, cut):
    """By one cut a row's sums do not depend on the experts that are held, so a shard has the whole's rows bit
    by bit, and sums differ by the order of their `top` fused steps alone, in the whole and in the
    parts."""
    whole = Shard(dev, 640, 512, 12, 4)
    x = torch.randn((70, 640), device=dev).bfloat16()
    y, starts, place, w = whole.rows(x, cut)
    want = ex.combine(y, place, w, dtype=torch.float32).double()
    mass = ex.combine(y.abs(), place, w, dtype=torch.float32).double()
    total = torch.zeros_like(want)
    for first in (0, 3, 6, 9):
        part = Shard(dev, 640, 512, 12, 4, first, 3)
        yp, sp, pp, wp = part.rows(x, cut)
        lo, hi = int(starts[first]), int(starts[first + 3])
        assert int(sp[-1]) == hi - lo and torch.equal(yp[:hi - lo], y[lo:hi])
        total += ex.combine(yp, pp, wp, dtype=torch.float32).double()
    assert ((total - want).abs() <= 2 * 4 * 2.0 ** -24 * mass).all()


@pytest.mark.parametrize("cuts", [(2, 3, 1, 8), (7, 5, 0, 2), (0, 0, 0, 0)])
def test_shards_by_other_cuts_add_up(dev, cuts):
    """A cut that sums K in other pieces changes h by a step of bfloat16 and so a code by a step: the parts'
    sum is held to the layer in float64, within the bound of test_layer."""
    x = torch.randn((40, 640), device=dev).bfloat16()
    want = Shard(dev, 640, 512, 12, 4).plain(x)
    got = torch.zeros_like(want)
    for first, cut in zip((0, 3, 6, 9), cuts):
        y, _, place, w = Shard(dev, 640, 512, 12, 4, first, 3).rows(x, cut)
        got += ex.combine(y, place, w).double()
    assert (got - want).norm() <= 0.104 * want.norm()


def test_layer_on_another_stream_and_in_a_graph(dev):
    layer = Layer(dev, 256, 256, 12, 4, seed=1)
    inputs = [torch.randn((33, 256), device=dev).to(torch.bfloat16) for _ in range(4)]
    want = [layer(x).clone() for x in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for x, w in zip(inputs, want):
        with torch.cuda.stream(side):
            got = layer(x)
        side.synchronize()
        assert torch.equal(got, w)
        got = layer(x, stream=side)  # and given to the calls
        side.synchronize()
        assert torch.equal(got, w)
    x = inputs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        layer(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = layer(x)
    for i in (1, 3, 0, 2, 1):
        x.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[i])
        assert torch.equal(layer(inputs[i]), want[i])  # the program's own calls between


def test_results_do_not_change_from_call_to_call(dev):
    """No sum depends on the order of workgroups."""
    rng = np.random.default_rng(12)
    ids = on(rng.integers(0, 9, (400, 3)).astype(np.int32), dev)
    starts, tokens, _ = ex.arrange(ids, 9)
    a, sfa, b, sfb = (on(v, dev) for v in operands(400, 9, 200, 512, seed=3))
    for cut in CUTS:
        outs = [ex.product(a, sfa, b, sfb, starts, tokens, cut=cut) for _ in range(5)]
        assert all(torch.equal(outs[0], o) for o in outs[1:])


# ---- refusals ----------------------------------------------------------------------------

def test_refusals(dev):
    x = torch.zeros((4, 16), device=dev)
    i = torch.zeros((4, 2), dtype=torch.int32, device=dev)
    for call, error in (
            (lambda: ex.route(x.half(), 2), TypeError), (lambda: ex.route(x[0], 2), ValueError),
            (lambda: ex.route(x.t(), 2), ValueError), (lambda: ex.route(x.cpu(), 2), ValueError),
            (lambda: ex.route(x, 0), ValueError), (lambda: ex.route(x, 17), GaError),
            (lambda: ex.route(x, 65), ValueError), (lambda: ex.route(x, 2 ** 32 + 2), ValueError),
            (lambda: ex.route(x, 2, groups=2 ** 32 + 2), ValueError),
            (lambda: ex.route(x, 2, groups=2, top_groups=2 ** 32 + 1), ValueError),
            (lambda: ex.route(x, 2, groups=2, group_rank=2 ** 32 + 2), ValueError),
            (lambda: ex.route(x, 2, groups=0), ValueError),
            (lambda: ex.route(x, 2, scale=1e39), GaError),
            (lambda: ex.arrange(i, 4, 2 ** 32), ValueError),
            (lambda: ex.arrange(i, 4, 2 ** 31 - 4), ValueError), (lambda: ex.route(x, 2, scores="tanh"), ValueError),
            (lambda: ex.route(x, 2, bias=x[0, :8]), ValueError),
            (lambda: ex.route(x, 2, bias=x[0].double()), TypeError),
            (lambda: ex.route(x, 2, groups=3), GaError),
            (lambda: ex.route(x, 2, groups=4, top_groups=5), ValueError),
            (lambda: ex.route(x, 2, ids=i.long()), TypeError),
            (lambda: ex.route(x, 2, weights=x[:, ::8]), ValueError),
            (lambda: ex.arrange(i.long(), 4), TypeError), (lambda: ex.arrange(i[:, ::2], 4), ValueError),
            (lambda: ex.arrange(i[0], 4), ValueError), (lambda: ex.arrange(i, 0), ValueError),
            (lambda: ex.arrange(i, 1025), ValueError), (lambda: ex.arrange(i, 4, -1), ValueError),
            (lambda: ex.arrange(i.cpu(), 4), ValueError),
            (lambda: ex.activate(x), ValueError), (lambda: ex.activate(x[0]), ValueError),
            (lambda: ex.activate(torch.zeros((2, 256), dtype=torch.float16, device=dev)), TypeError),
            (lambda: ex.activate(torch.zeros((2, 256), device=dev), i[0].long()), TypeError),
            (lambda: ex.combine(x, i, x[:, :2]), TypeError),
            (lambda: ex.combine(x.bfloat16(), i, x[:, :2]), ValueError),
            (lambda: ex.combine(x.bfloat16(), i, torch.zeros((4, 2), device=dev),
                                dtype=torch.float16), TypeError)):
        with pytest.raises(error):
            call()


def test_products_that_are_refused(dev):
    a = torch.zeros((6, 256), dtype=torch.uint8, device=dev)
    s = torch.zeros((2, 6), device=dev)
    b = torch.zeros((3, 20, 256), dtype=torch.uint8, device=dev)
    t = torch.zeros((3, 1, 2), device=dev)
    starts = torch.zeros(4, dtype=torch.int32, device=dev)
    rows = torch.zeros(5, dtype=torch.int32, device=dev)
    ok = dict(a=a, sfa=s, b=b, sfb=t, starts=starts, rows=rows)
    ex.product(**ok)
    for change, error in ((dict(a=a.char()), TypeError), (dict(a=a[0]), ValueError),
                          (dict(a=a[:, :128]), ValueError), (dict(a=a.cpu()), ValueError),
                          (dict(sfa=s.double()), TypeError), (dict(sfa=s[:, :5]), ValueError),
                          (dict(b=b[0]), ValueError), (dict(b=b.transpose(0, 2)), ValueError),
                          (dict(sfb=t[:, :, :1]), ValueError), (dict(starts=starts[:3]), ValueError),
                          (dict(starts=starts.long()), TypeError), (dict(rows=rows.long()), TypeError),
                          (dict(rows=rows[None]), ValueError), (dict(cut=9), ValueError),
                          (dict(cut=2 ** 32 + 1), ValueError),
                          (dict(out=torch.zeros((5, 21), dtype=torch.bfloat16, device=dev)), ValueError),
                          (dict(out=torch.zeros((5, 20), device=dev)), TypeError)):
        with pytest.raises(error):
            ex.product(**{**ok, **change})
    k = torch.zeros((6, 192), dtype=torch.uint8, device=dev)
    with pytest.raises((GaError, ValueError)):
        ex.product(k, s[:1], b[:, :, :192], t[:, :, :1], starts, rows)


def test_nothing_to_do(dev):
    i = torch.zeros((0, 2), dtype=torch.int32, device=dev)
    starts, tokens, place = ex.arrange(i, 3)
    assert starts.tolist() == [0, 0, 0, 0] and tokens.shape == (0,) and place.shape == (0, 2)
    a = torch.zeros((0, 256), dtype=torch.uint8, device=dev)
    b = torch.zeros((3, 20, 256), dtype=torch.uint8, device=dev)
    out = ex.product(a, torch.zeros((2, 0), device=dev), b, torch.zeros((3, 1, 2), device=dev), starts)
    assert out.shape == (0, 20)
    q, s = ex.activate(torch.zeros((0, 256), device=dev), starts)
    assert q.shape == (0, 128) and s.shape == (1, 0)
    y = ex.combine(torch.zeros((0, 20), dtype=torch.bfloat16, device=dev), place,
                   torch.zeros((0, 2), device=dev))
    assert y.shape == (0, 20)

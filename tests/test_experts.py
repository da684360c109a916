"""The experts' C entries without a GPU: what they refuse before any device call, and calls with
nothing to do."""
import ctypes
import importlib.util
import os

import numpy as np
import pytest

import experts_helpers as H
from gcnasm_amd import _lib

ARG, SHAPE = _lib.GA_ERR_ARG, _lib.GA_ERR_SHAPE


def set_all(x, kw):
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def route(**kw):
    a = _lib.ExpertsRouteArgs(0x1000, None, 0x2000, 0x3000, 64, 0, 3, 64, 6, 0, 1, 1, 1, 1, 1.0)
    return _lib.lib().ga_experts_route(ctypes.byref(set_all(a, kw)), None)


@pytest.mark.parametrize("change,status", [
    (dict(logits=None), ARG), (dict(ids=None), ARG), (dict(weights=None), ARG),
    (dict(in_dtype=2), ARG), (dict(in_dtype=-1), ARG), (dict(scores=2), ARG), (dict(scores=-1), ARG),
    (dict(tokens=-1), ARG), (dict(experts=0), ARG), (dict(experts=-5), ARG), (dict(top=0), ARG),
    (dict(top=-1), ARG), (dict(groups=0), ARG), (dict(top_groups=0), ARG), (dict(top_groups=2), ARG),
    (dict(group_rank=0), ARG), (dict(group_rank=3), ARG), (dict(scale=float("nan")), ARG),
    (dict(scale=float("inf")), ARG), (dict(experts=1025, stride_logits=1025), SHAPE),
    (dict(top=65), SHAPE), (dict(groups=65, top_groups=65, experts=650, stride_logits=650), SHAPE),
    (dict(groups=3, top_groups=3), SHAPE), (dict(groups=16, top_groups=1), SHAPE),
    (dict(stride_logits=63), SHAPE), (dict(stride_logits=-64), SHAPE)])
def test_routes_that_are_refused(change, status):
    assert route(**change) == status
    assert _lib.lib().ga_last_error()


def test_arrangements_that_are_refused():
    l = _lib.lib()
    ok = [0x1000, 3, 4, 8, 0, 0x2000, 0x3000, 0x4000, None]
    for at, bad, status in ((0, None, ARG), (1, -1, ARG), (2, 0, ARG), (3, 0, ARG), (4, -1, ARG),
                            (5, None, ARG), (6, None, ARG), (7, None, ARG), (2, 65, SHAPE),
                            (3, 1025, SHAPE), (1, 1 << 29, SHAPE), (4, 0x7FFFFFF8, SHAPE)):
        x = list(ok)
        x[at] = bad
        assert l.ga_experts_arrange(*x) == status, (at, bad)


def product(**kw):
    a = _lib.ExpertsProductArgs(0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000, 10, 256, 10,
                                300 * 256, 256, 6, 2, 300, 4, 20, 300, 256, 0)
    return _lib.lib().ga_experts_product(ctypes.byref(set_all(a, kw)), None)


@pytest.mark.parametrize("change,status", [
    (dict(a=None), ARG), (dict(sfa=None), ARG), (dict(b=None), ARG), (dict(sfb=None), ARG),
    (dict(starts=None), ARG), (dict(out=None), ARG), (dict(experts=0), ARG), (dict(rows=-1), ARG),
    (dict(n=0), ARG), (dict(k=0), ARG), (dict(cut=-1), ARG), (dict(cut=9), ARG), (dict(a_rows=-1), ARG), (dict(experts=1025), SHAPE), (dict(rows=0x7FFF0001), SHAPE),
    (dict(k=192), _lib.GA_ERR_GROUP), (dict(a_rows=0), SHAPE), (dict(rows_of=None), SHAPE),
    (dict(a=0x1008), SHAPE), (dict(b=0x3004), SHAPE), (dict(stride_a=264), SHAPE),
    (dict(stride_b=264), SHAPE), (dict(stride_b_expert=300 * 256 + 8), SHAPE),
    (dict(stride_a=240), SHAPE), (dict(stride_b=240), SHAPE), (dict(stride_out=299), SHAPE),
    (dict(stride_sfa=9), SHAPE), (dict(stride_sfb=1), SHAPE), (dict(stride_b_expert=-16), SHAPE),
    (dict(stride_sfb_expert=-1), SHAPE), (dict(stride_a=1 << 24), SHAPE),
    (dict(stride_b=1 << 24), SHAPE),
    # gathered rows of a past the offsets of 32 bits; without a map there is no such limit
    (dict(a_rows=1 << 24, stride_sfa=1 << 24), SHAPE),
    (dict(stride_sfa=0x0FFF0000 // 8 + 1), SHAPE),
    (dict(rows_of=None, rows=10, stride_sfa=(1 << 29) + 1), SHAPE),
    (dict(stride_sfb=1 << 29), SHAPE)])
def test_products_that_are_refused(change, status):
    assert product(**change) == status
    assert _lib.lib().ga_last_error()


def test_activations_that_are_refused():
    l = _lib.lib()
    ok = [0x1000, 1, 5, 256, 512, 0x2000, 256, 0x3000, 5, None, None]
    for at, bad, status in ((0, None, ARG), (1, 2, ARG), (2, -1, ARG), (3, 0, ARG), (3, 64, SHAPE),
                            (4, 511, SHAPE), (5, None, ARG), (5, 0x2004, SHAPE), (6, 255, SHAPE),
                            (6, 260, SHAPE), (7, None, ARG), (8, 4, SHAPE)):
        x = list(ok)
        x[at] = bad
        assert l.ga_experts_activate(*x) == status, (at, bad)
    x = list(ok)  # 2^31 rows of 2^30 elements are more than a launch
    x[2], x[3], x[4], x[6], x[8] = 0x7FFFFFFF, 0x3FFFFF80, 0x7FFFFF00, 0x3FFFFF80, 0x7FFFFFFF
    assert l.ga_experts_activate(*x) == SHAPE


def test_sums_that_are_refused():
    l = _lib.lib()
    ok = [0x1000, 9, 100, 100, 0x2000, 0x3000, 4, 3, 0x4000, 0, 100, None]
    for at, bad, status in ((0, None, ARG), (1, -1, ARG), (2, 0, ARG), (3, 99, SHAPE), (4, None, ARG),
                            (5, None, ARG), (6, -1, ARG), (7, 0, ARG), (8, None, ARG), (9, 2, ARG),
                            (10, 99, SHAPE), (2, 0x7FFF0001, SHAPE)):
        x = list(ok)
        x[at] = bad
        assert l.ga_experts_combine(*x) == status, (at, bad)


def test_nothing_to_do_is_no_error():
    l = _lib.lib()
    assert route(tokens=0, logits=None, ids=None, weights=None) == 0
    assert product(rows=0, a=None, sfa=None, a_rows=0) == 0
    assert l.ga_experts_activate(None, 1, 0, 256, 512, None, 256, None, 0, None, None) == 0
    assert l.ga_experts_combine(0x1000, 9, 100, 100, None, None, 0, 3, None, 0, 100, None) == 0


@pytest.mark.parametrize("args", [["--shards", "0"], ["--shards", "9", "--experts", "8"],
                                  ["--shards", "2", "--shard", "2"], ["--shard", "-1"]])
def test_shards_that_the_example_refuses(args, capsys):
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples",
                        "experts_layer.py")
    spec = importlib.util.spec_from_file_location("experts_layer_cpu", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    with pytest.raises(SystemExit):
        example.main(args)
    assert "--shard" in capsys.readouterr().err


def test_null_arguments():
    l = _lib.lib()
    assert l.ga_experts_route(None, None) == ARG
    assert l.ga_experts_product(None, None) == ARG


def test_the_definition_by_hand():
    """The oracle itself, on values worked out by hand."""
    ids, w = H.route([[0.0, 1.0, 1.0, -np.inf]], 2)
    assert ids.tolist() == [[1, 2]] and np.allclose(w, 0.5)
    ids, w = H.route([[0.0, 0.0, 0.0, 0.0]], 2, bias=[0, 0, 1, 0], kind="sigmoid", groups=2,
                     top_groups=1, scale=3.0)
    assert ids.tolist() == [[2, 3]] and np.allclose(w, 1.5)
    # the larger pair wins with group_rank 2, the largest single one with 1
    x = [[3.0, -9.0, 2.0, 2.0]]
    assert H.route(x, 1, kind="sigmoid", groups=2, top_groups=1, group_rank=2)[0].tolist() == [[2]]
    assert H.route(x, 1, kind="sigmoid", groups=2, top_groups=1, group_rank=1)[0].tolist() == [[0]]
    assert H.route([[-np.inf, np.nan]], 2)[0].tolist() == [[-1, -1]]
    s, t, p = H.arrange([[1, 0], [1, 7]], 2)
    assert s.tolist() == [0, 1, 3] and t.tolist() == [0, 0, 1, -1] and p.tolist() == [[1, 0], [2, -1]]
    assert H.ranges([-3, 5, 2, 99], 20) == [(0, 5), (5, 5), (5, 20)]

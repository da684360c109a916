"""Eviction's selection in each of its forms: which one runs goes by the most tokens that may be looked
at (table and weights' width), up to 8192, up to 65536, or more; a short sequence under a wide table
takes the form of the wide one. Indices, weights and bytes against the definition."""
import numpy as np
import pytest
import torch

import mx4_helpers as H
from gcnasm_amd import mx4_cache as mc
from test_gpu_mx4_cache import host

pytestmark = pytest.mark.gpu

KINDS = ["random", "equal", "few values", "nan", "both zeros"]


def weights_of(kind, shape, rng):
    w = rng.standard_normal(shape).astype(np.float32)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "few values":
        w = rng.integers(0, 3, shape).astype(np.float32)
    elif kind == "nan":
        w[rng.random(shape) < 0.02] = np.nan
    elif kind == "both zeros":
        w = np.where(rng.random(shape) < 0.5, np.float32(0.0), np.float32(-0.0))
    return w


def chosen(w, length, keep, recent):
    """As H.evict, by a stable sort (which takes a hundred thousand tokens at once)."""
    if length <= keep:
        return np.arange(length)
    old = length - recent
    x = w[:old].astype(np.float64)
    x = np.where(np.isnan(x), np.inf, x)
    order = np.lexsort((np.arange(old), -x, ~np.isnan(w[:old])))
    return np.concatenate([np.sort(order[:keep - recent]), np.arange(old, length)]).astype(int)


def test_the_oracles_agree():
    rng = np.random.default_rng(1)
    for kind in KINDS:
        w = weights_of(kind, 700, rng)
        for length, keep, recent in ((700, 100, 10), (650, 1, 0), (640, 64, 64), (20, 30, 3)):
            assert np.array_equal(chosen(w, length, keep, recent), H.evict(w, length, keep, recent))


# width: around the cuts between the forms; lens: around the stretches that a wave takes
# (64 tokens for each 1024) and the groups of registers (16 of them)
SHAPES = [(8192, [8192, 8191, 1025, 1024, 63]), (8193, [8193, 4097, 700, 300, 0]),
          (17000, [16385, 17000, 15360, 1040]), (65536, [65536, 65535, 49153, 5]),
          (65537, [65537, 65536, 1024, 130]), (100001, [100001, 99000, 66000, 2000, 1])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width,lens", SHAPES, ids=[str(w) for w, _ in SHAPES])
def test_selection(dev, width, lens, kind):
    print("selection", width, lens, kind, flush=True)
    D, P, h, n = 64, 64, 1, len(lens)
    rng = np.random.default_rng(width)
    pages = -(-width // P)
    w = weights_of(kind, (n, h, width), rng)
    for keep, recent in ((200, 20), (1000, 0), (129, 129)):
        need = -(-keep // P)
        table = np.arange(n * pages, dtype=np.int32).reshape(n, pages)
        dst = np.arange(n * need, dtype=np.int32).reshape(n, need) + n * pages
        cache = torch.randint(0, 255, (n * (pages + need), h, mc.page_bytes(P, D)), device=dev,
                              dtype=torch.uint8)
        before = host(cache).copy()
        kept, new_lens, nw = mc.evict(cache, torch.from_numpy(table).to(dev),
                                      torch.tensor(lens, dtype=torch.int32, device=dev),
                                      torch.from_numpy(w).to(dev), keep, recent,
                                      torch.from_numpy(dst).to(dev), D)
        kept, nw, after = host(kept), host(nw), host(cache)
        assert host(new_lens).tolist() == [min(x, keep) for x in lens]
        places = H.places(P, D)
        for b, length in enumerate(lens):
            want = chosen(w[b, 0], length, keep, recent)
            m = len(want)
            np.testing.assert_array_equal(kept[b, 0, :m], want)
            np.testing.assert_array_equal(nw[b, 0, :m], w[b, 0][want])
            assert (kept[b, 0, m:] == -1).all() and (nw[b, 0, m:] == 0).all()
            j = np.arange(m)
            for p in places:
                np.testing.assert_array_equal(after[dst[b][j // P], 0][j[:, None], p[j % P]],
                                              before[table[b][want // P], 0][j[:, None],
                                                                             p[want % P]])

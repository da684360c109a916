"""The serving example: its lengths and pages through evictions, and its output before
the first one against the layer computed in float64 from what the cache holds."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import mx4_helpers as H

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples",
                    "mx4_cache_serving.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("mx4_cache_serving", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_runs_through_evictions(example, capsys):
    server, y = example.main(["--seqs", "3", "--prompt", "150", "--steps", "60", "--keep", "96",
                              "--recent", "32", "--slack", "20", "--hidden", "256", "--heads", "4",
                              "--kv-heads", "2", "--head-dim", "64"])
    assert torch.isfinite(y.float()).all() and tuple(y.shape) == (3, 256)
    assert server.evictions >= 2 and max(server.lens) < 96 + 60
    held = [p for h in server.pages.held for p in h]
    assert len(set(held)) == len(held) and not set(held) & set(server.pages.free)
    assert len(held) + len(server.pages.free) == server.cache.shape[0]
    w = server.weights.cpu()
    for b, n in enumerate(server.lens):
        assert (w[b, :, :n] >= 0).all() and (w[b, :, n:] == 0).all()
    assert "a step" in capsys.readouterr().out


def test_weights_follow_their_tokens(example):
    """Every row of a sequence gives its 1 to the tokens it sees, group heads a kv head: the sums
    over the tokens before the first eviction, and the kept tokens' after it."""
    dev = torch.device("cuda")
    layer = example.Layer(256, 4, 2, 64, dev)
    server = example.Server(layer, 2, keep=64, recent=16, slack=8, prompt=40)
    x = torch.randn((40 + 25, 256), device=dev).bfloat16()
    server.step(x, [40, 25])
    rows = [40, 25]
    while server.evictions == 0:
        before = server.weights
        total = before.double().sum(-1).cpu().numpy()
        want = 2.0 * np.array(rows)[:, None]
        # a term's score and exponential: 2^-20 of it covers fp32's roundings here
        assert (np.abs(total - want) <= want * 2.0 ** -14).all()
        server.step(torch.randn((2, 256), device=dev).bfloat16(), [1, 1])
        rows = [r + 1 for r in rows]
    assert server.lens == [64, min(rows[1], 64)]
    total = server.weights.double().sum(-1).cpu().numpy()
    assert (total <= 2.0 * np.array(rows)[:, None] * (1 + 2.0 ** -14)).all()
    # the second sequence was short enough to be moved whole
    assert abs(total[1] - 2.0 * rows[1]).max() <= 2.0 * rows[1] * 2.0 ** -14


def test_output_of_a_step(example):
    dev = torch.device("cuda")
    layer = example.Layer(512, 8, 2, 128, dev)
    server = example.Server(layer, 2, keep=200, recent=50, slack=20, prompt=130)
    layer.finish = lambda out: out
    x = torch.randn((130 + 77, 512), device=dev).bfloat16()
    got = server.step(x, [130, 77])
    q = layer.project(x)[0].double().cpu().numpy()
    cache, table = server.cache.cpu().numpy(), server.pages.table.cpu().numpy()
    at = 0
    for b, n in enumerate((130, 77)):
        k, v, there = H.tokens(cache, table[b], 64, 128, n)
        out, _, _, tol, _ = H.attention(q[at:at + n], k, v, there, n, n, True, 0, 128 ** -0.5, 0.0)
        assert (np.abs(got[at:at + n].double().cpu().numpy() - out) <= tol).all()
        at += n

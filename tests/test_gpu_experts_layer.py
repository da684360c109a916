"""The example of a layer of experts: its step against the layer computed in float64 from the
quantised weights, its shards against the whole, its captured form against the eager one."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "experts_layer.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("experts_layer", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def values(q, s):
    """Weights [experts, N, K] in float64."""
    s = s.double().repeat_interleave(128, 1)[:, :q.shape[1]].repeat_interleave(128, 2)
    return q.view(torch.float8_e4m3fn).double() * s


@pytest.mark.parametrize("args", [[], ["--graph"], ["--groups", "4", "--top-groups", "2"],
                                  ["--scores", "softmax", "--shards", "2", "--shard", "1"]])
def test_runs(dev, example, args, capsys):
    layer, y = example.main(["--tokens", "9", "--hidden", "256", "--inner", "128", "--experts", "8",
                             "--top", "2", "--steps", "5"] + args)
    assert tuple(y.shape) == (9, 256) and y.dtype == torch.bfloat16
    assert torch.isfinite(y.float()).all()
    assert "a step" in capsys.readouterr().out


@pytest.mark.parametrize("experts,shards", [(10, 3), (7, 7), (9, 2)])
def test_every_expert_is_one_shards(dev, example, experts, shards):
    held = []
    for i in range(shards):
        layer, _ = example.main(["--tokens", "3", "--hidden", "128", "--inner", "128", "--experts",
                                 str(experts), "--top", "2", "--steps", "1", "--shards", str(shards),
                                 "--shard", str(i)])
        assert len(layer.w1) == layer.held
        held += range(layer.first, layer.first + layer.held)
    assert held == list(range(experts))


def test_a_step(dev, example):
    """Rounding activations to e4m3 twice is off by up to 2^-4 of an element each, at the most
    2^-4 / sqrt(3) of the root mean square; two such errors come to 0.052 of the output's norm, and twice
    that is the bound."""
    layer = example.Layer(256, 384, 10, 3, dev, groups=5, top_groups=2)
    x = torch.randn((40, 256), device=dev).bfloat16()
    ids, w = layer.route(x)
    w1, w2 = values(layer.w1, layer.s1), values(layer.w2, layer.s2)
    want = torch.zeros((40, 256), dtype=torch.float64, device=dev)
    for j in range(3):
        h = torch.matmul(w1[ids[:, j].long()], x.double()[..., None]).squeeze(2)
        gate, up = h.chunk(2, 1)
        h = up * gate * torch.sigmoid(gate)
        want += w[:, j, None].double() * torch.matmul(w2[ids[:, j].long()], h[..., None]).squeeze(2)
    assert (layer(x).double() - want).norm() <= 0.104 * want.norm()


def test_shards_add_up(dev, example):
    """Each expert's rows are the same on its shard as in the whole, so the parts' sum is off by
    the roundings to bf16 alone, half a step (2^-8) of the whole and of each part, and those of fp32
    sums."""
    x = torch.randn((70, 256), device=dev).bfloat16()
    whole = example.Layer(256, 256, 12, 4, dev)(x).double()
    parts = [example.Layer(256, 256, 12, 4, dev, first, 3)(x).double() for first in (0, 3, 6, 9)]
    bound = 2.0 ** -8 * (whole.abs() + sum(p.abs() for p in parts)) + 2.0 ** -20
    assert ((sum(parts) - whole).abs() <= bound).all()


def test_captured_steps(dev, example):
    layer = example.Layer(256, 128, 16, 4, dev, scores="softmax")
    step = example.Graph(layer, 33, 256, dev)
    xs = [torch.randn((33, 256), device=dev).bfloat16() for _ in range(3)]
    for i in (0, 2, 1, 1, 0):
        got = step(xs[i]).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, layer(xs[i]))

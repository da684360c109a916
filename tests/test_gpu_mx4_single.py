"""One token, one row, one head: a dimension of one element has a stride that says nothing, and a
tensor that is contiguous all the same (so .contiguous() is itself) may have any there."""
import pytest
import torch

from gcnasm_amd import mx4_cache as mc
from test_gpu_mx4_cache import Setup

pytestmark = pytest.mark.gpu


def odd(x, dims):
    """x where dimensions `dims`, of one element, have strides that are no multiple of 4."""
    stride = list(x.stride())
    for d in dims:
        assert x.shape[d] == 1
        stride[d] = 4099
    y = x.as_strided(x.shape, stride)
    assert y.is_contiguous() and y.data_ptr() == x.data_ptr()
    return y


@pytest.mark.parametrize("h,dims", [(2, (0,)), (1, (0,)), (1, (1,)), (1, (0, 1))])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_strides_of_one_element(dev, D, h, dims):
    print("single", D, h, dims, flush=True)
    s = Setup(dev, [300], [1], h, h, D, 64, seed=71)
    for dtype in (torch.float32, torch.bfloat16):
        k, v = (torch.randn((1, h, D), device=dev).to(dtype) for _ in range(2))
        a, b = s.cache.clone(), s.cache.clone()
        slot = torch.tensor([int(s.slots[299])], device=dev)
        mc.append(a, k, v, slot)
        mc.append(b, odd(k, dims), odd(v, dims), slot)
        assert torch.equal(a, b) and not torch.equal(a, s.cache)
    out, lse = mc.attention(s.q, s.cache, s.table_d, s.lens_d)
    given = torch.empty_like(s.q)
    got = mc.attention(odd(s.q, dims), s.cache, s.table_d, s.lens_d, out=odd(given, dims))
    assert torch.equal(given, out) and torch.equal(got[1], lse)
    s.check(out, lse, s.expected())
    w = mc.attention_weights(s.q, s.cache, s.table_d, s.lens_d, lse)
    assert torch.equal(w, mc.attention_weights(odd(s.q, dims), s.cache, s.table_d, s.lens_d, lse))


def test_strides_of_more_are_refused(dev):
    s = Setup(dev, [30, 20], [1, 1], 2, 2, 128, 64, seed=72)
    wide = torch.zeros((2, 2 * 128 + 2), dtype=torch.bfloat16, device=dev)
    with pytest.raises(Exception, match="multiples of"):
        mc.attention(wide[:, :256].view(2, 2, 128), s.cache, s.table_d, s.lens_d)
    with pytest.raises(Exception, match="multiples of"):
        mc.append(s.cache, wide[:, :256].view(2, 2, 128), s.q, torch.arange(2, device=dev))

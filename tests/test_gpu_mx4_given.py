"""Workspaces and results that the caller of the MXFP4 cache's operators keeps: sizes asked for,
exactly so large, too small; a whole step with an eviction that allocates nothing."""
import numpy as np
import pytest
import torch

from gcnasm_amd import GaError, _lib, mx4_cache as mc
from test_gpu_mx4_cache import Setup, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,window", [([200, 30], 0), ([300, 250], 40), ([1, 1], 0)])
def test_a_workspace_for_the_weights(dev, rows, window):
    print("workspace", rows, window, flush=True)
    s = Setup(dev, [400, 310], rows, 8, 2, 128, 64, seed=61)
    kw = dict(q_starts=s.starts_d, max_q=max(rows), max_len=400, window=window)
    lse = torch.from_numpy(np.concatenate([p[1] for p in s.expected(window=window)]).astype(
        np.float32)).to(dev)
    args = (s.q, s.cache, s.table_d, s.lens_d)
    need = mc.attention_weights_workspace_bytes(*args, 410, **kw)
    assert (need > 0) == (max(rows) > 1)
    want = mc.attention_weights(*args, lse, width=410, **kw)
    ws = torch.full((need + 256,), 0x5A, dtype=torch.uint8, device=dev)
    got = mc.attention_weights(*args, lse, width=410, workspace=ws[:need], **kw)
    assert torch.equal(got, want) and (ws[need:] == 0x5A).all()
    if need:
        with pytest.raises(GaError) as e:
            mc.attention_weights(*args, lse, width=410, workspace=ws[:need - 4], **kw)
        assert e.value.status == _lib.GA_ERR_WORKSPACE
    with pytest.raises((GaError, ValueError)):
        mc.attention_weights_workspace_bytes(*args, -1, **kw)
    with pytest.raises((GaError, ValueError)):
        mc.attention_weights_workspace_bytes(*args, 2 ** 32 + 1, **kw)


def test_evictions_results_are_given(dev):
    s = Setup(dev, [300, 77], [1, 1], 4, 2, 128, 16, seed=62)
    w = torch.rand((2, 2, 300), device=dev)
    first = s.cache.shape[0]
    pool = torch.cat([s.cache] * 2)
    dst = torch.arange(first, first + 14, dtype=torch.int32, device=dev).view(2, 7)
    want = mc.evict(pool, s.table_d, s.lens_d, w, 100, 9, dst, 128)
    kept = torch.full((2, 2, 100), -9, dtype=torch.int32, device=dev)
    lens = torch.full((4,), -9, dtype=torch.int32, device=dev)
    nw = torch.full((2, 2, 120), 7.0, device=dev)
    got = mc.evict(pool, s.table_d, s.lens_d, w, 100, 9, dst, 128, nw, kept=kept, new_lens=lens[1:3])
    assert got[0] is kept and got[1].data_ptr() == lens[1:].data_ptr() and got[2] is nw
    assert torch.equal(kept, want[0]) and host(lens).tolist() == [-9, 100, 77, -9]
    assert torch.equal(nw[:, :, :100], want[2]) and (nw[:, :, 100:] == 0).all()
    bad = [dict(kept=kept[:, :, :99]), dict(kept=kept.long()), dict(new_lens=lens),
           dict(kept=torch.empty((2, 100, 2), dtype=torch.int32, device=dev).transpose(1, 2)),
           dict(new_lens=lens[1:3].cpu())]
    for kw in bad:
        with pytest.raises((GaError, ValueError, TypeError)):
            mc.evict(pool, s.table_d, s.lens_d, w, 100, 9, dst, 128, **kw)


def test_a_step_into_given_tensors_allocates_nothing(dev):
    s = Setup(dev, [700, 300], [100, 120], 8, 2, 128, 64, seed=63)
    rows = dict(q_starts=s.starts_d, max_q=120, max_len=700)
    args = (s.q, s.cache, s.table_d, s.lens_d)
    out, lse = torch.empty_like(s.q), torch.empty((220, 8), device=dev)
    ws = torch.empty(max(1, mc.attention_workspace_bytes(*args, **rows)), dtype=torch.uint8,
                     device=dev)
    ww = torch.empty(max(1, mc.attention_weights_workspace_bytes(*args, 700, **rows)),
                     dtype=torch.uint8, device=dev)
    w = torch.zeros((2, 2, 700), device=dev)
    kept = torch.empty((2, 2, 128), dtype=torch.int32, device=dev)
    new_lens, nw = torch.empty_like(s.lens_d), torch.empty((2, 2, 128), device=dev)
    dst = s.table_d[:, :2].clone().fill_(-1)  # a page outside the cache takes nothing

    def step():
        mc.attention(*args, out=out, lse=lse, workspace=ws, **rows)
        mc.attention_weights(*args, lse, out=w, workspace=ww, **rows)
        mc.evict(s.cache, s.table_d, s.lens_d, w, 128, 16, dst, 128, nw, kept=kept,
                 new_lens=new_lens)

    step()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    step()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    s.check(out, lse, s.expected())
    assert host(new_lens).tolist() == [128, 128]

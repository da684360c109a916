"""Calls whose bounds ask for more threads than a launch takes (2^32): max_q, which only chooses the
launch, is every row of the call by default."""
import numpy as np
import pytest
import torch

import mx4_helpers as H
from gcnasm_amd import mx4_cache as mc
from test_gpu_mx4_cache import Setup, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,seqs,n,group", [(64, 2048, 4, 16), (256, 4096, 2, 16)])
def test_rows_of_many_sequences_without_a_bound(dev, D, seqs, n, group):
    """seqs * 8 kv heads * (seqs * n * group / 128) workgroups of 256 threads: 2^32 threads."""
    assert seqs * 8 * (seqs * n * group // 128) * 256 >= 1 << 32
    print("launch", D, seqs, n, flush=True)
    s = Setup(dev, [20, 17], [n, n], 8 * group, 8, D, 16, seed=51)
    copies = seqs // 2
    q = s.q.repeat(copies, 1, 1)
    table, lens = s.table_d.repeat(copies, 1), s.lens_d.repeat(copies)
    starts = torch.arange(seqs + 1, dtype=torch.int32, device=dev) * n
    out, lse = mc.attention(q, s.cache, table, lens, starts)
    assert (out.view((copies,) + s.q.shape) == out[:2 * n]).all()
    assert (lse.view(copies, 2 * n, -1) == lse[:2 * n]).all()
    s.check(out[:2 * n], lse[:2 * n], s.expected())

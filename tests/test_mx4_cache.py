"""The MXFP4 cache's C entries without a GPU: what they refuse before any device call, and the
sizes and layout that the header gives."""
import ctypes

import numpy as np
import pytest

import mx4_helpers as H
from gcnasm_amd import _lib


def cache(**kw):
    c = _lib.Mx4Cache(0x10000, 8, 4 * 2 * 8704, 2, 128, 64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attention(**kw):
    a = _lib.Mx4AttentionArgs()
    for n in ("q", "out", "lse", "table", "lens"):
        setattr(a, n, 0x10000)
    a.stride_q_row = a.stride_out_row = 4 * 128
    a.stride_q_head = a.stride_out_head = 128
    a.stride_lse_row, a.stride_table = 4, 5
    a.seqs = a.rows = 3
    a.heads, a.table_pages, a.max_q, a.max_len, a.causal = 4, 5, 1, 100, 1
    a.scale = 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_page_bytes():
    l = _lib.lib()
    for P in (16, 32, 64, 128, 256):
        for D in (64, 128, 256):
            assert l.ga_mx4_page_bytes(P, D) == P * D * 17 // 16
            every = np.concatenate([x.ravel() for x in H.places(P, D)])
            assert np.array_equal(np.sort(every), np.arange(P * D * 17 // 16))  # no byte twice
    for P, D in ((8, 128), (24, 128), (512, 128), (0, 128), (-16, 128), (64, 32), (64, 96), (64, 0)):
        assert l.ga_mx4_page_bytes(P, D) == 0


@pytest.mark.parametrize("change,status", [
    (dict(pages=None), _lib.GA_ERR_ARG), (dict(pages=0x10008), _lib.GA_ERR_ARG),
    (dict(num_pages=0), _lib.GA_ERR_ARG), (dict(num_pages=-1), _lib.GA_ERR_ARG),
    (dict(kv_heads=0), _lib.GA_ERR_ARG), (dict(head_dim=80), _lib.GA_ERR_SHAPE),
    (dict(page_size=48), _lib.GA_ERR_SHAPE), (dict(stride_page=8704), _lib.GA_ERR_ARG),
    (dict(stride_page=2 * 8704 + 8), _lib.GA_ERR_ARG)])
def test_caches_that_are_refused(change, status):
    l = _lib.lib()
    c, a, e = cache(**change), attention(), _lib.Mx4EvictArgs()
    r = ctypes.byref
    need = ctypes.c_size_t(7)
    assert l.ga_mx4_append(r(c), 0x1000, 0x1000, 0, 1, 256, 128, 256, 128, 0x1000, 0, None) == status
    assert l.ga_mx4_read(r(c), 0x1000, 1, 0x1000, 0x1000, 0, None) == status
    assert l.ga_mx4_attention(r(c), r(a), None, 0, None) == status
    assert l.ga_mx4_attention_workspace_bytes(r(c), r(a), r(need)) == status
    assert l.ga_mx4_attention_weights(r(c), r(a), None, 0, 0, 0x1000, 8, 8, 8, None, 0, None) == status
    assert l.ga_mx4_evict(r(c), r(e), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(q=None), _lib.GA_ERR_ARG), (dict(lens=None), _lib.GA_ERR_ARG),
    (dict(table=None), _lib.GA_ERR_ARG), (dict(seqs=-1), _lib.GA_ERR_ARG),
    (dict(rows=-1), _lib.GA_ERR_ARG), (dict(heads=0), _lib.GA_ERR_ARG),
    (dict(heads=3), _lib.GA_ERR_SHAPE), (dict(rows=4), _lib.GA_ERR_SHAPE),
    (dict(window=-1), _lib.GA_ERR_ARG), (dict(window=3, causal=0), _lib.GA_ERR_ARG),
    (dict(softcap=-1.0), _lib.GA_ERR_ARG), (dict(softcap=float("nan")), _lib.GA_ERR_ARG),
    (dict(q=0x10004), _lib.GA_ERR_SHAPE), (dict(stride_q_row=516), _lib.GA_ERR_SHAPE),
    (dict(stride_q_head=129), _lib.GA_ERR_SHAPE), (dict(max_len=-1), _lib.GA_ERR_ARG),
    (dict(max_q=-1), _lib.GA_ERR_ARG), (dict(table_pages=-1), _lib.GA_ERR_ARG)])
def test_attention_arguments_that_are_refused(change, status):
    l = _lib.lib()
    c, a = cache(), attention(**change)
    r = ctypes.byref
    assert l.ga_mx4_attention(r(c), r(a), None, 0, None) == status
    assert l.ga_mx4_attention_weights(r(c), r(a), None, 0, 0, 0x1000, 8, 8, 8, None, 0, None) == status
    assert l.ga_last_error()


def test_other_arguments_that_are_refused():
    l = _lib.lib()
    c, a = cache(), attention()
    r = ctypes.byref
    assert l.ga_mx4_attention(r(c), None, None, 0, None) == _lib.GA_ERR_ARG
    assert l.ga_mx4_attention(None, r(a), None, 0, None) == _lib.GA_ERR_ARG
    assert l.ga_mx4_attention_workspace_bytes(r(c), r(a), None) == _lib.GA_ERR_ARG
    for change in (dict(out=None), dict(out=0x10002), dict(stride_out_row=514),
                   dict(stride_out_head=4)):
        assert l.ga_mx4_attention(r(c), r(attention(**change)), None, 0, None) == _lib.GA_ERR_SHAPE
    # weights
    assert l.ga_mx4_attention_weights(r(c), r(a), None, 0, 0, None, 8, 8, 8, None, 0, None) == _lib.GA_ERR_ARG
    assert l.ga_mx4_attention_weights(r(c), r(a), None, 0, 0, 0x1000, 8, 8, -1,
                                      None, 0, None) == _lib.GA_ERR_ARG
    assert l.ga_mx4_attention_weights(r(c), r(attention(lse=None)), None, 0, 0, 0x1000, 8, 8, 8,
                                      None, 0, None) == _lib.GA_ERR_ARG
    assert l.ga_mx4_attention_weights_workspace_bytes(r(c), r(a), 8, None) == _lib.GA_ERR_ARG
    assert l.ga_mx4_attention_weights_workspace_bytes(r(c), r(a), -1, ctypes.byref(
        ctypes.c_size_t())) == _lib.GA_ERR_ARG
    # append and read
    ok = [r(c), 0x1000, 0x1000, 0, 1, 256, 128, 256, 128, 0x1000, 0, None]
    for at, bad, status in ((1, None, 1), (2, None, 1), (9, None, 1), (3, 2, 1), (4, -1, 1),
                            (10, 3, 1), (10, -1, 1), (1, 0x1008, 2), (5, 258, 2), (8, 130, 2)):
        x = list(ok)
        x[at] = bad
        assert l.ga_mx4_append(*x) == status, (at, bad)
    ok = [r(c), 0x1000, 1, 0x1000, 0x1000, 0, None]
    for at, bad, status in ((1, None, 1), (2, -1, 1), (3, None, 1), (4, 0x1008, 1), (5, 2, 1)):
        x = list(ok)
        x[at] = bad
        assert l.ga_mx4_read(*x) == status, (at, bad)
    big = cache(kv_heads=1 << 20, stride_page=(1 << 20) * 8704)
    assert l.ga_mx4_append(r(big), 0x1000, 0x1000, 0, 1 << 20, 256, 128, 256, 128, 0x1000, 0,
                           None) == _lib.GA_ERR_SHAPE
    assert l.ga_mx4_read(r(big), 0x1000, 1 << 20, 0x1000, 0x1000, 0, None) == _lib.GA_ERR_SHAPE


def test_evictions_that_are_refused():
    l = _lib.lib()
    c = cache()

    def evict(**kw):
        e = _lib.Mx4EvictArgs()
        for n in ("table", "lens", "dst_table", "weights", "kept", "new_lens", "new_weights"):
            setattr(e, n, 0x10000)
        e.seqs, e.table_pages, e.dst_pages, e.width, e.new_width, e.keep, e.recent = 2, 4, 2, 200, \
            100, 100, 10
        for k, v in kw.items():
            setattr(e, k, v)
        return l.ga_mx4_evict(ctypes.byref(c), ctypes.byref(e), None)

    assert l.ga_mx4_evict(ctypes.byref(c), None, None) == _lib.GA_ERR_ARG
    for n in ("table", "lens", "dst_table", "weights", "kept", "new_lens", "new_weights"):
        assert evict(**{n: None}) == _lib.GA_ERR_ARG
    for kw in (dict(keep=0), dict(keep=-4), dict(recent=-1), dict(recent=101), dict(seqs=-1),
               dict(width=-1), dict(new_width=99), dict(table_pages=-1), dict(dst_pages=-1)):
        assert evict(**kw) == _lib.GA_ERR_ARG
    assert evict(dst_pages=1) == _lib.GA_ERR_SHAPE


def test_nothing_to_do_is_no_error():
    l = _lib.lib()
    c = cache()
    r = ctypes.byref
    need = ctypes.c_size_t(7)
    assert l.ga_mx4_append(r(c), None, None, 0, 0, 256, 128, 256, 128, None, 0, None) == 0
    assert l.ga_mx4_read(r(c), None, 0, None, None, 0, None) == 0
    for kw in (dict(seqs=0, rows=0), dict(rows=0, q_starts=0x1000)):
        assert l.ga_mx4_attention(r(c), r(attention(q=None, **kw)), None, 0, None) == 0
        assert l.ga_mx4_attention_workspace_bytes(r(c), r(attention(**kw)), r(need)) == 0
        assert need.value == 0
    assert l.ga_mx4_attention_weights(r(c), r(attention()), None, 0, 0, None, 8, 8, 0, None, 0, None) == 0

"""A key/value cache in MXFP4 and what reads it, on torch tensors.

A cache is a uint8 tensor [pages, kv heads, page bytes] (new_cache); a page
holds page_size tokens (16, 32, 64, 128 or 256) of every kv head, as e2m1 codes
with one E8M0 scale per 32 elements: 4.25 bits an element, the format of
ops.quant_mxfp4 in the layout that include/gcnasm_amd.h gives. Head sizes are
64, 128 and 256. The pages of a sequence stand in a row of an int32 table
[sequences, pages]; token t lies in slot table[b, t // page_size] * page_size +
t % page_size. Which pages a sequence has, and its length, is the caller's
business.

  append             quantises keys and values into slots
  read               the values that slots hold
  attention          rows of this step over the cached tokens: prompts, pieces of
                     prompts, single tokens; grouped heads, sliding window, capped scores
  attention_weights  what those rows have given to each token, added up
  evict              keeps the latest tokens and those with the most weight

Nothing here waits for the GPU; the checks are of what the host knows (types,
shapes, strides). Page numbers, lengths and slots stay on the GPU and are kept
inside the operands by the kernels. Results and scratch are allocated on the
stream that the call runs on.
"""
import contextlib
import ctypes
import math

import torch

from . import _lib
from ._lib import check, lib
from .f4gemm import _stream_handle


def page_bytes(page_size, head_dim):
    """Bytes of one kv head's page."""
    n = lib().ga_mx4_page_bytes(page_size, head_dim)
    if not n:
        raise ValueError("no page of %r tokens with head size %r" % (page_size, head_dim))
    return n


def new_cache(num_pages, kv_heads, head_dim, page_size=64, device="cuda"):
    """An empty cache: uint8 [num_pages, kv_heads, page bytes]. What it holds
    before the first append is never read as a token."""
    return torch.zeros((num_pages, kv_heads, page_bytes(page_size, head_dim)), dtype=torch.uint8,
                       device=device)


def _cache(cache, head_dim):
    if cache.dtype != torch.uint8 or cache.dim() != 3:
        raise TypeError("a cache is a uint8 tensor [pages, kv heads, page bytes]")
    pages, heads, size = cache.shape
    page = size * 16 // (17 * head_dim) if head_dim > 0 else 0
    if size == 0 or lib().ga_mx4_page_bytes(page, head_dim) != size:
        raise ValueError("pages of %d bytes hold no tokens of head size %d" % (size, head_dim))
    if cache.stride(2) != 1 or (heads > 1 and cache.stride(1) != size):
        raise ValueError("the heads of a page must be contiguous (strides %s)"
                         % (tuple(cache.stride()),))
    _on_device(cache, "cache")
    stride = cache.stride(0) if pages > 1 else heads * size
    return _lib.Mx4Cache(cache.data_ptr(), pages, stride, heads, head_dim, page)


def _on_device(x, what, like=None):
    if x.device.type != "cuda":
        raise ValueError("%s must be on the GPU" % what)
    index = torch.cuda.current_device() if like is None else like.device.index
    if x.device.index != index:
        raise ValueError("%s is on %s, not on the device of the call (cuda:%d)"
                         % (what, x.device, index))


def _whole(x, what, dtype, shape, cache):
    """Checks a tensor of whole numbers whose last dimension is contiguous."""
    if x.dtype != dtype:
        raise TypeError("%s must be %s" % (what, dtype))
    if tuple(x.shape) != tuple(shape):
        raise ValueError("%s must be %s, is %s" % (what, tuple(shape), tuple(x.shape)))
    if x.numel() > 1 and x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError("%s must be contiguous along its last dimension" % what)
    _on_device(x, what, cache)


def _inner(x, what):
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError("%s must be contiguous along its last dimension (strides %s)"
                         % (what, tuple(x.stride())))


def _on(stream):
    """Allocations belong to the stream that the call runs on."""
    if stream is None:
        return contextlib.nullcontext()
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream)
    return torch.cuda.stream(stream)


def append(cache, k, v, slots, scale_rule=_lib.GA_MX_SCALE_FLOOR_448, stream=None):
    """Quantises k, v [tokens, kv heads, D] (float32 or bfloat16, any row and head
    strides that are multiples of 4) into slots, int64 [tokens]. A slot outside the
    cache, such as -1, writes nothing; the others have to differ. The rules are
    those of ops.quant_mxfp4."""
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k and v must be [tokens, kv heads, D] of one type (%s %s, %s %s)"
                         % (tuple(k.shape), k.dtype, tuple(v.shape), v.dtype))
    if k.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("k and v must be float32 or bfloat16")
    tokens, heads, dim = k.shape
    c = _cache(cache, dim)
    if heads != c.kv_heads:
        raise ValueError("k has %d heads, the cache %d" % (heads, c.kv_heads))
    _whole(slots, "slots", torch.int64, (tokens,), cache)
    for x, what in ((k, "k"), (v, "v")):
        _inner(x, what)
        _on_device(x, what, cache)
    kind = _lib.GA_IN_F32 if k.dtype == torch.float32 else _lib.GA_IN_BF16
    check(lib().ga_mx4_append(ctypes.byref(c), k.data_ptr(), v.data_ptr(), kind, tokens,
                              k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                              slots.data_ptr(), scale_rule, _stream_handle(stream)))


def read(cache, slots, head_dim, dtype=torch.bfloat16, stream=None):
    """Keys and values [tokens, kv heads, D] that slots (int64 [tokens]) hold, bfloat16
    or float32 (both hold them exactly); zeros for a slot outside the cache."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("dtype must be float32 or bfloat16")
    c = _cache(cache, head_dim)
    _whole(slots, "slots", torch.int64, (slots.numel(),), cache)
    with _on(stream):
        k = torch.empty((slots.numel(), c.kv_heads, head_dim), dtype=dtype, device=cache.device)
        v = torch.empty_like(k)
    kind = _lib.GA_DTYPE_F32 if dtype == torch.float32 else _lib.GA_DTYPE_BF16
    check(lib().ga_mx4_read(ctypes.byref(c), slots.data_ptr(), slots.numel(), k.data_ptr(),
                            v.data_ptr(), kind, _stream_handle(stream)))
    return k, v


def _args(q, cache, table, lens, q_starts, max_q, max_len, scale, causal, window, softcap):
    if q.dim() != 3 or q.dtype != torch.bfloat16:
        raise TypeError("q must be bfloat16 [rows, heads, D]")
    rows, heads, dim = q.shape
    c = _cache(cache, dim)
    seqs = lens.shape[0] if lens.dim() == 1 else -1
    _whole(lens, "lens", torch.int32, (seqs,), cache)
    if table.dim() != 2:
        raise ValueError("table must be [sequences, pages]")
    _whole(table, "table", torch.int32, (seqs, table.shape[1]), cache)
    if q_starts is not None:
        _whole(q_starts, "q_starts", torch.int32, (seqs + 1,), cache)
    _inner(q, "q")
    _on_device(q, "q", cache)
    a = _lib.Mx4AttentionArgs()
    a.q = q.data_ptr()
    a.table, a.lens = table.data_ptr(), lens.data_ptr()
    a.q_starts = None if q_starts is None else q_starts.data_ptr()
    a.stride_q_row, a.stride_q_head = q.stride(0), q.stride(1)
    a.stride_table = table.stride(0)
    a.seqs, a.rows, a.heads, a.table_pages = seqs, rows, heads, table.shape[1]
    a.max_q = rows if max_q is None else max_q
    full = table.shape[1] * c.page_size
    a.max_len = min(full, 0x7FFFFFFF) if max_len is None else max_len
    a.causal, a.window = int(bool(causal)), window
    a.scale = 1.0 / math.sqrt(dim) if scale is None else scale
    a.softcap = softcap
    return c, a


def attention(q, cache, table, lens, q_starts=None, max_q=None, max_len=None, scale=None,
              causal=True, window=0, softcap=0.0, out=None, lse=None, workspace=None, stream=None):
    """softmax(scale q k^T) v of the rows q [rows, heads, D] (bfloat16) over the
    cached tokens of their sequences -> (out [rows, heads, D] bfloat16, lse [rows,
    heads] float32, the natural logarithm of the sum of exponentials).

    table int32 [sequences, pages], lens int32 [sequences]: the tokens of each
    sequence, this step's among them (append them first). q_starts int32 [sequences +
    1]: the first row of each sequence, the last entry the number of rows; None: one row
    for each sequence. Row i of a sequence's n stands at position len - n + i and
    sees, if causal, the tokens up to it, of these the last `window` if window is
    not 0. softcap c > 0: scores c tanh(s / c). A row that sees nothing
    gets zeros and lse -inf. heads is a multiple of the cache's kv heads.

    max_q and max_len bound the rows and tokens of a sequence on the host; they
    choose the launch and may be larger than what the tensors hold (default: all
    rows, all of the table). workspace: a tensor of at least
    attention_workspace_bytes, for callers that keep one."""
    c, a = _args(q, cache, table, lens, q_starts, max_q, max_len, scale, causal, window, softcap)
    return _attention(c, a, q, out, lse, workspace, stream)


def _attention(c, a, q, out, lse, workspace, stream):
    l = lib()
    need = ctypes.c_size_t(0)
    check(l.ga_mx4_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(a), ctypes.byref(need)))
    with _on(stream):
        if out is None:
            out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        if lse is None:
            lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        if workspace is None and need.value:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device)
    if out.dtype != torch.bfloat16 or out.shape != q.shape:
        raise ValueError("out must be bfloat16 %s" % (tuple(q.shape),))
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2]:
        raise ValueError("lse must be float32 %s" % (tuple(q.shape[:2]),))
    for x, what in ((out, "out"), (lse, "lse")):
        _inner(x, what)
        _on_device(x, what, q)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    a.stride_out_row, a.stride_out_head = out.stride(0), out.stride(1)
    a.stride_lse_row = lse.stride(0)
    ptr, size = None, 0
    if workspace is not None:
        _on_device(workspace, "workspace", q)
        ptr, size = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    check(l.ga_mx4_attention(ctypes.byref(c), ctypes.byref(a), ptr, size, _stream_handle(stream)))
    return out, lse


def attention_workspace_bytes(q, cache, table, lens, q_starts=None, max_q=None, max_len=None,
                              causal=True, window=0):
    """Bytes of scratch that attention() takes for these sizes."""
    c, a = _args(q, cache, table, lens, q_starts, max_q, max_len, None, causal, window, 0.0)
    need = ctypes.c_size_t(0)
    check(lib().ga_mx4_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(a),
                                                 ctypes.byref(need)))
    return need.value


def _weights(x, what, seqs, heads, cache):
    if x.dtype != torch.float32 or x.dim() != 3 or tuple(x.shape[:2]) != (seqs, heads):
        raise ValueError("%s must be float32 [%d, %d, tokens]" % (what, seqs, heads))
    _inner(x, what)
    _on_device(x, what, cache)


def attention_weights(q, cache, table, lens, lse, weights=None, q_starts=None, max_q=None,
                      max_len=None, scale=None, causal=True, window=0, softcap=0.0, width=None,
                      out=None, stream=None):
    """weights [sequences, kv heads, tokens] float32 (None: zeros) plus what the rows
    q give to each cached token: the sum of exp(score - lse) over the rows that see it
    and the query heads of the kv head. q, lse and the rest as of the attention()
    call. -> out, float32 [sequences, kv heads, width] (width: weights', or
    max_len), zeros from a sequence's length on; out may be weights."""
    c, a = _args(q, cache, table, lens, q_starts, max_q, max_len, scale, causal, window, softcap)
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2]:
        raise ValueError("lse must be float32 %s" % (tuple(q.shape[:2]),))
    _inner(lse, "lse")
    _on_device(lse, "lse", cache)
    a.lse, a.stride_lse_row = lse.data_ptr(), lse.stride(0)
    if weights is not None:
        _weights(weights, "weights", a.seqs, c.kv_heads, cache)
    if out is None:
        if width is None:
            width = a.max_len if weights is None else weights.shape[2]
        with _on(stream):
            out = torch.empty((a.seqs, c.kv_heads, width), dtype=torch.float32,
                              device=cache.device)
    _weights(out, "out", a.seqs, c.kv_heads, cache)
    if weights is not None and weights.shape[2] < out.shape[2]:
        raise ValueError("weights hold %d tokens, out %d" % (weights.shape[2], out.shape[2]))
    w, sw = (None, (0, 0)) if weights is None else (weights.data_ptr(), weights.stride())
    check(lib().ga_mx4_attention_weights(ctypes.byref(c), ctypes.byref(a), w, sw[0], sw[1],
                                         out.data_ptr(), out.stride(0), out.stride(1),
                                         out.shape[2], _stream_handle(stream)))
    return out


def evict(cache, table, lens, weights, keep, recent, dst_table, head_dim, new_weights=None,
          stream=None):
    """Keeps, of each sequence and kv head, the last `recent` tokens and of the
    others the keep - recent with the most weight (equal ones: the lowest index
    first), moved in their order to the pages of dst_table, int32 [sequences, at least
    keep / page_size pages]; a sequence of at most `keep` tokens is moved whole.

    -> (kept int32 [sequences, kv heads, keep], -1 behind a shorter sequence;
    new_lens int32 [sequences]; new_weights float32 [sequences, kv heads, keep, or
    the width of the new_weights given], zeros behind). The pages of dst_table must
    be pages that no table holds for tokens in use; those of `table` are free
    for others once the call has run on its stream."""
    c = _cache(cache, head_dim)
    seqs = lens.shape[0] if lens.dim() == 1 else -1
    _whole(lens, "lens", torch.int32, (seqs,), cache)
    for x, what in ((table, "table"), (dst_table, "dst_table")):
        if x.dim() != 2:
            raise ValueError("%s must be [sequences, pages]" % what)
        _whole(x, what, torch.int32, (seqs, x.shape[1]), cache)
    _weights(weights, "weights", seqs, c.kv_heads, cache)
    if keep <= 0 or not 0 <= recent <= keep:
        raise ValueError("keep must be positive and recent 0 .. keep")
    with _on(stream):
        kept = torch.empty((seqs, c.kv_heads, keep), dtype=torch.int32, device=cache.device)
        new_lens = torch.empty_like(lens)
        if new_weights is None:
            new_weights = torch.empty((seqs, c.kv_heads, keep), dtype=torch.float32,
                                      device=cache.device)
    _weights(new_weights, "new_weights", seqs, c.kv_heads, cache)
    a = _lib.Mx4EvictArgs()
    a.table, a.lens, a.dst_table = table.data_ptr(), lens.data_ptr(), dst_table.data_ptr()
    a.weights, a.kept = weights.data_ptr(), kept.data_ptr()
    a.new_lens, a.new_weights = new_lens.data_ptr(), new_weights.data_ptr()
    a.stride_table, a.stride_dst_table = table.stride(0), dst_table.stride(0)
    a.stride_w_seq, a.stride_w_head = weights.stride(0), weights.stride(1)
    a.stride_new_seq, a.stride_new_head = new_weights.stride(0), new_weights.stride(1)
    a.seqs, a.table_pages, a.dst_pages = seqs, table.shape[1], dst_table.shape[1]
    a.width, a.new_width = weights.shape[2], new_weights.shape[2]
    a.keep, a.recent = keep, recent
    check(lib().ga_mx4_evict(ctypes.byref(c), ctypes.byref(a), _stream_handle(stream)))
    return kept, new_lens, new_weights

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

import torch

from . import _lib
from ._lib import check, lib
from .f4gemm import _stream_handle


# (page bytes, head size) -> tokens of a page, for every page there is
_PAGE_SIZES = {(p * d * 17 // 16, d): p for p in (16, 32, 64, 128, 256) for d in (64, 128, 256)}


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


# The checks below run on every call, of which a decode step makes several for each
# layer: they ask a tensor for as little as they can. The current device and its stream come
# from torch's own functions beneath the public ones where this version has them (0.1 us each
# instead of 0.3).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream, device):
    if stream is None and _current_stream is not None:
        return _current_stream(device)
    return _stream_handle(stream)


def _cache(cache, head_dim):
    if cache.dtype is not torch.uint8 or cache.dim() != 3:
        raise TypeError("a cache is a uint8 tensor [pages, kv heads, page bytes]")
    pages, heads, size = cache.shape
    page = _PAGE_SIZES.get((size, head_dim))
    if page is None:
        raise ValueError("pages of %d bytes hold no tokens of head size %d" % (size, head_dim))
    stride, head_stride, inner = cache.stride()
    if inner != 1 or (heads > 1 and head_stride != size):
        raise ValueError("the heads of a page must be contiguous (strides %s)"
                         % (tuple(cache.stride()),))
    device = cache.get_device()
    if device < 0 or device != _current_device():
        raise ValueError("the cache is on %s, not on the current GPU" % cache.device)
    return _lib.Mx4Cache(cache.data_ptr(), pages, stride if pages > 1 else heads * size, heads,
                         head_dim, page), device


def _check(x, what, dtype, shape, device):
    """Checks type, shape and place of a tensor whose last dimension is contiguous, and
    returns its strides."""
    if x.dtype is not dtype:
        raise TypeError("%s must be %s, is %s" % (what, dtype, x.dtype))
    if x.shape != shape:
        raise ValueError("%s must be %s, is %s" % (what, tuple(shape), tuple(x.shape)))
    strides = x.stride()
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError("%s must be contiguous along its last dimension (strides %s)"
                         % (what, tuple(strides)))
    if x.get_device() != device:
        raise ValueError("%s is on %s, not on the cache's GPU" % (what, x.device))
    return strides


def _scratch(workspace, device):
    if workspace is None:
        return None, 0
    if workspace.get_device() != device or not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous on the cache's GPU")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


_HERE = contextlib.nullcontext()


def _on(stream):
    """Allocations belong to the stream that the call runs on."""
    if stream is None:
        return _HERE
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream)
    return torch.cuda.stream(stream)


_IN_TYPES = {torch.float32: _lib.GA_IN_F32, torch.bfloat16: _lib.GA_IN_BF16}
_OUT_TYPES = {torch.float32: _lib.GA_DTYPE_F32, torch.bfloat16: _lib.GA_DTYPE_BF16}


def append(cache, k, v, slots, scale_rule=_lib.GA_MX_SCALE_FLOOR_448, stream=None):
    """Quantises k, v [tokens, kv heads, D] (float32 or bfloat16, any row and head
    strides that are multiples of 4) into slots, int64 [tokens]. A slot outside the
    cache, such as -1, writes nothing; the others have to differ. The rules are
    those of ops.quant_mxfp4; the default is that of the library's products, which
    cuts a block's largest values by up to half. GA_MX_SCALE_OCP loses less: of
    normally distributed values 0.115 of their root mean square instead of 0.20, of an
    attention output over such a cache 0.19 instead of 0.34 (4096 tokens, D = 128, keys
    with strong channels)."""
    if k.dim() != 3:
        raise ValueError("k must be [tokens, kv heads, D], is %s" % (tuple(k.shape),))
    kind = _IN_TYPES.get(k.dtype)
    if kind is None:
        raise TypeError("k and v must be float32 or bfloat16")
    tokens, heads, dim = shape = k.shape
    c, device = _cache(cache, dim)
    if heads != c.kv_heads:
        raise ValueError("k has %d heads, the cache %d" % (heads, c.kv_heads))
    _check(slots, "slots", torch.int64, (tokens,), device)
    sk = _check(k, "k", k.dtype, shape, device)
    sv = _check(v, "v", k.dtype, shape, device)
    # the stride of a dimension of one element can be anything
    if tokens == 1:
        sk, sv = (0, sk[1]), (0, sv[1])
    if heads == 1:
        sk, sv = (sk[0], 0), (sv[0], 0)
    check(lib().ga_mx4_append(c, k.data_ptr(), v.data_ptr(), kind, tokens, sk[0], sk[1], sv[0],
                              sv[1], slots.data_ptr(), scale_rule, _stream(stream, device)))


def read(cache, slots, head_dim, dtype=torch.bfloat16, stream=None):
    """Keys and values [tokens, kv heads, D] that slots (int64 [tokens]) hold, bfloat16
    or float32 (both hold them exactly); zeros for a slot outside the cache."""
    kind = _OUT_TYPES.get(dtype)
    if kind is None:
        raise TypeError("dtype must be float32 or bfloat16")
    c, device = _cache(cache, head_dim)
    tokens = slots.numel()
    _check(slots, "slots", torch.int64, (tokens,), device)
    with _on(stream):
        k = cache.new_empty((tokens, c.kv_heads, head_dim), dtype=dtype)
        v = torch.empty_like(k)
    check(lib().ga_mx4_read(c, slots.data_ptr(), tokens, k.data_ptr(), v.data_ptr(), kind,
                            _stream(stream, device)))
    return k, v


_INT_MAX = 0x7FFFFFFF


def _args(q, cache, table, lens, q_starts, max_q, max_len, scale, causal, window, softcap):
    if q.dim() != 3:
        raise ValueError("q must be [rows, heads, D], is %s" % (tuple(q.shape),))
    rows, heads, dim = q.shape
    c, device = _cache(cache, dim)
    sq = _check(q, "q", torch.bfloat16, q.shape, device)
    if lens.dim() != 1 or table.dim() != 2:
        raise ValueError("lens must be [sequences], table [sequences, pages]")
    seqs, pages = lens.shape[0], table.shape[1]
    _check(lens, "lens", torch.int32, (seqs,), device)
    st = _check(table, "table", torch.int32, (seqs, pages), device)
    starts = None
    if q_starts is not None:
        _check(q_starts, "q_starts", torch.int32, (seqs + 1,), device)
        starts = q_starts.data_ptr()
    # what passes an int is more than any sequence has; ctypes would take its low 32 bits
    if max_q is None or max_q > _INT_MAX:
        max_q = rows
    if max_len is None or max_len > _INT_MAX:
        max_len = min(pages * c.page_size, _INT_MAX)
    if window > _INT_MAX:
        window = _INT_MAX
    return c, device, _lib.Mx4AttentionArgs(
        q.data_ptr(), None, None, table.data_ptr(), lens.data_ptr(), starts,
        sq[0] if rows > 1 else 0, sq[1] if heads > 1 else 0, 0, 0, 0,
        st[0], seqs, rows, heads, pages, max_q, max_len,
        1 if causal else 0, window, dim ** -0.5 if scale is None else scale, softcap)


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
    gets zeros and lse -inf. heads is a multiple of the cache's kv heads. Positions are
    places in the cache: after evict() a window counts the tokens that were kept.

    With more than 64 rows of a kv head in a sequence the probabilities p enter the sum of
    the values as bf16 (those over a 16th of a running sum with 16 bits): out is off by up
    to 2^-8 of sum p |v - out| besides its own rounding, in all 1.1 to 1.4 times that
    rounding for random values. With fewer rows all have 16 bits.

    max_q and max_len bound the rows and tokens of a sequence on the host; they
    choose the launch and may be larger than what the tensors hold (default: all
    rows, all of the table). workspace: a tensor of at least
    attention_workspace_bytes, for callers that keep one."""
    c, device, a = _args(q, cache, table, lens, q_starts, max_q, max_len, scale, causal, window,
                         softcap)
    need = ctypes.c_size_t(0)
    check(lib().ga_mx4_attention_workspace_bytes(c, a, need))
    heads, dim = a.heads, c.head_dim
    so, sl = (heads * dim, dim), (heads,)
    if out is not None:
        so = _check(out, "out", torch.bfloat16, q.shape, device)
        so = so[0] if a.rows > 1 else 0, so[1] if heads > 1 else 0
    if lse is not None:
        sl = _check(lse, "lse", torch.float32, q.shape[:2], device)
    with _on(stream):
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if lse is None:
            lse = q.new_empty((a.rows, heads), dtype=torch.float32)
        if workspace is None and need.value:
            workspace = q.new_empty(need.value, dtype=torch.uint8)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    a.stride_out_row, a.stride_out_head, a.stride_lse_row = so[0], so[1], sl[0]
    ptr, size = _scratch(workspace, device)
    check(lib().ga_mx4_attention(c, a, ptr, size, _stream(stream, device)))
    return out, lse


def attention_workspace_bytes(q, cache, table, lens, q_starts=None, max_q=None, max_len=None,
                              causal=True, window=0):
    """Bytes of scratch that attention() takes for these sizes."""
    c, _, a = _args(q, cache, table, lens, q_starts, max_q, max_len, None, causal, window, 0.0)
    need = ctypes.c_size_t(0)
    check(lib().ga_mx4_attention_workspace_bytes(c, a, need))
    return need.value


def _weights(x, what, seqs, heads, device):
    if x.dim() != 3:
        raise ValueError("%s must be [%d, %d, tokens]" % (what, seqs, heads))
    return _check(x, what, torch.float32, (seqs, heads, x.shape[2]), device)


def attention_weights(q, cache, table, lens, lse, weights=None, q_starts=None, max_q=None,
                      max_len=None, scale=None, causal=True, window=0, softcap=0.0, width=None,
                      out=None, workspace=None, stream=None):
    """weights [sequences, kv heads, tokens] float32 (None: zeros) plus what the rows
    q give to each cached token: the sum of exp(score - lse) over the rows that see it
    and the query heads of the kv head. q, lse and the rest as of the attention()
    call. -> out, float32 [sequences, kv heads, width] (width: weights', or
    max_len), zeros from a sequence's length on; out may be weights. workspace: a tensor of
    at least attention_weights_workspace_bytes."""
    c, device, a = _args(q, cache, table, lens, q_starts, max_q, max_len, scale, causal, window,
                         softcap)
    a.stride_lse_row = _check(lse, "lse", torch.float32, q.shape[:2], device)[0]
    a.lse = lse.data_ptr()
    ptr, sw = None, (0, 0)
    if weights is not None:
        sw = _weights(weights, "weights", a.seqs, c.kv_heads, device)
        ptr = weights.data_ptr()
    if width is None:
        width = a.max_len if weights is None else weights.shape[2]
    if out is not None:
        width = out.shape[-1]
    if width > _INT_MAX:
        raise ValueError("width %d is more than a call takes" % width)
    if weights is not None and weights.shape[2] < width:
        raise ValueError("weights hold %d tokens, out %d" % (weights.shape[2], width))
    need = ctypes.c_size_t(0)
    check(lib().ga_mx4_attention_weights_workspace_bytes(c, a, width, need))
    so = (c.kv_heads * width, width)
    if out is not None:
        so = _weights(out, "out", a.seqs, c.kv_heads, device)
    with _on(stream):
        if out is None:
            out = q.new_empty((a.seqs, c.kv_heads, width), dtype=torch.float32)
        if workspace is None and need.value:
            workspace = q.new_empty(need.value, dtype=torch.uint8)
    ws, size = _scratch(workspace, device)
    check(lib().ga_mx4_attention_weights(c, a, ptr, sw[0], sw[1], out.data_ptr(), so[0], so[1],
                                         width, ws, size, _stream(stream, device)))
    return out


def attention_weights_workspace_bytes(q, cache, table, lens, width, q_starts=None, max_q=None,
                                      max_len=None, causal=True, window=0):
    """Bytes of scratch that attention_weights() takes for these sizes; width as its out has it."""
    c, _, a = _args(q, cache, table, lens, q_starts, max_q, max_len, None, causal, window, 0.0)
    if width > _INT_MAX:
        raise ValueError("width %d is more than a call takes" % width)
    need = ctypes.c_size_t(0)
    check(lib().ga_mx4_attention_weights_workspace_bytes(c, a, width, need))
    return need.value


def evict(cache, table, lens, weights, keep, recent, dst_table, head_dim, new_weights=None,
          stream=None, kept=None, new_lens=None):
    """Keeps, of each sequence and kv head, the last `recent` tokens and of the
    others the keep - recent with the most weight (equal ones: the lowest index
    first), moved in their order to the pages of dst_table, int32 [sequences, at least
    keep / page_size pages]; a sequence of at most `keep` tokens is moved whole.

    -> (kept int32 [sequences, kv heads, keep], -1 behind a shorter sequence;
    new_lens int32 [sequences]; new_weights float32 [sequences, kv heads, keep, or
    the width of the new_weights given], zeros behind). weights hold every length. A window of
    later attention counts kept tokens, not positions in the text. kept (contiguous), new_lens and
    new_weights can be given to write to. The pages of dst_table must
    be pages that no table holds for tokens in use; those of `table` are free
    for others once the call has run on its stream."""
    c, device = _cache(cache, head_dim)
    if lens.dim() != 1 or table.dim() != 2 or dst_table.dim() != 2:
        raise ValueError("lens must be [sequences], the tables [sequences, pages]")
    seqs, pages, dst_pages = lens.shape[0], table.shape[1], dst_table.shape[1]
    _check(lens, "lens", torch.int32, (seqs,), device)
    st = _check(table, "table", torch.int32, (seqs, pages), device)
    sd = _check(dst_table, "dst_table", torch.int32, (seqs, dst_pages), device)
    sw = _weights(weights, "weights", seqs, c.kv_heads, device)
    if not 0 < keep <= _INT_MAX or not 0 <= recent <= keep:
        raise ValueError("keep must be positive (and an int) and recent 0 .. keep")
    sn, new_width = (c.kv_heads * keep, keep), keep
    if new_weights is not None:
        sn = _weights(new_weights, "new_weights", seqs, c.kv_heads, device)
        new_width = new_weights.shape[2]
    if kept is not None:
        _check(kept, "kept", torch.int32, (seqs, c.kv_heads, keep), device)
        if not kept.is_contiguous():
            raise ValueError("kept must be contiguous (strides %s)" % (tuple(kept.stride()),))
    if new_lens is not None:
        _check(new_lens, "new_lens", torch.int32, (seqs,), device)
    with _on(stream):
        if kept is None:
            kept = lens.new_empty((seqs, c.kv_heads, keep))
        if new_lens is None:
            new_lens = torch.empty_like(lens)
        if new_weights is None:
            new_weights = weights.new_empty((seqs, c.kv_heads, keep))
    a = _lib.Mx4EvictArgs(
        table.data_ptr(), lens.data_ptr(), dst_table.data_ptr(), weights.data_ptr(),
        kept.data_ptr(), new_lens.data_ptr(), new_weights.data_ptr(), st[0], sd[0], sw[0], sw[1],
        sn[0], sn[1], seqs, pages, dst_pages, weights.shape[2], new_width, keep, recent)
    check(lib().ga_mx4_evict(c, a, _stream(stream, device)))
    return kept, new_lens, new_weights

"""Layers of experts, on torch tensors: the choice of each token's experts, the
experts' products in FP8 block scale, and what lies between.

  route     a token's experts and their weights, from its logits
  arrange   the map of rows: pairs (token, choice) in the order of their experts
  product   each expert's rows times its weights (E4M3, a scale per 128 elements of a row
            and per 128 x 128 tile of the weights: ops.quant_fp8_1x128 and quant_fp8_128x128)
  activate  the gated activation between two products, quantised for the second
  combine   the weighted sum of a token's rows

A layer: ids, w = route(logits, top); starts, tokens, place = arrange(ids, experts);
h = product(*quant_fp8_1x128(x), w1, s1, starts, rows=tokens); q, s = activate(h, starts);
y = combine(product(q, s, w2, s2, starts), place, w). Of a process that has some of
the experts only (arrange's first and experts), rows behind the last expert's, from
starts[-1] on, are neither read nor written.

Nothing here waits for the GPU; the checks are of what the host knows (types,
shapes, strides). Ids, counts and row numbers stay on the GPU and are kept inside
the operands by the kernels. Results are allocated on the stream that the call runs
on. For inference: nothing here has a gradient.
"""
import torch

from . import _lib
from ._lib import check, lib
from .mx4_cache import _IN_TYPES, _OUT_TYPES, _current_device, _on, _stream

_SCORES = {"softmax": _lib.GA_EXPERTS_SOFTMAX, "sigmoid": _lib.GA_EXPERTS_SIGMOID}


_INT_MAX = 0x7FFFFFFF


# ctypes takes the low 32 bits of what passes an int: counts are checked here.
def _count(n, what, least, most):
    if not least <= n <= most:
        raise ValueError("%s must be %d .. %d, is %d" % (what, least, most, n))
    return n


# The checks below run on every call, of which a decode step makes several for each layer: they
# ask a tensor for as little as they can.
def _matrix(x, what):
    """Rows, columns, row stride and GPU of a matrix whose rows are contiguous."""
    shape, strides, device = x.shape, x.stride(), x.get_device()
    if len(shape) != 2:
        raise ValueError("%s must be a matrix, is %s" % (what, tuple(shape)))
    if shape[0] > _INT_MAX or shape[1] > _INT_MAX:
        raise ValueError("%s is more than a call takes: %s" % (what, tuple(shape)))
    if strides[1] != 1 and shape[1] > 1 and x.numel():
        raise ValueError("%s must be contiguous along its rows (strides %s)" % (what, strides))
    if device < 0 or device != _current_device():
        raise ValueError("%s is on %s, not on the current GPU" % (what, x.device))
    return shape[0], shape[1], strides[0], device


def _check(x, what, dtype, shape, device):
    """Checks type, shape and place of a tensor whose last dimension is contiguous, and
    returns its strides."""
    if x.dtype is not dtype:
        raise TypeError("%s must be %s, is %s" % (what, dtype, x.dtype))
    if x.shape != shape:
        raise ValueError("%s must be %s, is %s" % (what, tuple(shape), tuple(x.shape)))
    strides = x.stride()
    if strides[-1] != 1 and shape[-1] > 1 and x.numel():
        raise ValueError("%s must be contiguous along its last dimension (strides %s)"
                         % (what, strides))
    if x.get_device() != device:
        raise ValueError("%s is on %s, not on the current GPU" % (what, x.device))
    return strides


def _dense(x, what, dtype, shape, device):
    _check(x, what, dtype, shape, device)
    if not x.is_contiguous():
        raise ValueError("%s must be contiguous (strides %s)" % (what, x.stride()))


def route(logits, top, bias=None, scores="softmax", groups=1, top_groups=None, group_rank=1,
          renormalise=True, scale=1.0, ids=None, weights=None, stream=None):
    """The experts of each token: logits [tokens, experts] (float32 or bfloat16) ->
    (ids int32 [tokens, top], weights float32 [tokens, top]).

    scores: "softmax" over a token's logits or the "sigmoid" of each. An expert's key is
    its score + bias (float32 [experts], for the choice alone) in 64 bits, without a
    bias its logit. With top_groups (default: groups) < groups only the experts of so
    many groups (of experts / groups consecutive ones) can be chosen: those of the largest
    key (group_rank 1) or sum of the two largest (2; without a bias, of scores). The `top`
    largest keys are chosen, in their order, of equal ones the lowest index first; weights
    are their scores, divided by their sum if renormalise, times scale.

    A logit or bias of -inf or NaN takes an expert out; where fewer than `top` are left, ids
    are -1 and weights 0. At most 1024 experts, 64 choices, 64 groups. ids and weights
    (contiguous) can be given to write to."""
    kind, by = _IN_TYPES.get(logits.dtype), _SCORES.get(scores)
    if kind is None:
        raise TypeError("logits must be float32 or bfloat16")
    if by is None:
        raise ValueError('scores must be "softmax" or "sigmoid"')
    tokens, experts, stride, device = _matrix(logits, "logits")
    _count(top, "top", 1, _lib.GA_EXPERTS_MAX_TOP)
    if groups != 1:
        _count(groups, "groups", 1, _lib.GA_EXPERTS_MAX_GROUPS)
    if top_groups is None:
        top_groups = groups
    elif top_groups != groups:
        _count(top_groups, "top_groups", 1, groups)
    if group_rank != 1:
        _count(group_rank, "group_rank", 1, 2)
    ptr = None
    if bias is not None:
        _check(bias, "bias", torch.float32, (experts,), device)
        ptr = bias.data_ptr()
    if ids is not None:
        _dense(ids, "ids", torch.int32, (tokens, top), device)
    if weights is not None:
        _dense(weights, "weights", torch.float32, (tokens, top), device)
    if ids is None or weights is None:
        with _on(stream):
            if ids is None:
                ids = logits.new_empty((tokens, top), dtype=torch.int32)
            if weights is None:
                weights = logits.new_empty((tokens, top), dtype=torch.float32)
    check(lib().ga_experts_route(_lib.ExpertsRouteArgs(
        logits.data_ptr(), ptr, ids.data_ptr(), weights.data_ptr(), stride, kind, tokens, experts,
        top, by, groups, top_groups, group_rank,
        1 if renormalise else 0, scale), _stream(stream, device)))
    return ids, weights


def arrange(ids, experts, first=0, stream=None):
    """The map of rows: ids int32 [tokens, top] -> (starts int32 [experts + 1], tokens int32
    [tokens * top], place int32 [tokens, top]).

    The experts first .. first + experts - 1 are those of this call; other ids (-1 among
    them) are left out. Expert e has the sorted rows starts[e] .. starts[e + 1] - 1, in the
    order of their tokens and choices; tokens gives the token of each sorted row (-1 from
    starts[experts] on), place the row of each choice (-1 where it is left out)."""
    count, top, _, device = _matrix(ids, "ids")
    if ids.dtype is not torch.int32:
        raise TypeError("ids must be torch.int32, is %s" % ids.dtype)
    if not ids.is_contiguous():
        raise ValueError("ids must be contiguous (strides %s)" % (ids.stride(),))
    _count(experts, "experts", 1, _lib.GA_EXPERTS_MAX)
    if first:
        _count(first, "first", 0, _INT_MAX - experts)
    if count * top > _INT_MAX:
        raise ValueError("%d x %d choices are more than a call takes" % (count, top))
    with _on(stream):
        starts = ids.new_empty(experts + 1)
        tokens = ids.new_empty(count * top)
        place = torch.empty_like(ids)
    check(lib().ga_experts_arrange(ids.data_ptr(), count, top, experts, first, starts.data_ptr(),
                                   tokens.data_ptr(), place.data_ptr(), _stream(stream, device)))
    return starts, tokens, place


def product(a, sfa, b, sfb, starts, rows=None, out=None, stream=None, cut=0):
    """Each expert's rows times its weights: out[r] = a[m] b[e]^T (bfloat16), m = rows[r] or,
    without rows, r; e the expert with starts[e] <= r < starts[e + 1].

    a uint8 [A, K] E4M3 codes, sfa float32 [K / 128, A] (ops.quant_fp8_1x128); b uint8
    [experts, N, K], sfb float32 [experts, ceil(N / 128), K / 128] (ops.quant_fp8_128x128);
    starts int32 [experts + 1] and rows int32 [R] as arrange() gives them. out [R, N]
    (without rows R = A); its rows from starts[-1] on are left as they are. A row outside a
    counts as zeros. Sums are fp32, in the order of K (for few rows of an expert in up to 4
    pieces). cut: 0, or 1 .. GA_EXPERTS_CUTS for one of the ways of cutting the product in place
    of the one that its sizes choose (include/gcnasm_amd.h), for callers that tune."""
    count, k, sa, device = _matrix(a, "a")
    if a.dtype is not torch.uint8:
        raise TypeError("a must be torch.uint8, is %s" % a.dtype)
    if b.dim() != 3 or k == 0:
        raise ValueError("a must be [rows, K], b [experts, N, K]")
    experts, n = b.shape[0], b.shape[1]
    sb = _check(b, "b", torch.uint8, (experts, n, k), device)
    ssa = _check(sfa, "sfa", torch.float32, (k // 128, count), device)[0]
    ssb = _check(sfb, "sfb", torch.float32, (experts, (n + 127) // 128, k // 128), device)
    _check(starts, "starts", torch.int32, (experts + 1,), device)
    total, ptr = count, None
    if rows is not None:
        if rows.dim() != 1:
            raise ValueError("rows must be [R], is %s" % (tuple(rows.shape),))
        total = _count(rows.shape[0], "the number of rows", 0, _INT_MAX)
        _check(rows, "rows", torch.int32, (total,), device)
        ptr = rows.data_ptr()
    if out is None:
        with _on(stream):
            out = a.new_empty((total, n), dtype=torch.bfloat16)
        so = n
    else:
        so = _check(out, "out", torch.bfloat16, (total, n), device)[0]
    if cut:
        _count(cut, "cut", 0, _lib.GA_EXPERTS_CUTS)
    # the stride of a dimension of one element can be anything
    check(lib().ga_experts_product(_lib.ExpertsProductArgs(
        a.data_ptr(), sfa.data_ptr(), b.data_ptr(), sfb.data_ptr(), starts.data_ptr(), ptr,
        out.data_ptr(), count, sa if count > 1 else k, ssa if k > 128 else count,
        sb[0] if experts > 1 else 0, sb[1] if n > 1 else k, ssb[0] if experts > 1 else 0,
        ssb[1] if n > 128 else k // 128, so if total > 1 else n, experts, total, n, k, cut),
        _stream(stream, device)))
    return out


def activate(x, starts=None, stream=None):
    """The gated activation of x [rows, 2 I] (float32 or bfloat16; I a multiple of 128), its
    first half the gate g, the second u: u g / (1 + exp(-g)) in fp32, quantised as by
    ops.quant_fp8_1x128 -> (q uint8 [rows, I], scales float32 [I / 128, rows]). With starts (as
    arrange() gives them) rows from starts[-1] on are left out: theirs of q and scales
    are not written."""
    kind = _IN_TYPES.get(x.dtype)
    if kind is None:
        raise TypeError("x must be float32 or bfloat16")
    rows, both, stride, device = _matrix(x, "x")
    inner = both // 2
    if both % 256 or not both:
        raise ValueError("x must be [rows, 2 I], I a multiple of 128, is %s" % (tuple(x.shape),))
    limit = None
    if starts is not None:
        if starts.dim() != 1 or not starts.shape[0]:
            raise ValueError("starts must be [experts + 1]")
        _check(starts, "starts", torch.int32, starts.shape, device)
        limit = starts.data_ptr() + 4 * (starts.shape[0] - 1)
    with _on(stream):
        q = x.new_empty((rows, inner), dtype=torch.uint8)
        scales = x.new_empty((inner // 128, rows), dtype=torch.float32)
    check(lib().ga_experts_activate(x.data_ptr(), kind, rows, inner, stride, q.data_ptr(), inner,
                                    scales.data_ptr(), rows, limit, _stream(stream, device)))
    return q, scales


def combine(y, place, weights, dtype=torch.bfloat16, out=None, stream=None):
    """The weighted sum of each token's rows: y [rows, N] (bfloat16), place int32 and
    weights float32 [tokens, top] -> out [tokens, N] (bfloat16 or float32), out[t] the sum over j of
    weights[t, j] * y[place[t, j]] in fp32, in the order of j. A place outside y, such as -1,
    is left out."""
    rows, n, sy, device = _matrix(y, "y")
    if y.dtype is not torch.bfloat16:
        raise TypeError("y must be torch.bfloat16, is %s" % y.dtype)
    if place.dim() != 2:
        raise ValueError("place must be [tokens, top], is %s" % (tuple(place.shape),))
    tokens, top = shape = place.shape
    if tokens > _INT_MAX:
        raise ValueError("%d tokens are more than a call takes" % tokens)
    _dense(place, "place", torch.int32, shape, device)
    _dense(weights, "weights", torch.float32, shape, device)
    if out is not None:
        dtype = out.dtype
    kind = _OUT_TYPES.get(dtype)
    if kind is None:
        raise TypeError("out must be float32 or bfloat16")
    if out is None:
        with _on(stream):
            out = y.new_empty((tokens, n), dtype=dtype)
        so = n
    else:
        so = _check(out, "out", dtype, (tokens, n), device)[0]
    check(lib().ga_experts_combine(y.data_ptr(), rows, n, sy, place.data_ptr(), weights.data_ptr(),
                                   tokens, top, out.data_ptr(), kind, so, _stream(stream, device)))
    return out

"""The key/value cache in MXFP4 and what reads it, as the calls of a server.

A cache is a uint8 tensor [pages, kv heads, page bytes]; a page holds P tokens
of one kv head: e2m1 codes (two per byte, the even element in the low nibble)
and one E8M0 scale for each 32 elements of a token's key or value. In a page,
in this order:

  K codes   [P][D/2]            token by token
  V codes   [P/4][16][4][D/32]  four tokens side by side: of d = i*D/16 ..
                                (i+1)*D/16 - 1 the bytes of tokens 4q .. 4q+3
  K scales  [P][D/32]
  V scales  [P/4][D/32][4]

A table [sequences, pages of a sequence] says where a sequence's tokens lie.
The operators: append (quantise into the cache), read (back), attention (rows
of the current tokens over the cache), attention_weights (what each cached
token has been given), evict (keep the latest tokens and those with the most
weight, moved to fresh pages).

prepare() holds what a server has between calls: the cache with its pages in no
order, the tables and lengths, the rows of this step. The plain form is the
definition in elementary torch operations on padded batches, in 32 bits.
"""
import math
import types

import numpy as np
import torch

own = False

LUT = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _case(name, kind, **kw):
    c = {"name": name, "kind": kind, "seqs": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "len": 512, "rows": 1, "ragged": False, "window": 0, "softcap": 0.0, "fp32": False,
         "keep": 0, "recent": 0}
    c.update(kw)
    return c


def listed():
    return [
        # One sequence's next token after a short prompt: launches and latency.
        _case("decode_1x513", "attention", len=513),
        # A full serving batch whose sequences have any length.
        _case("decode_64x8192_ragged", "attention", seqs=64, heads=64, len=8192, ragged=True),
        # A few very long documents: reading the cache is all of it.
        _case("decode_4x131072", "attention", seqs=4, heads=64, len=131072),
        # Wide heads with capped scores and a sliding window.
        _case("decode_16x4111_d256_capped", "attention", seqs=16, heads=16, kv_heads=4, dim=256,
              len=4111, ragged=True, window=1024, softcap=50.0, page=32),
        # A whole prompt at once: bound by the matrix products.
        _case("prompt_8192", "attention", len=8192, rows=8192),
        # Pieces of prompts over what is cached already, odd sizes, narrow heads.
        _case("prompt_4x1000_over_8191_d64", "attention", seqs=4, heads=64, dim=64, len=8191,
              rows=1000, ragged=True, page=16),
        # A decode step of a server that evicts: append, attend, add up the weights.
        _case("step_32x4096_ragged", "step", seqs=32, len=4096, ragged=True),
        # A prompt's keys and values into the cache, and what the cache then holds.
        _case("write_8191", "write", len=8191, rows=8191),
        # The same from float32, narrow heads, a few tokens.
        _case("write_16x1_d64_fp32", "write", seqs=16, dim=64, len=100, rows=1, fp32=True),
        # Weights that a prompt's rows give to its tokens.
        _case("weights_2048", "weights", len=2048, rows=2048),
        # Eviction after a prompt, and of a whole batch.
        _case("evict_1x5000", "evict", len=5000, keep=1000, recent=128),
        _case("evict_16x32768", "evict", seqs=16, len=32768, ragged=True, keep=2048, recent=512),
    ]


def _log_int(rng, lo, hi):
    """An integer from lo to hi, its logarithm spread evenly; odd more often than not."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n if rng.random() < 0.3 else min(hi, n | 1)


def draw(rng):
    most = {k: max((work(c)[k] for c in listed() if c["kind"] == "attention")) for k in
            ("bytes", "flops")}
    while True:
        kind = rng.choice(["attention", "attention", "attention", "prompt", "step", "write",
                           "weights", "evict"])
        kv = rng.choice([1, 2, 4, 8])
        c = _case("", "attention" if kind == "prompt" else kind, kv_heads=kv,
                  heads=kv * rng.choice([1, 2, 4, 5, 7, 8, 16]),
                  dim=rng.choice([64, 128, 128, 256]),
                  page=rng.choice([16, 32, 64, 128, 256]), ragged=rng.random() < 0.6,
                  seqs=_log_int(rng, 1, 64), len=_log_int(rng, 1, 131072))
        if rng.random() < 0.3:
            c["window"] = _log_int(rng, 1, 4096)
        if rng.random() < 0.2:
            c["softcap"] = 30.0
        if kind == "prompt" or kind == "weights":
            c["seqs"], c["len"] = _log_int(rng, 1, 8), _log_int(rng, 2, 8192)
            c["rows"] = _log_int(rng, 2, c["len"]) if kind == "prompt" else rng.choice(
                [1, _log_int(rng, 1, c["len"])])
        elif kind == "write":
            c["rows"], c["fp32"] = min(c["len"], _log_int(rng, 1, 8192)), rng.random() < 0.5
        elif kind == "evict":
            c["seqs"], c["len"] = _log_int(rng, 1, 16), _log_int(rng, 64, 32768)
            c["keep"] = _log_int(rng, 1, min(c["len"], 4096))
            c["recent"] = rng.randint(0, c["keep"])
        del c["name"]
        w = work(c)
        tokens = c["seqs"] * c["len"] * c["kv_heads"] * c["dim"]
        if (w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and tokens <= 1 << 29 and
                c["seqs"] * c["heads"] * c["rows"] * c["len"] <= 1 << 31):
            return c


def _lengths(case):
    """Cached tokens of each sequence and its rows of this step, from the case alone."""
    n, top = case["seqs"], case["len"]
    frac = [1.0 if i == 0 or not case["ragged"] else 0.25 + 0.75 * ((i * 37 + 11) % 64) / 64
            for i in range(n)]
    lens = [max(1, int(top * f)) for f in frac]
    rows = [min(l, max(1, int(case["rows"] * f))) for l, f in zip(lens, frac)]
    return lens, rows


def _visible(case):
    """(row, token) pairs that see each other, and the cached tokens that some row sees."""
    pairs = tokens = 0
    for l, n in zip(*_lengths(case)):
        w = case["window"] or l
        # row i of n is at l - n + i and sees min(position + 1, w) tokens
        full = max(0, min(n, l - w + 1))
        short = n - full
        first = l - n + 1
        pairs += full * w + short * first + short * (short - 1) // 2
        tokens += min(l, n + w - 1)
    return pairs, tokens


def work(case):
    lens, rows = _lengths(case)
    hq, h, d = case["heads"], case["kv_heads"], case["dim"]
    code = h * d * 17 // 32  # bytes of a token's keys, or of its values
    pairs, seen = _visible(case)
    kind, total = case["kind"], sum(rows)
    attend = {"bytes": 2 * seen * code + total * hq * (4 * d + 4), "flops": 4.0 * pairs * hq * d}
    weigh = {"bytes": seen * code + total * hq * (2 * d + 4) + 8 * h * sum(lens),
             "flops": 2.0 * pairs * hq * d}
    size = 4 if case["fp32"] else 2
    if kind == "attention":
        return attend
    if kind == "weights":
        return weigh
    if kind == "write":  # input, codes written, codes read, values written
        return {"bytes": total * (2 * h * d * size + 4 * code + 4 * h * d), "flops": 0.0}
    if kind == "step":
        return {"bytes": attend["bytes"] + weigh["bytes"] + total * (4 * h * d + 2 * code),
                "flops": attend["flops"] + weigh["flops"]}
    kept = sum(min(l, case["keep"]) for l in lens)  # moved, then read back as bf16
    return {"bytes": 4 * h * sum(lens) + kept * (6 * code + 8 * h + 4 * h * d), "flops": 0.0}


# ---- the format, in elementary operations ----------------------------------------


def _codes(x):
    """Codes [..., D] and scale bytes [..., D/32] of x: the exponent is
    floor(log2(amax / 6)), values are rounded to the nearest code, ties to the
    even one, and saturate."""
    b = x.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1); 6 = 0.75 * 2^3
    e = torch.where(amax == 0, torch.full_like(e, -127), e - 3 - (m < 0.75).to(e.dtype))
    e = e.clamp(-127, 127)
    a = torch.ldexp(b.abs(), -e[..., None]).clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    r = torch.round(a / step) * step  # to even multiples: the even codes
    code = torch.where(r < 2, r * 2, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(b).to(torch.uint8) << 3)
    return code.flatten(-2), (e + 127).to(torch.uint8)


def _pairs(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _nibbles(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _pack(k, v):
    """Pages [n, h, bytes] of k, v [n, h, P, D]."""
    n, h, p, d = k.shape
    kc, ks = _codes(k)
    vc, vs = _codes(v)
    vc = _pairs(vc).view(n, h, p // 4, 4, 16, d // 32).transpose(3, 4)
    vs = vs.view(n, h, p // 4, 4, d // 32).transpose(3, 4)
    return torch.cat([t.reshape(n, h, -1) for t in (_pairs(kc), vc, ks, vs)], 2)


def _split(pages, d):
    """Views of the four parts of pages [..., bytes]."""
    p = pages.shape[-1] * 16 // (17 * d)
    kc, vc, ks, vs = pages.split([p * d // 2, p * d // 2, p * d // 32, p * d // 32], -1)
    return (kc.unflatten(-1, (p, d // 2)), vc.unflatten(-1, (p // 4, 16, 4, d // 32)),
            ks.unflatten(-1, (p, d // 32)), vs.unflatten(-1, (p // 4, d // 32, 4)))


def _values(code, scale, lut):
    x = lut[_nibbles(code).int()].unflatten(-1, (-1, 32))
    return torch.ldexp(x, scale.int()[..., None] - 127).flatten(-2)


def _unpack(pages, d, lut, keys=True, values=True):
    """Keys and values [..., P, D] in 32 bits."""
    kc, vc, ks, vs = _split(pages, d)
    k = _values(kc, ks, lut) if keys else None
    v = _values(vc.transpose(-3, -2).flatten(-2).flatten(-3, -2),
                vs.transpose(-2, -1).flatten(-3, -2), lut) if values else None
    return k, v


# ---- what a program has in hand ----------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    lens, rows = _lengths(case)
    n, hq, h, d, p = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    s = types.SimpleNamespace(case=case, dim=d, page=p, lens_list=lens, rows_list=rows)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    per = (max(lens) + p - 1) // p  # pages of a sequence
    fresh = (case["keep"] + p - 1) // p
    total = n * (per + fresh)
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    s.table = order[:n * per].view(n, per)
    s.dst_table = order[n * per:].view(n, fresh) if fresh else None
    # keys have strong channels, as after a rotary embedding; values do not
    gain = torch.exp(0.5 * normal(h, 1, d))
    if case["kind"] == "write":
        s.cache = torch.zeros((total, h, p * d * 17 // 16), dtype=torch.uint8, device=dev)
    else:
        s.cache = torch.cat([_pack(normal(m, h, p, d) * gain, normal(m, h, p, d)) for m in
                             _pieces(total, max(1, (1 << 28) // (h * p * d)))])
    s.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    s.total, s.max_q, s.max_len = starts[-1], max(rows), max(lens)
    s.q_starts = torch.tensor(starts, dtype=torch.int32, device=dev)
    # where row r of all rows lies: its sequence, and its token there
    seq = torch.repeat_interleave(torch.arange(n, device=dev),
                                  torch.tensor(rows, device=dev), output_size=s.total)
    at = torch.arange(s.total, device=dev) - s.q_starts[seq] + (s.lens - s.q_starts.diff())[seq]
    s.row_seq, s.row_at = seq, at
    s.slots = s.table[seq, at // p].long() * p + at % p
    s.q = (normal(s.total, hq, d) / gain.mean()).to(torch.bfloat16)
    kind = torch.float32 if case["fp32"] else torch.bfloat16
    if case["kind"] in ("write", "step"):
        s.k = (normal(s.total, h, d) * gain[:, 0]).to(kind)
        s.v = normal(s.total, h, d).to(kind)
    s.lut = torch.tensor(LUT, device=dev)
    if case["kind"] in ("weights", "step", "evict"):
        # weights so far: most tokens little, a few a lot
        s.weights = torch.exp(2 * normal(n, h, s.max_len) - 4)
        s.weights *= torch.arange(s.max_len, device=dev) < s.lens[:, None, None]
    if case["kind"] == "weights":
        s.lse = _attention(s)[1]
    if case["kind"] == "evict":
        j = torch.arange(case["keep"], device=dev)
        s.dst_slots = (s.dst_table[:, j // p].long() * p + j % p).reshape(-1)
    return s


def _pieces(total, most):
    full, rest = divmod(total, most)
    return [most] * full + ([rest] if rest else [])


# ---- the plain form -----------------------------------------------------------------


def _append(s):
    """Codes of k and v into the bytes of their slots."""
    n, h, d = s.k.shape
    p, size = s.page, s.cache.shape[2]
    kc, ks = _codes(s.k)
    vc, vs = _codes(s.v)
    at = (s.slots % p)[:, None, None]
    base = ((s.slots // p)[:, None] * h + torch.arange(h, device=s.k.device))[..., None] * size
    b2, b32 = torch.arange(d // 2, device=s.k.device), torch.arange(d // 32, device=s.k.device)
    where = (base + at * (d // 2) + b2,
             base + p * d // 2 + (at // 4) * (2 * d) + (b2 // (d // 32)) * (d // 8) +
             (at % 4) * (d // 32) + b2 % (d // 32),
             base + p * d + at * (d // 32) + b32,
             base + p * d + p * d // 32 + (at // 4) * (d // 8) + b32 * 4 + at % 4)
    flat = s.cache.view(-1)
    flat[torch.cat([w.reshape(-1) for w in where])] = torch.cat(
        [t.reshape(-1) for t in (_pairs(kc), _pairs(vc), ks, vs)])


def _read(s, slots):
    """Keys and values [slots, heads, D] in bfloat16 (which holds them exactly)."""
    p = s.page
    kc, vc, ks, vs = _split(s.cache, s.dim)
    page, at = slots // p, slots % p
    k = _values(kc[page, :, at], ks[page, :, at], s.lut)
    v = _values(vc[page, :, at // 4, :, at % 4].flatten(-2), vs[page, :, at // 4, :, at % 4], s.lut)
    return k.bfloat16(), v.bfloat16()


def _gathered(s, values=True):
    """Keys and values [seqs, kv heads, tokens, D] of the tables' tokens."""
    k, v = _unpack(s.cache[s.table.long()], s.dim, s.lut, values=values)
    return [None if x is None else x.transpose(1, 2).flatten(2, 3)[:, :, :s.max_len]
            for x in (k, v)]


def _scores(s, k):
    """Scores [seqs, kv heads, group * rows, tokens] of padded rows, -inf where not seen."""
    n, h = k.shape[:2]
    g = s.q.shape[1] // h
    at_row = s.q_starts[:-1, None] + torch.arange(s.max_q, device=k.device)  # [seqs, rows]
    rows = s.q_starts.diff()[:, None]
    q = s.q[at_row.clamp(max=s.total - 1).long()].float()  # [seqs, rows, heads, D]
    q = q.unflatten(2, (h, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(s.dim))
    if s.case["softcap"]:
        x = x.div_(s.case["softcap"]).tanh_().mul_(s.case["softcap"])
    i = torch.arange(s.max_q, device=k.device)
    pos = (s.lens[:, None] - rows + i)[..., None]  # [seqs, rows, 1]
    t = torch.arange(s.max_len, device=k.device)
    seen = (t <= pos) & (i[:, None] < rows[..., None])
    if s.case["window"]:
        seen &= t > pos - s.case["window"]
    x.unflatten(2, (g, s.max_q)).masked_fill_(~seen[:, None, None], -math.inf)
    return x


def _rows_of(s, x):
    """[seqs, kv heads, group * rows, ...] of padded rows back to [all rows, heads, ...]."""
    x = x.unflatten(2, (-1, s.max_q)).flatten(1, 2)
    return x[s.row_seq, :, torch.arange(s.total, device=x.device) - s.q_starts[s.row_seq]]


def _attention(s):
    k, v = _gathered(s)
    x = _scores(s, k)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    x = x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    out = torch.matmul(x, v) / torch.where(l == 0, torch.ones_like(l), l)
    return (_rows_of(s, out).to(torch.bfloat16).contiguous(),
            _rows_of(s, (m + l.log()).squeeze(-1)).contiguous())


def _attention_weights(s, lse):
    k, _ = _gathered(s, values=False)
    x = _scores(s, k)
    n, h = k.shape[:2]
    at_row = s.q_starts[:-1, None] + torch.arange(s.max_q, device=k.device)
    y = lse[at_row.clamp(max=s.total - 1).long()].unflatten(2, (h, -1))  # [seqs, rows, h, g]
    y = y.permute(0, 2, 3, 1).flatten(2)[..., None]
    w = x.sub_(y).exp_().sum(2)
    live = torch.arange(s.max_len, device=k.device) < s.lens[:, None, None]
    return torch.where(live, s.weights + w, torch.zeros_like(w))


def _evict(s):
    keep, recent = s.case["keep"], s.case["recent"]
    n, h, width = s.weights.shape
    t = torch.arange(width, device=s.lens.device)
    lens = s.lens[:, None, None]
    # the latest first, then by weight, what lies past the length last
    rank = torch.where(t >= lens - recent, math.inf, s.weights)
    rank = torch.where(t < lens, rank, -math.inf)
    first = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    new_lens = s.lens.clamp(max=keep)
    live = torch.arange(keep, device=t.device) < new_lens[:, None, None]
    kept = torch.where(live, first, torch.full_like(first, width)).sort(dim=-1).values
    kept = torch.where(live, kept, torch.full_like(kept, -1))
    weights = torch.where(live, s.weights.gather(2, kept.clamp(min=0)),
                          torch.zeros((), device=t.device))
    # the kept tokens' bytes, part by part
    p = s.page
    b = torch.arange(n, device=t.device)[:, None, None]
    head = torch.arange(h, device=t.device)[None, :, None]
    src = kept.clamp(min=0)
    sp, sa = s.table[b, src // p].long(), src % p
    j = torch.arange(keep, device=t.device)
    dp, da = s.dst_table[b, j // p].long(), (j % p).expand(n, h, keep)
    kc, vc, ks, vs = _split(s.cache, s.dim)
    kc[dp, head, da] = kc[sp, head, sa]
    ks[dp, head, da] = ks[sp, head, sa]
    vc[dp, head, da // 4, :, da % 4] = vc[sp, head, sa // 4, :, sa % 4]
    vs[dp, head, da // 4, :, da % 4] = vs[sp, head, sa // 4, :, sa % 4]
    return kept.int(), new_lens, weights


def _plain(s):
    kind = s.case["kind"]
    if kind == "attention":
        return _attention(s)
    if kind == "weights":
        return _attention_weights(s, s.lse)
    if kind == "step":
        _append(s)
        out, lse = _attention(s)
        return out, lse, _attention_weights(s, lse)
    if kind == "write":
        _append(s)
        return _read(s, s.slots)
    kept, lens, weights = _evict(s)
    return (kept, lens, weights) + _kept_values(s, lens, *_read(s, s.dst_slots))


def _kept_values(s, lens, k, v):
    """Keys and values of the kept tokens, zeros behind a sequence that is shorter."""
    if min(s.lens_list) >= s.case["keep"]:
        return k, v
    live = (torch.arange(s.case["keep"], device=k.device) < lens[:, None]).view(-1, 1, 1)
    zero = torch.zeros((), dtype=k.dtype, device=k.device)
    return torch.where(live, k, zero), torch.where(live, v, zero)


# ---- one pass -------------------------------------------------------------------------


def run(s):
    if not own:
        return _plain(s)
    from gcnasm_amd import mx4_cache as mc

    c = s.case
    kind = c["kind"]
    # a decode step of one row for each sequence needs no starts
    starts = None if s.max_q == 1 else s.q_starts
    rule = dict(q_starts=starts, max_q=s.max_q, max_len=s.max_len, window=c["window"],
                softcap=c["softcap"])
    if kind == "attention":
        return mc.attention(s.q, s.cache, s.table, s.lens, **rule)
    if kind == "weights":
        return mc.attention_weights(s.q, s.cache, s.table, s.lens, s.lse, s.weights, **rule)
    if kind == "step":
        mc.append(s.cache, s.k, s.v, s.slots)
        out, lse = mc.attention(s.q, s.cache, s.table, s.lens, **rule)
        return out, lse, mc.attention_weights(s.q, s.cache, s.table, s.lens, lse, s.weights, **rule)
    if kind == "write":
        mc.append(s.cache, s.k, s.v, s.slots)
        return mc.read(s.cache, s.slots, s.dim)
    kept, lens, weights = mc.evict(s.cache, s.table, s.lens, s.weights, c["keep"], c["recent"],
                                   s.dst_table, s.dim)
    k, v = mc.read(s.cache, s.dst_slots, s.dim)
    return (kept, lens, weights) + _kept_values(s, lens, k, v)


# ---- the definition in 64 bits ----------------------------------------------------------


def _value64(nibble, byte):
    """(-1)^sign * m * 2^x of an e2m1 code, times 2^(byte - 127)."""
    mag = (nibble & 7).double()
    x = torch.where(mag >= 2, torch.floor(mag / 2) - 1, torch.zeros_like(mag))
    m = torch.where(mag >= 2, 1 + 0.5 * torch.remainder(mag, 2), 0.5 * mag)
    sign = 1 - 2 * (nibble >> 3).double()
    return sign * m * torch.exp2(x + byte.double() - 127)


def _tokens64(s, table, t):
    """Keys and values [heads, tokens, D] of tokens t [heads or 1, tokens] of a table's row."""
    d, p = s.dim, s.page
    h, size = s.cache.shape[1:]
    e = torch.arange(d, device=t.device)
    head = torch.arange(h, device=t.device)[:, None]
    base = ((table.long()[t // p] * h + head) * size)[..., None]
    at = (t % p)[..., None]
    flat = s.cache.view(-1)

    def nibble(offset):
        return (flat[base + offset].int() >> (4 * (e % 2).int())) & 15

    quad, sub, per = at // 4, at % 4, d // 16
    k = _value64(nibble(at * (d // 2) + e // 2), flat[base + p * d + at * (d // 32) + e // 32])
    v_byte = ((quad * 16 + e // per) * 4 + sub) * (per // 2) + e % per // 2
    v = _value64(nibble(p * d // 2 + v_byte),
                 flat[base + p * d + p * d // 32 + (quad * (d // 32) + e // 32) * 4 + sub])
    return k, v


def _nearest64(x):
    """The values that the cache holds for rows x [..., D]: of each 32, the
    exponent e with 6 * 2^e <= amax < 6 * 2^(e+1), and the nearest of the
    format's values times 2^e, the one with the even code where two are."""
    b = x.double().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(amax / 6))
    e = torch.where(amax < 6 * torch.exp2(e), e - 1, e)
    e = torch.where(amax >= 12 * torch.exp2(e), e + 1, e).clamp(-127, 127)
    a = b.abs() / torch.exp2(e)
    grid = torch.tensor(LUT[:8], dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    up, down = torch.bucketize(a, mid, right=True), torch.bucketize(a, mid)
    code = torch.where(up % 2 == 0, up, down)
    return (torch.sign(b) * grid[code] * torch.exp2(e)).flatten(-2)


def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind == "write":
        return _nearest64(s.k), _nearest64(s.v)
    return _evict64(s) if kind == "evict" else _attention64(s)


def _evict64(s):
    """Weights, keys and values of what is kept; the whole numbers are not computed ones."""
    keep, recent = s.case["keep"], s.case["recent"]
    n, h = s.weights.shape[:2]
    host = s.weights.double().cpu().numpy()
    weights = torch.zeros((n, h, keep), dtype=torch.float64, device=s.cache.device)
    k = torch.zeros((n, keep, h, s.dim), dtype=torch.float64, device=s.cache.device)
    v = torch.zeros_like(k)
    for b, length in enumerate(s.lens_list):
        kept = []
        old = max(0, length - recent) if length > keep else length
        for x in host[b]:
            # numpy's stable sort of the negated weights: the lowest index first among equals
            best = np.argsort(-x[:old], kind="stable")[:max(0, min(keep, length) - (length - old))]
            kept.append(np.concatenate([np.sort(best), np.arange(old, length)]))
        t = torch.from_numpy(np.stack(kept)).to(k.device)
        m = t.shape[1]
        weights[b, :, :m] = s.weights[b].double().gather(1, t)
        kb, vb = _tokens64(s, s.table[b], t)
        k[b, :m], v[b, :m] = kb.transpose(0, 1), vb.transpose(0, 1)
    return None, None, weights, k.flatten(0, 1), v.flatten(0, 1)


def _attention64(s):
    case, kind = s.case, s.case["kind"]
    hq, h, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((s.total, hq, d), dtype=torch.float64, device=s.q.device)
    lse = torch.full((s.total, hq), -math.inf, dtype=torch.float64, device=s.q.device)
    weights = torch.zeros((case["seqs"], h, s.max_len), dtype=torch.float64, device=s.q.device)
    begin = 0
    for b, (length, n) in enumerate(zip(s.lens_list, s.rows_list)):
        t = torch.arange(length, device=s.q.device)
        k, v = _tokens64(s, s.table[b], t[None])
        if kind == "step":  # the new tokens' rows are not in the cache yet
            k[:, length - n:] = _nearest64(s.k[begin:begin + n]).transpose(0, 1)
            v[:, length - n:] = _nearest64(s.v[begin:begin + n]).transpose(0, 1)
        most = max(1, (1 << 27) // length)
        for lo in range(0, n, most):
            hi = min(n, lo + most)
            pos = torch.arange(length - n + lo, length - n + hi, device=k.device)[:, None]
            hidden = t > pos
            if case["window"]:
                hidden |= t <= pos - case["window"]
            for head in range(hq):
                x = s.q[begin + lo:begin + hi, head].double() @ k[head * h // hq].t()
                x = x / math.sqrt(d)
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                x = x.masked_fill(hidden, -math.inf)
                y = torch.logsumexp(x, -1)
                pr = torch.exp(x - y[:, None])
                out[begin + lo:begin + hi, head] = pr @ v[head * h // hq]
                lse[begin + lo:begin + hi, head] = y
                if kind == "weights":
                    pr = torch.exp(x - s.lse[begin + lo:begin + hi, head].double()[:, None])
                weights[b, head * h // hq, :length] += pr.sum(0)
        begin += n
    if kind == "attention":
        return out, lse
    weights += s.weights.double() * (
        torch.arange(s.max_len, device=t.device) < s.lens[:, None, None])
    return weights if kind == "weights" else (out, lse, weights)

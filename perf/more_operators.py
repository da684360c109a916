"""Layers of experts in 8-bit floating point, as the calls of a server.

A token's logits choose `top` of the experts (route). The pairs (token, choice)
are put in the order of their experts (arrange): row r of the sorted rows
belongs to expert e for starts[e] <= r < starts[e + 1], tokens[r] is its token
and place[t, j] the row of a token's j-th choice, -1 where that expert is not one
of this process's. The experts' products (product) take rows of e4m3 codes with a
scale for each 128 elements of a row, and weights with a scale for each 128 x 128
tile; the first gathers its rows from the tokens. Between the two products lies the
gated activation, quantised for the second (activate); the weighted sum of a token's
rows ends the layer (combine).

prepare() holds what a server has between calls: the weights, the rows of this
step, the maps. The plain form is the definition in elementary torch operations,
products on padded batches in 32 bits, the choice of experts in 64.
"""
import math
import types

import torch

own = False


def _case(name, kind, **kw):
    c = {"name": name, "kind": kind, "tokens": 1, "top": 8, "experts": 64, "share": 1, "cols": 0,
         "depth": 0, "gather": False, "fp32": False, "scores": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_rank": 1, "renormalise": True}
    c.update(kw)
    return c


def listed():
    return [
        # A single token's choice among few experts: latency.
        _case("route_1x6_of_64", "route", top=6, renormalise=False),
        # A large batch of prompts, scores with a bias for balance, groups of experts.
        _case("route_16384x6_of_192_grouped", "route", tokens=16384, top=6, experts=192,
              scores="sigmoid", bias=True, groups=8, top_groups=3, group_rank=2, fp32=True),
        # The map of a single token, and of that large batch.
        _case("arrange_1x8_of_128", "arrange", experts=128),
        _case("arrange_16384x6_of_192", "arrange", tokens=16384, top=6, experts=192),
        # A single token through its experts: their weights, once.
        _case("product_1x8_of_128", "product", experts=128, cols=2048, depth=4096, gather=True),
        # A decode step of a full batch: nearly every expert has a few rows.
        _case("product_64x8_of_128", "product", tokens=64, experts=128, cols=2048, depth=4096,
              gather=True),
        # A short prompt, odd counts, the second product.
        _case("product_1000x6_of_60", "product", tokens=1000, top=6, experts=60, cols=2048,
              depth=1408),
        # A large batch of prompts: bound by the matrix products.
        _case("product_8192x8_of_64", "product", tokens=8192, cols=4096, depth=4096, gather=True),
        # Between the products: a few rows, and those of a large batch.
        _case("activate_8x1024", "activate", cols=1024),
        _case("activate_65536x2048", "activate", tokens=8192, cols=2048),
        # The end of the layer: a single token, a prompt of odd length.
        _case("combine_1x8", "combine", cols=4096),
        _case("combine_8191x8", "combine", tokens=8191, cols=4096),
    ]


def _log_int(rng, lo, hi):
    """An integer from lo to hi, its logarithm spread evenly; odd more often than not."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n if rng.random() < 0.3 else min(hi, n | 1)


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["kind"], {"bytes": 0, "flops": 0})
        for k in m:
            m[k] = max(m[k], w[k])
    while True:
        kind = rng.choice(["route", "arrange", "product", "product", "product", "activate",
                           "combine"])
        c = _case("", kind, tokens=_log_int(rng, 1, 16384), fp32=rng.random() < 0.4,
                  experts=rng.choice([8, 16, 32, 60, 64, 96, 128, 160, 192, 256]),
                  share=rng.choice([1, 1, 1, 2, 4]), top=rng.randint(1, 8))
        if kind == "route":
            c["share"], c["scores"] = 1, rng.choice(["softmax", "sigmoid"])
            c["bias"], c["renormalise"] = rng.random() < 0.5, rng.random() < 0.6
            if rng.random() < 0.5:
                c["groups"] = rng.choice([2, 4])
                c["top_groups"] = rng.randint(1, c["groups"])
                c["group_rank"] = rng.choice([1, 2])
                c["top"] = min(c["top"], c["experts"] // c["groups"] * c["top_groups"])
        elif kind == "product":
            c["cols"], c["depth"] = _log_int(rng, 64, 8192), 128 * _log_int(rng, 1, 56)
            c["gather"] = rng.random() < 0.5
        elif kind == "activate":
            c["cols"] = 128 * _log_int(rng, 1, 56)
        elif kind == "combine":
            c["cols"] = _log_int(rng, 64, 8192)
        del c["name"]
        w = work(c)
        if (all(w[k] <= most[kind][k] for k in w) and
                (kind != "product" or c["experts"] * c["cols"] * c["depth"] <= 1 << 30)):
            return c


def _rows(case):
    """The expected number of rows of this process's experts, and of its experts that have one."""
    total = case["experts"] * case["share"]
    rows = case["tokens"] * case["top"] / case["share"]
    return rows, case["experts"] * (1 - (1 - min(1, case["top"] / total)) ** case["tokens"])


def work(case):
    t, top, e, n, k = (case[x] for x in ("tokens", "top", "experts", "cols", "depth"))
    size = 4 if case["fp32"] else 2
    kind, pairs = case["kind"], t * top
    if kind == "route":
        return {"bytes": t * e * size + 8 * pairs + (4 * e if case["bias"] else 0),
                "flops": 4.0 * t * e}
    if kind == "arrange":
        return {"bytes": 12 * pairs + 4 * (e + 1), "flops": 0.0}
    if kind == "activate":
        return {"bytes": pairs * n * (2 * size + 1 + 1 / 32), "flops": 8.0 * pairs * n}
    if kind == "combine":
        return {"bytes": pairs * (2 * n + 8) + t * n * size, "flops": 2.0 * pairs * n}
    rows, active = _rows(case)
    read = min(t, rows) if case["gather"] else rows
    return {"bytes": active * n * k * (1 + 1 / 4096) + read * k * (1 + 1 / 32) + 2 * rows * n +
            (4 * rows if case["gather"] else 0), "flops": 2.0 * rows * n * k}


# ---- what a program has in hand ----------------------------------------------------


def _codes(x, amax):
    """e4m3 codes of x and scales: amax / 448 (1 for zeros), amax of x's blocks, spread over x."""
    s = torch.where(amax == 0, torch.ones_like(amax), amax / 448)
    return (x / s).to(torch.float8_e4m3fn).view(torch.uint8), s


def _quantised_rows(x):
    """Codes [rows, K] and scales [K / 128, rows]."""
    b = x.unflatten(-1, (-1, 128))
    q, s = _codes(b, b.abs().amax(-1, keepdim=True))
    return q.flatten(-2), s.squeeze(-1).t().contiguous()


def _quantised_weights(x):
    """Codes [N, K] and scales [ceil(N / 128), K / 128]."""
    n, k = x.shape
    b = torch.nn.functional.pad(x, (0, 0, 0, -n % 128)).unflatten(0, (-1, 128)).unflatten(2, (-1, 128))
    q, s = _codes(b, b.abs().amax((1, 3), keepdim=True))
    return q.flatten(2, 3).flatten(0, 1)[:n], s[:, 0, :, 0]


def _experts_of(case, g):
    """ids [tokens, top] of unequally liked experts, -1 for those of other processes."""
    dev = torch.device("cuda")
    total = case["experts"] * case["share"]
    liked = 0.5 * torch.randn(total, generator=g, device=dev)
    x = torch.randn((case["tokens"], total), generator=g, device=dev) + liked
    ids = x.topk(min(case["top"], total), dim=1).indices
    return torch.where(ids < case["experts"], ids, -1).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    t, top, e, n, k = (case[x] for x in ("tokens", "top", "experts", "cols", "depth"))
    s = types.SimpleNamespace(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    kind = torch.float32 if case["fp32"] else torch.bfloat16
    if case["kind"] == "route":
        s.logits = (1.5 * normal(t, e) + 0.5 * normal(e)).to(kind)
        s.bias = 0.1 * normal(e) if case["bias"] else None
        return s
    if case["kind"] == "activate":
        s.x = (normal(t * top, 2 * n) * torch.exp(0.5 * normal(2 * n))).to(kind)
        return s
    s.ids = _experts_of(case, g)
    if case["kind"] == "arrange":
        return s
    s.starts, s.tokens, s.place = _arrange(s)
    if case["kind"] == "combine":
        s.y = normal(t * top, n).to(torch.bfloat16)
        s.weights = torch.softmax(normal(t, top), 1)
        return s
    # weights of a step behind each other in memory, as a server keeps them
    s.b = torch.empty((e, n, k), dtype=torch.uint8, device=dev)
    s.sfb = torch.empty((e, (n + 127) // 128, k // 128), device=dev)
    for i in range(e):
        s.b[i], s.sfb[i] = _quantised_weights(normal(n, k) / math.sqrt(k))
    s.a, s.sfa = _quantised_rows(normal(t if case["gather"] else t * top, k) *
                                 torch.exp(0.5 * normal(k)))
    s.rows = s.tokens if case["gather"] else None
    # what a program knows of the counts: a bound for its padded batches
    s.most = int(s.starts.diff().max())
    s.out = torch.zeros((t * top, n), dtype=torch.bfloat16, device=dev)
    return s


# ---- the plain form -----------------------------------------------------------------


def _best(key, count):
    """The `count` largest of each row, the lowest index first among equals."""
    return key.sort(dim=-1, descending=True, stable=True).indices[..., :count]


def _route(s):
    c = s.case
    x = s.logits.double()
    if c["scores"] == "softmax":
        score = torch.exp(x - x.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    key = x if s.bias is None else score + s.bias.double()
    if c["top_groups"] < c["groups"]:
        by = (key if c["group_rank"] == 1 else score if s.bias is None else key)
        by = by.unflatten(1, (c["groups"], -1))
        value = by.sort(dim=-1, descending=True).values[..., :c["group_rank"]].sum(-1)
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, _best(value, c["top_groups"]),
                                                                  True)
        key = key.masked_fill(~keep.repeat_interleave(by.shape[2], 1), -math.inf)
    ids = _best(key, c["top"])
    w = score.gather(1, ids)
    if c["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return ids.int(), (2.5 * w).float()


def _arrange(s):
    t, top = s.ids.shape
    e = s.case["experts"]
    flat = s.ids.flatten().long()
    mine = (flat >= 0) & (flat < e)
    order = torch.where(mine, flat, e).sort(stable=True).indices
    counts = (torch.zeros(e, dtype=torch.int64, device=flat.device)
              .index_add_(0, torch.where(mine, flat, 0), mine.long()))
    starts = torch.nn.functional.pad(counts.cumsum(0), (1, 0))
    row = torch.arange(t * top, device=flat.device)
    tokens = torch.where(row < starts[-1], order // top, -1)
    place = torch.empty_like(order).scatter_(0, order, row)
    place = torch.where(mine, place, -1).view(t, top)
    return starts.int(), tokens.int(), place.int()


def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _product(s):
    e, n, k = s.b.shape
    r = torch.arange(s.out.shape[0], device=s.b.device)
    expert = (r[:, None] >= s.starts[1:]).sum(1)
    live = (expert < e)[:, None]
    expert = expert.clamp(max=e - 1)
    a = (_values(s.a).unflatten(1, (-1, 128)) * s.sfa.t()[..., None]).flatten(1)
    a = a[r if s.rows is None else s.rows.clamp(min=0).long()]
    scale = s.sfb.repeat_interleave(128, 1)[:, :n, :, None]
    if len(r) <= e:  # few rows: each with its expert's weights
        w = _values(s.b[expert]).unflatten(2, (-1, 128)).mul_(scale[expert]).flatten(2)
        y = torch.matmul(w, a[..., None]).squeeze(2)
    else:
        w = _values(s.b).unflatten(2, (-1, 128)).mul_(scale).flatten(2)
        at = s.starts[:-1, None] + torch.arange(s.most, device=r.device)
        x = a[at.clamp(max=len(r) - 1).long()]  # [experts, most, K]
        y = torch.matmul(w, x.transpose(1, 2).contiguous())
        y = y[expert, :, (r - s.starts[expert]).clamp(max=s.most - 1)]
    return torch.where(live, y.to(torch.bfloat16), s.out)


def _activate(s):
    gate, up = s.x.float().chunk(2, 1)
    q, scales = _quantised_rows(gate / (1 + torch.exp(-gate)) * up)
    return q.view(torch.float8_e4m3fn), scales


def _combine(s):
    y = s.y[s.place.clamp(min=0).long()].float()
    w = torch.where(s.place >= 0, s.weights, torch.zeros_like(s.weights))
    return (y * w[..., None]).sum(1).to(torch.float32 if s.case["fp32"] else torch.bfloat16)


# ---- one pass -------------------------------------------------------------------------


def run(s):
    c = s.case
    kind = c["kind"]
    if not own:
        return {"route": _route, "arrange": _arrange, "product": _product, "activate": _activate,
                "combine": _combine}[kind](s)
    from gcnasm_amd import experts

    if kind == "route":
        return experts.route(s.logits, c["top"], bias=s.bias, scores=c["scores"],
                             groups=c["groups"], top_groups=c["top_groups"],
                             group_rank=c["group_rank"], renormalise=c["renormalise"], scale=2.5)
    if kind == "arrange":
        return experts.arrange(s.ids, c["experts"])
    if kind == "product":
        return experts.product(s.a, s.sfa, s.b, s.sfb, s.starts, rows=s.rows, out=s.out)
    if kind == "activate":
        q, scales = experts.activate(s.x)
        return q.view(torch.float8_e4m3fn), scales
    return experts.combine(s.y, s.place, s.weights,
                           dtype=torch.float32 if c["fp32"] else torch.bfloat16)


# ---- the definition in 64 bits ----------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "arrange":
        return None
    if kind == "route":
        return None, _weights64(s)
    if kind == "product":
        return _product64(s)
    if kind == "activate":
        return _activate64(s)
    out = torch.zeros((case["tokens"], case["cols"]), dtype=torch.float64, device=s.y.device)
    for j in range(s.place.shape[1]):
        here = torch.nonzero(s.place[:, j] >= 0)[:, 0]
        out[here] += s.weights[here, j, None].double() * s.y[s.place[here, j].long()].double()
    return out


def _weights64(s):
    """Row by row on the host: the experts in the order of their keys, by Python's stable sort."""
    c = s.case
    x = s.logits.double().cpu()
    score = torch.softmax(x, 1) if c["scores"] == "softmax" else torch.sigmoid(x)
    key = x if s.bias is None else score + s.bias.double().cpu()
    by = score if s.bias is None and c["group_rank"] > 1 else key
    per = c["experts"] // c["groups"]
    weights = []
    for p, k, b in zip(score.tolist(), key.tolist(), by.tolist()):
        value = [sum(sorted(b[i * per:i * per + per])[-c["group_rank"]:])
                 for i in range(c["groups"])]
        kept = sorted(range(c["groups"]), key=lambda i: -value[i])[:c["top_groups"]]
        among = [i for i in range(c["experts"]) if i // per in kept]
        chosen = [p[i] for i in sorted(among, key=lambda i: -k[i])[:c["top"]]]
        total = math.fsum(chosen) if c["renormalise"] else 1.0
        weights.append([2.5 * w / total for w in chosen])
    return torch.tensor(weights, dtype=torch.float64)


def _table64():
    """The values of the 256 codes: 1 sign bit, 4 of the exponent (bias 7), 3 of the mantissa."""
    v = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        v.append((-1) ** (code >> 7) * (2.0 ** -9 * m if e == 0 else 2.0 ** (e - 7) * (1 + m / 8)))
    v[127] = v[255] = math.nan
    return torch.tensor(v, dtype=torch.float64, device="cuda")


def _product64(s):
    table, starts = _table64(), s.starts.tolist()
    out = s.out.double()
    n, k = s.b.shape[1:]
    col, depth = torch.arange(n, device=out.device) // 128, torch.arange(k, device=out.device) // 128
    for e, (lo, hi) in enumerate(zip(starts, starts[1:])):
        if lo == hi:
            continue
        w = table[s.b[e].int()] * s.sfb[e].double()[col][:, depth]
        m = torch.arange(lo, hi, device=out.device) if s.rows is None else s.rows[lo:hi].long()
        out[lo:hi] = (table[s.a[m].int()] * s.sfa.double()[depth][:, m].t()) @ w.t()
    return out


def _activate64(s):
    """Of each 128 the largest magnitude is 448 scales; the nearest of the format's values times
    the scale, the one with the even code where two are."""
    gate, up = s.x.double().chunk(2, 1)
    y = (up * gate * torch.sigmoid(gate)).unflatten(1, (-1, 128))
    amax = y.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    grid = _table64()[:127]
    a = (y / scale).abs()
    mid = (grid[1:] + grid[:-1]) / 2
    up_, down = torch.bucketize(a, mid, right=True), torch.bucketize(a, mid)
    v = grid[torch.where(up_ % 2 == 0, up_, down)]
    return (torch.sign(y) * v).flatten(1), scale.squeeze(-1).t().contiguous()

"""Attention over long paged caches, as measured cases.

Two ways that a serving loop has around reading every cached token for every
sequence at every step:

  sparse  one new token of every sequence attends to the pages that a cheap score
          selects for it: the bounds of the pages that got new keys are brought up
          to date, the pages are scored and selected, and attended to
  shared  one new token of every sequence of a batch whose sequences begin with the
          same long prefix: the prefix's pages are read once for all of them, and
          joined with what each sequence has behind it

With `own` false `run` computes them in elementary torch operations; with `own`
true it calls sapphire_b200.attention.  `exact` states the definitions again in
64 bits.

The cache's bytes.  A page holds `page` token slots of every KV head; its bytes
are, for each KV head, [K rows | V rows | K scales | V scales].  A row of a dense
cache is its head_dim values.  A row of a quantised cache is nb = head_dim / 32
blocks of 32 codes (Q8_0: 8 bits, code + 128; Q4_0: 4 bits, low nibble first),
stored as 8 * nb words of 4 codes in the order [8][nb]: word w of block b at
w * nb + b.  Its scales are nb fp32 numbers, padded to 2, 4 or 8.

The summary's bytes.  For each page, for each KV head: the upper bounds of its
keys in each dim as head_dim signed bytes, then the lower bounds; behind the KV
heads their scales, one fp32 number each, the whole padded to 16 bytes.  With lo
and hi the least and the largest key of a dim among the page's tokens,
s = max(|lo|, |hi| over dims) / 127 and r = 1 / s (both 0 where s is below 2^-126):
codes ceil(hi r) and floor(lo r), within -127 .. 127; every step rounded to fp32.
A page of keys that are not all finite has s = inf and codes 0.

The score of a page for a KV head.  Each query head's values as codes
c = round(q r), half away from zero, with t = max |q| / 127 and r = 1 / t as above
(a head that is not finite: 0).  n = sum over dims of the larger of c hi and c lo,
a whole number.  score = max over the KV head's query heads of n t, times s; 0
where s is 0, inf where s is inf; every step rounded to fp32.  A sequence of up to
`budget` pages keeps all of them; else the first `first` and the last `last` pages
are in, and of the others those of the largest scores, the earlier of two alike.
The selected pages keep their order.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
FIRST, LAST = 1, 2          # pages that are always selected: the sequence's beginning, and its newest tokens


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # The repository's decode configuration (4 query heads, 1 KV head of 256), one
        # sequence over an fp32 cache: the smallest call, where latency is everything.
        {"name": "sparse_one_f32", "op": "sparse", "seqs": 1, "longest": 2047, "even": True, "new": 1, "budget": 32,
         "heads": 4, "kv_heads": 1, "dim": 256, "page": 16, "cache": "f32", "type": "f32"},
        # An ordinary batch in bf16, ragged, some sequences empty.
        {"name": "sparse_16_bf16", "op": "sparse", "seqs": 16, "longest": 16001, "even": False, "new": 1, "budget": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "cache": "bf16", "type": "bf16"},
        # One KV head per query head, head_dim 64, f16, pages of 24 tokens.
        {"name": "sparse_48_f16_mha", "op": "sparse", "seqs": 48, "longest": 5800, "even": False, "new": 1, "budget": 40,
         "heads": 24, "kv_heads": 24, "dim": 64, "page": 24, "cache": "f16", "type": "f16"},
        # The first step behind three ragged prompts of an 8-bit cache, whose pages all get their bounds.
        {"name": "sparse_3_prompts_q8", "op": "sparse", "seqs": 3, "longest": 8001, "even": False, "new": 8001, "budget": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "cache": "q8_0", "type": "bf16"},
        # Two long documents over a 4-bit cache, five query heads to a KV head.
        {"name": "sparse_2_long_q4", "op": "sparse", "seqs": 2, "longest": 131071, "even": True, "new": 1, "budget": 64,
         "heads": 40, "kv_heads": 8, "dim": 128, "page": 64, "cache": "q4_0", "type": "bf16"},
        # A large batch over an 8-bit cache.
        {"name": "sparse_64_q8", "op": "sparse", "seqs": 64, "longest": 16384, "even": False, "new": 1, "budget": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "cache": "q8_0", "type": "bf16"},
        # Four answers to one prompt of the repository's decode configuration, fp32 cache.
        {"name": "shared_4_f32", "op": "shared", "seqs": 4, "prefix": 1531, "longest": 130, "heads": 4, "kv_heads": 1,
         "dim": 256, "page": 16, "cache": "f32", "type": "f32"},
        # An ordinary batch behind one system prompt.
        {"name": "shared_16_bf16", "op": "shared", "seqs": 16, "prefix": 4099, "longest": 700, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "cache": "bf16", "type": "bf16"},
        # One KV head per query head, head_dim 64, f16, pages of 24 tokens.
        {"name": "shared_48_f16_mha", "op": "shared", "seqs": 48, "prefix": 6001, "longest": 300, "heads": 24, "kv_heads": 24,
         "dim": 64, "page": 24, "cache": "f16", "type": "f16"},
        # Questions about one document held in 4 bits, five query heads to a KV head.
        {"name": "shared_24_q4", "op": "shared", "seqs": 24, "prefix": 60001, "longest": 250, "heads": 40, "kv_heads": 8,
         "dim": 128, "page": 64, "cache": "q4_0", "type": "bf16"},
        # The same of a large batch over an 8-bit cache.
        {"name": "shared_96_q8", "op": "shared", "seqs": 96, "prefix": 16385, "longest": 500, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 32, "cache": "q8_0", "type": "bf16"},
        # A large batch behind a long document in bf16.
        {"name": "shared_64_bf16", "op": "shared", "seqs": 64, "prefix": 32768, "longest": 500, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "cache": "bf16", "type": "bf16"},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sparse", "shared"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    dim = rng.choice([64, 96, 128, 128, 192, 256])
    kind = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    cache = rng.choice(["bf16", "bf16", "f16", "q8_0", "q8_0", "q4_0", "f32"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100])
    width = {"f32": 4, "bf16": 2, "f16": 2, "q8_0": 1, "q4_0": 1}[cache]
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache, "type": kind}
    if op == "sparse":
        room = 64 * 8192 * 8 * 128 // (kv_heads * dim * width * (2 if page == 1 else 1) * (1 + group // 8))
        seqs = _spread(rng, 1, 64)
        longest = _spread(rng, page, max(page, min(131071, room // seqs)))
        case.update(seqs=seqs, longest=longest, even=rng.random() < 0.3, new=rng.choice([1, 1, 1, longest]),
                    budget=_spread(rng, FIRST + LAST, max(FIRST + LAST, 4096 // page)))
        while work(case)["bytes"] > 340e6:     # no more than the largest listed
            case["longest"] = case["longest"] * 3 // 4
        return case
    rows = 64 * 32 * 32768 * 128 // (8 if "f32" in (kind, cache) else 1)     # rows of queries times tokens times dims
    seqs = _spread(rng, 2, 128)
    room = rows // (seqs * kv_heads * group * dim)
    prefix = _spread(rng, 1, max(1, min(65536, room)))
    case.update(seqs=seqs, prefix=prefix, longest=_spread(rng, 1, max(1, min(1000, room, 64 * 500 * 16 * 128 // (seqs * kv_heads * dim)))))
    return case


# ------------------------------------------------------- shapes of a case --
def _lengths(case):
    """Tokens of each sequence (of a shared prefix: behind it): the case's, not the seed's."""
    rng = random.Random("%d %d" % (case["seqs"], case["longest"]))
    n = [case["longest"] if case.get("even") else rng.randint(case["longest"] // 2, case["longest"])
         for _ in range(case["seqs"])]
    if not case.get("even") and len(n) > 4:
        n[1], n[3] = 0, 1                     # a slot without a sequence (or with nothing behind the prefix), one just begun
    n[-1] = case["longest"]
    return n


def _layout(case):
    """(bytes of a row, padded scales of a row, offsets of K rows, V rows, K scales, V scales, bytes of a page and KV head)."""
    dim, page, nb = case["dim"], case["page"], case["dim"] // 32
    row = {"f32": 4 * dim, "bf16": 2 * dim, "f16": 2 * dim, "q8_0": dim, "q4_0": dim // 2}[case["cache"]]
    ns = (2 if nb <= 2 else 4 if nb <= 4 else 8) if case["cache"][0] == "q" else 0
    at = [0, page * row, 2 * page * row, 2 * page * row + 4 * page * ns]
    return row, ns, at, at[3] + 4 * page * ns


def _summary_bytes(case):
    return case["kv_heads"] * 2 * case["dim"] + -(-4 * case["kv_heads"] // 16) * 16


def _pages(n, page):
    return -(-n // page)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    row, ns, _, _ = _layout(case)
    keys = case["kv_heads"] * (row + 4 * (case["dim"] // 32 if ns else 0))   # K of one token
    n, page = _lengths(case), case["page"]
    io = 2 * case["seqs"] * case["heads"] * case["dim"] * size
    if case["op"] == "shared":
        seen = case["prefix"] + sum(n)
        tables = 4 * (_pages(case["prefix"], page) + sum(_pages(m, page) for m in n) + case["seqs"])
        return {"bytes": 2 * keys * seen + io + tables,
                "flops": 4 * case["heads"] * case["dim"] * (case["seqs"] * case["prefix"] + sum(n))}
    one = case["kv_heads"] * (2 * case["dim"] + 4)                           # a page's bounds
    b = io + 4 * (2 * case["seqs"] + case["seqs"] * case["kv_heads"] * case["budget"])
    flops = 0
    for m in n:
        pages = _pages(m, page)
        kept = min(pages, case["budget"])
        seen = kept * page - (pages * page - m)
        begin = max(0, m - case["new"]) // page                              # the first page with new keys
        b += (m - begin * page) * keys + 2 * (pages - begin) * one + begin * one + 2 * keys * seen + 4 * pages
        flops += case["heads"] * case["dim"] * (4 * pages + 4 * seen)
    return {"bytes": b, "flops": flops}


# ---------------------------------------------------------------- quantise --
def _codes(x, cache):
    """Codes (uint8, one a value) and scales of blocks of 32 values, by the library's formulas in fp32."""
    x = x.float().unflatten(-1, (-1, 32))
    a = x.abs()
    top = a.amax(-1, keepdim=True)
    if cache == "q8_0":
        d = top / 127.0
        inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
        t = x * inv
        t = torch.where(t < 0, -torch.floor(0.5 - t), torch.floor(t + 0.5))       # half away from zero
        return t.clamp(-127, 127).add(128).to(torch.uint8), d[..., 0]
    at = torch.where(a == top, torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)   # the first of the largest
    d = x.gather(-1, at) / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    return (x * inv + 8.5).floor().clamp(0, 15).to(torch.uint8), d[..., 0]


def _row_bytes(codes, cache):
    """Codes [..., nb, 32] as the bytes of a row: words of 4 codes in the order [8][nb]."""
    w = codes.unflatten(-1, (8, 4)).transpose(-3, -2)
    if cache == "q4_0":
        w = w[..., 0::2] | (w[..., 1::2] << 4)
    return w.flatten(-3)


def _row_values(rows, scales, case):
    """fp32 values [..., dim] of quantised rows."""
    nb = case["dim"] // 32
    if case["cache"] == "q4_0":
        rows = torch.stack((rows & 15, rows >> 4), -1).flatten(-2)
    c = rows.unflatten(-1, (8, nb, 4)).transpose(-3, -2).flatten(-2).float()     # [..., nb, 32]
    return ((c - (128 if case["cache"] == "q8_0" else 8)) * scales[..., :nb, None]).flatten(-2)


def _planes(pages, case):
    """Views of the cache's bytes: K rows, V rows [pages, kv_heads, page, ...], and their scales (None of a dense cache)."""
    row, ns, at, chunk = _layout(case)
    p = pages.view(pages.shape[0], case["kv_heads"], chunk)
    kind = torch.uint8 if ns else TYPES[case["cache"]]
    rows = [p[..., o:o + case["page"] * row].view(kind).unflatten(-1, (case["page"], -1)) for o in at[:2]]
    if not ns:
        return rows[0], rows[1], None, None
    sc = [p[..., o:o + case["page"] * ns * 4].view(torch.float32).unflatten(-1, (case["page"], ns)) for o in at[2:]]
    return rows[0], rows[1], sc[0], sc[1]


def _values(planes, j, pages, case):
    """fp32 K (j = 0) or V (j = 1) rows [..., kv_heads, page, dim] of these pages."""
    x = planes[j][pages]
    return _row_values(x, planes[2 + j][pages], case) if case["cache"][0] == "q" else x.float()


# ----------------------------------------------------------------- prepare --
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, kind = "cuda", TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    s, n, page = {"case": case}, _lengths(case), case["page"]
    parts = ([case["prefix"]] if case["op"] == "shared" else []) + n
    pages_of = [_pages(max(m, 1), page) for m in parts]
    used = sum(pages_of)
    order = torch.randperm(used + 3, device=dev, generator=g).to(torch.int32)
    order_cpu, at = order.cpu(), 0
    if case["op"] == "shared":
        s["prefix_table"] = order[:pages_of[0]].clone()
        s["prefix_length"] = torch.tensor([case["prefix"]], dtype=torch.int32, device=dev)
        at = pages_of.pop(0)
    table = torch.full((case["seqs"], max(pages_of)), -1, dtype=torch.int32)
    for i, m in enumerate(pages_of):
        table[i, :m] = order_cpu[at:at + m]
        at += m
    s["table"] = table.to(dev)
    row, ns, _, chunk = _layout(case)
    s["pages"] = torch.zeros(used + 3, case["kv_heads"] * chunk, dtype=torch.uint8, device=dev)
    # Keys and values as a model writes them: heads with scales of their own, a
    # few channels far larger than the rest in the keys, and neighbouring tokens
    # about the same thing, so that some pages matter more than others.
    planes = _planes(s["pages"], case)
    loud = 1 + 7 * (torch.rand(case["kv_heads"], 1, case["dim"], device=dev, generator=g) > 0.97).float()
    step = max(1, (1 << 27) // (case["kv_heads"] * page * case["dim"]))
    for a in range(0, used + 3, step):
        m = min(step, used + 3 - a)
        for j, plane in enumerate(planes[:2]):
            x = normal(m, case["kv_heads"], page, case["dim"])
            if j == 0:
                x = (0.7 * x + 0.7 * normal(m, case["kv_heads"], 1, case["dim"])) * loud
            if ns:
                codes, d = _codes(x.to(kind), case["cache"])
                plane[a:a + m] = _row_bytes(codes, case["cache"])
                planes[2 + j][a:a + m, ..., :d.shape[-1]] = d
            else:
                plane[a:a + m] = x.to(kind).to(plane.dtype)
            del x
    s["q"] = normal(case["seqs"], case["heads"], case["dim"]).to(kind)
    s["out"] = torch.empty_like(s["q"])
    s["lengths"] = torch.tensor(n, dtype=torch.int32, device=dev)
    if case["op"] == "sparse":
        # The step's new tokens are written; the bounds are of the tokens before them.
        new = [min(m, case["new"]) for m in n]
        s["start"] = torch.tensor([m - a for m, a in zip(n, new)], dtype=torch.int32, device=dev)
        s["cu"] = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device=dev)
        s["new"] = sum(new)
        s["summary"] = torch.zeros(used + 3, _summary_bytes(case), dtype=torch.uint8, device=dev)
        _summarise(s, torch.zeros_like(s["start"]), s["start"])
        s["selected"] = torch.empty(case["seqs"], case["kv_heads"], case["budget"], dtype=torch.int32, device=dev)
        s["selected_lengths"] = torch.empty(case["seqs"], dtype=torch.int32, device=dev)
    return s


# --------------------------------------------------------------------- run --
def run(s):
    if own:
        return {"sparse": _sparse_own, "shared": _shared_own}[s["case"]["op"]](s)
    return {"sparse": _sparse_plain, "shared": _shared_plain}[s["case"]["op"]](s)


_kept = {}          # what a program keeps beside its model: the context


def _handle(s):
    if "handle" not in s:
        import sapphire_b200 as sp
        from sapphire_b200.attention import KVCache
        if "ctx" not in _kept:
            _kept["ctx"] = sp.Context(num_threads=1)
            _kept["ctx"].set_stream(torch.cuda.current_stream().cuda_stream)
        c = s["case"]
        s["handle"] = KVCache(_kept["ctx"], c["cache"], c["page"], c["kv_heads"], c["dim"], s["pages"])
    return s["handle"]


def _sparse_own(s):
    kv = _handle(s)
    kv.summarise(s["summary"], s["table"], tokens=s["new"], start=s["start"], cu_tokens=s["cu"])
    kv.select(s["q"], s["summary"], s["table"], s["lengths"], s["selected"], s["selected_lengths"], first=FIRST, last=LAST)
    kv.attend(s["q"], s["selected"], s["selected_lengths"], s["out"])
    return s["selected"], s["selected_lengths"], s["out"]


def _shared_own(s):
    _handle(s).attend_shared(s["q"], s["prefix_table"], s["prefix_length"], s["table"], s["lengths"], s["out"])
    return s["out"]


# -------------------------------------------------------------- plain forms --
def _over_127(x):
    """max |x| / 127 of the last dim, and its reciprocal, both 0 where that is below 2^-126."""
    s = x / torch.full_like(x, 127.0)          # (a number as the divisor would be multiplied by its reciprocal)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    return s, torch.where(s != 0, 1.0 / s, torch.zeros_like(s))


def _bounds(summary, case):
    """Views of a summary: codes [pages, kv_heads, 2, dim] and scales [pages, kv_heads]."""
    n, d = case["kv_heads"], case["dim"]
    codes = summary[:, :n * 2 * d].view(torch.int8).unflatten(-1, (n, 2, d))
    return codes, summary[:, n * 2 * d:n * 2 * d + 4 * n].view(torch.float32)


def _summarise(s, start, end):
    """Bounds of the pages that hold positions start .. end - 1 of each sequence, of their tokens below end."""
    c = s["case"]
    planes, page = _planes(s["pages"], c), c["page"]
    codes, scales = _bounds(s["summary"], c)
    at = torch.arange(s["table"].shape[1], device=start.device)
    seq, pg = torch.nonzero((at >= start[:, None] // page) & (at * page < end[:, None]) & (start < end)[:, None], as_tuple=True)
    step = max(1, (1 << 27) // (c["kv_heads"] * page * c["dim"]))
    for a in range(0, len(seq), step):
        ids = s["table"][seq[a:a + step], pg[a:a + step]].long()
        k = _values(planes, 0, ids, c)
        there = (pg[a:a + step, None] * page + torch.arange(page, device=k.device) < end[seq[a:a + step], None])[:, None, :, None]
        finite = (torch.isfinite(k) | ~there).all(-1).all(-1)
        hi = k.masked_fill(~there, -math.inf).amax(2)
        lo = k.masked_fill(~there, math.inf).amin(2)
        d, r = _over_127(torch.maximum(hi.abs(), lo.abs()).amax(-1, keepdim=True))
        both = torch.stack(((hi * r).ceil(), (lo * r).floor()), 2).clamp(-127, 127)
        codes[ids] = both.masked_fill(~finite[..., None, None], 0).to(torch.int8)
        scales[ids] = torch.where(finite, d[..., 0], math.inf)


def _select_plain(s):
    c, n = s["case"], s["lengths"].long()
    page, budget, group = c["page"], c["budget"], c["heads"] // c["kv_heads"]
    codes, scales = _bounds(s["summary"], c)
    q = s["q"].float().unflatten(1, (c["kv_heads"], group))
    t, r = _over_127(q.abs().amax(-1, keepdim=True))
    x = q * r
    x = torch.where(x < 0, -torch.floor(0.5 - x), torch.floor(x + 0.5))
    bad = ~torch.isfinite(q).all(-1, keepdim=True)
    x, t = x.masked_fill(bad, 0), t.masked_fill(bad, 0)
    ids = s["table"].clamp(min=0).long()
    pages = -(-n // page)
    at = torch.arange(ids.shape[1], device=n.device)
    score = torch.empty(c["seqs"], c["kv_heads"], ids.shape[1], device=n.device)
    signed = torch.cat((x.clamp(min=0), x.clamp(max=0)), -1)                      # what meets the upper and the lower bounds
    for i in range(c["seqs"]):
        b = codes[ids[i]].float().flatten(2).transpose(0, 1)                      # [kv_heads, pages, 2 dim]
        whole = b @ signed[i].transpose(-1, -2)                                   # whole numbers below 2^24: exact
        d = scales[ids[i]].T
        v = (whole * t[i].transpose(-1, -2)).amax(-1) * d
        score[i] = torch.where(d == 0, 0.0, torch.where(d == math.inf, math.inf, v)) + 0.0
    always = (at < FIRST) | (at >= pages[:, None] - LAST) | (pages[:, None] <= budget)
    there = at < pages[:, None]
    rank = torch.where(always[:, None], 2, 1).masked_fill(~there[:, None], 0)     # by rank, then by score, then by place
    by_score = torch.sort(score, dim=-1, descending=True, stable=True).indices
    best = by_score.gather(-1, torch.sort(rank.expand_as(score).gather(-1, by_score), dim=-1, descending=True, stable=True).indices)
    kept = pages.clamp(max=budget)
    if best.shape[-1] < budget:
        best = torch.nn.functional.pad(best, (0, budget - best.shape[-1]))
    k = torch.arange(budget, device=n.device)
    inside = (k < kept[:, None])[:, None].expand(-1, c["kv_heads"], -1)
    best = best[..., :budget].masked_fill(~inside, 1 << 30).sort(-1).values
    physical = s["table"].long()[:, None].expand(-1, c["kv_heads"], -1).gather(-1, best.masked_fill(~inside, 0))
    s["selected"].copy_(physical.masked_fill(~inside, -1))
    s["selected_lengths"].copy_(n - (pages - kept) * page)


def _sparse_plain(s):
    c = s["case"]
    _summarise(s, s["start"], s["lengths"])
    _select_plain(s)
    ids, n = s["selected"], s["selected_lengths"]
    planes = _planes(s["pages"], c)
    heads = torch.arange(c["kv_heads"], device=n.device)[:, None]
    group = c["heads"] // c["kv_heads"]
    seen = torch.arange(c["budget"] * c["page"], device=n.device) < n[:, None]
    step = max(1, (1 << 27) // (c["heads"] * c["budget"] * c["page"] + c["kv_heads"] * c["budget"] * c["page"] * c["dim"]))
    for a in range(0, c["seqs"], step):
        b = slice(a, a + step)
        at = ids[b].clamp(min=0).long()

        def rows(j):                               # [seqs, kv_heads, tokens, dim] in fp32
            x = planes[j][at, heads]
            x = _row_values(x, planes[2 + j][at, heads], c) if c["cache"][0] == "q" else x.float()
            return x.flatten(2, 3)

        score = s["q"][b].float().unflatten(1, (c["kv_heads"], group)) @ rows(0).transpose(-1, -2) / math.sqrt(c["dim"])
        score = score.masked_fill(~seen[b, None, None], -math.inf)
        top = score.amax(-1, keepdim=True)
        p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
        total = p.sum(-1, keepdim=True)
        v = rows(1).masked_fill(~seen[b, None, :, None], 0.0)
        s["out"][b] = (p @ v / torch.where(total == 0, 1.0, total)).flatten(1, 2).to(s["out"].dtype)
    return s["selected"], s["selected_lengths"], s["out"]


def _shared_plain(s):
    c, q = s["case"], s["q"]
    planes, page = _planes(s["pages"], c), c["page"]
    group, n = c["heads"] // c["kv_heads"], s["lengths"]

    def prefix(j):                                 # [kv_heads, tokens, dim]
        return _values(planes, j, s["prefix_table"].long(), c).transpose(0, 1).flatten(1, 2)[:, :c["prefix"]]

    def behind(j):                                 # [seqs, kv_heads, tokens, dim]
        return _values(planes, j, s["table"].clamp(min=0).long(), c).transpose(1, 2).flatten(2, 3)

    qs = q.float().unflatten(1, (c["kv_heads"], group)) / math.sqrt(c["dim"])
    by_head = qs.transpose(0, 1).flatten(1, 2)     # [kv_heads, seqs * group, dim]
    front = by_head @ prefix(0).transpose(-1, -2)
    front = front.unflatten(1, (c["seqs"], group)).transpose(0, 1)               # [seqs, kv_heads, group, prefix]
    back = qs @ behind(0).transpose(-1, -2)
    seen = torch.arange(back.shape[-1], device=q.device) < n[:, None]
    back = back.masked_fill(~seen[:, None, None], -math.inf)
    top = torch.maximum(front.amax(-1, keepdim=True), back.amax(-1, keepdim=True))
    front, back = (front - top).exp(), (back - top).exp()
    total = front.sum(-1, keepdim=True) + back.sum(-1, keepdim=True)
    out = (front.transpose(0, 1).flatten(1, 2) @ prefix(1)).unflatten(1, (c["seqs"], group)).transpose(0, 1)
    out = out + back @ behind(1).masked_fill(~seen[:, None, :, None], 0.0)
    return (out / total).flatten(1, 2).to(q.dtype)


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    """The definitions, in 64 bits, sequence by sequence."""
    s = prepare(case, seed)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def attended(q, k, v):
        return torch.softmax(q.double() @ k.T * case["dim"] ** -0.5, -1) @ v

    def tokens(ids, h, j, n):
        return _head_values(s["pages"], ids, h, case, j).reshape(-1, case["dim"])[:n]

    if case["op"] == "shared":
        for h in range(case["kv_heads"]):
            k, v = (tokens(s["prefix_table"].long(), h, j, case["prefix"]) for j in (0, 1))
            for i, n in enumerate(_lengths(case)):
                at = slice(h * group, (h + 1) * group)
                ids = s["table"][i, :_pages(n, page)].long()
                out[i, at] = attended(s["q"][i, at], torch.cat((k, tokens(ids, h, 0, n))), torch.cat((v, tokens(ids, h, 1, n))))
        return out
    selected = torch.full(s["selected"].shape, -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros_like(s["selected_lengths"])
    for i, n in enumerate(_lengths(case)):
        pages = _pages(n, page)
        ids = s["table"][i, :pages].long()
        kept = min(pages, case["budget"])
        lengths[i] = n - (pages - kept) * page
        if n == 0:
            continue
        for h in range(case["kv_heads"]):
            at = slice(h * group, (h + 1) * group)
            if pages <= case["budget"]:
                chosen = list(range(pages))
            else:
                score = _exact_scores(s, i, ids, h, n, case).tolist()
                middle = sorted(range(FIRST, pages - LAST), key=lambda p: (-score[p], p))
                chosen = sorted(list(range(FIRST)) + middle[:kept - FIRST - LAST] + list(range(pages - LAST, pages)))
            mine = ids[torch.tensor(chosen, device="cuda")]
            selected[i, h, :kept] = mine.to(torch.int32)
            k, v = (tokens(mine, h, j, int(lengths[i])) for j in (0, 1))
            out[i, at] = attended(s["q"][i, at], k, v)
    return selected, lengths, out


def _exact_scores(s, i, ids, h, n, case):
    """Scores of sequence i's pages for KV head h: every step that rounds to fp32 rounded there."""
    def r(y):
        return y.float().double()

    def unit(top):
        d = r(top / 127)
        d = torch.where(d < 2.0 ** -126, 0.0, d)
        return d, torch.where(d == 0, 0.0, r(1 / d))

    page, group = case["page"], case["heads"] // case["kv_heads"]
    k = r(_head_values(s["pages"], ids, h, case, 0))
    k[-1, n - (len(ids) - 1) * page:] = k[-1, 0]                 # behind the last token: nothing new
    hi, lo = k.max(1).values, k.min(1).values
    d, inv = unit(k.abs().flatten(1).max(1).values[:, None])
    up, down = torch.ceil(r(hi * inv)).clamp(-127, 127), torch.floor(r(lo * inv)).clamp(-127, 127)
    q = s["q"][i, h * group:(h + 1) * group].double()
    t, inv = unit(q.abs().max(1).values[:, None])
    x = r(q * inv)
    code = x.sign() * (x.abs() + 0.5).floor()
    whole = torch.maximum(code[:, None] * up, code[:, None] * down).sum(-1)      # [group, pages]
    return r(r(whole * t).max(0).values * d[:, 0]) + 0.0


def _head_values(pages, ids, h, c, j):
    """The numbers that the K (j = 0) or V (j = 1) rows of these pages stand for, of one KV head: [ids, page, dim]."""
    row, ns, at, chunk = _layout(c)
    p = pages.reshape(-1, c["kv_heads"], chunk)[ids, h]
    rows = p[:, at[j]:at[j] + c["page"] * row].reshape(-1, c["page"], row)
    if not ns:
        return rows.contiguous().view(TYPES[c["cache"]]).double()
    nb = c["dim"] // 32
    scales = p[:, at[2 + j]:at[2 + j] + 4 * ns * c["page"]].contiguous().view(torch.float32)
    scales = scales.reshape(-1, c["page"], ns)[..., :nb].double()
    out = torch.empty(*rows.shape[:-1], c["dim"], dtype=torch.float64, device=pages.device)
    for word in range(8):
        for block in range(nb):
            for i in range(4):
                if c["cache"] == "q8_0":
                    q = rows[..., 4 * (word * nb + block) + i].to(torch.int16) - 128
                else:
                    q = (rows[..., 2 * (word * nb + block) + i // 2] >> (4 * (i % 2)) & 15).to(torch.int16) - 8
                out[..., 32 * block + 4 * word + i] = q * scales[..., block]
    return out

"""The serving operators around a paged key-value cache, as measured cases.

Three operators that one decoding step uses together:

  rope    rotary positions of the query and key heads, both layouts, part of a
          head, frequencies scaled for long contexts
  cache   new keys and values written into a paged cache (kept as they are or
          quantised to 8 or 4 bits a code with one fp32 scale per 32 dims) and
          whole sequences read back from it
  attend  attention of one new token of every sequence over its pages

With `own` false `run` computes them in elementary torch operations; with `own`
true it calls sapphire_b200.attention.  `exact` states the definitions again in
64 bits.

The cache's bytes.  A page holds `page` token slots of every KV head; its bytes
are, for each KV head, [K rows | V rows | K scales | V scales].  A row of a dense
cache is its head_dim values.  A row of a quantised cache is nb = head_dim / 32
blocks of 32 codes (Q8_0: 8 bits, code + 128; Q4_0: 4 bits, low nibble first),
stored as 8 * nb words of 4 codes in the order [8][nb]: word w of block b at
w * nb + b.  Its scales are nb fp32 numbers, padded to 2, 4 or 8.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # One token of the repository's decode configuration (4 query heads, 1 KV
        # head of 256): the smallest call, where latency is everything.
        {"name": "rope_one_token", "op": "rope", "tokens": 1, "heads": 4, "kv_heads": 1, "dim": 256, "rot": 256,
         "layout": "half", "type": "f32", "theta": 1e6, "scaling": "none", "factor": 1.0, "far": 2048},
        # A serving step of 65 sequences: half of each head rotated, interleaved pairs.
        {"name": "rope_step_65", "op": "rope", "tokens": 65, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64,
         "layout": "interleaved", "type": "bf16", "theta": 1e4, "scaling": "linear", "factor": 4.0, "far": 32768},
        # The largest: prompts of 16381 tokens together, long-context frequencies.
        {"name": "rope_prompt_16381", "op": "rope", "tokens": 16381, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "layout": "half", "type": "bf16", "theta": 5e5, "scaling": "banded", "factor": 8.0, "far": 131072},
        # One new token of 32 sequences stored as it is.
        {"name": "cache_step_32_bf16", "op": "cache", "seqs": 32, "new": 32, "before": 250, "kv_heads": 8, "dim": 128,
         "page": 16, "cache": "bf16", "type": "bf16", "read": False},
        # A 512-token prompt of the repository's decode configuration into a 4-bit cache, read back in fp32.
        {"name": "cache_prompt_512_q4", "op": "cache", "seqs": 1, "new": 512, "before": 0, "kv_heads": 1, "dim": 256,
         "page": 32, "cache": "q4_0", "type": "f32", "read": True},
        # Chunks of three ragged prompts behind what they wrote before, 8 bits, read back for the prefill.
        {"name": "cache_chunk_3001_q8", "op": "cache", "seqs": 3, "new": 3001, "before": 5000, "kv_heads": 8, "dim": 128,
         "page": 16, "cache": "q8_0", "type": "bf16", "read": True},
        # The largest: a chunk of a long document; the whole of it is read back.
        {"name": "cache_long_8192_q8", "op": "cache", "seqs": 1, "new": 8192, "before": 57001, "kv_heads": 8, "dim": 128,
         "page": 64, "cache": "q8_0", "type": "f16", "read": True},
        # The repository's decode configuration: one sequence, a 512-token window, fp32 cache.
        {"name": "attend_one_f32", "op": "attend", "seqs": 1, "longest": 577, "even": True, "window": 512, "heads": 4,
         "kv_heads": 1, "dim": 256, "page": 16, "cache": "f32", "type": "f32"},
        # An ordinary batch in bf16, ragged, some sequences empty.
        {"name": "attend_16_bf16", "op": "attend", "seqs": 16, "longest": 4000, "even": False, "window": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "cache": "bf16", "type": "bf16"},
        # One KV head per query head, head_dim 64, f16, pages of 24 tokens.
        {"name": "attend_48_f16_mha", "op": "attend", "seqs": 48, "longest": 2900, "even": False, "window": 0, "heads": 24,
         "kv_heads": 24, "dim": 64, "page": 24, "cache": "f16", "type": "f16"},
        # A large batch over an 8-bit cache.
        {"name": "attend_64_q8", "op": "attend", "seqs": 64, "longest": 8192, "even": False, "window": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "cache": "q8_0", "type": "bf16"},
        # Two long documents over a 4-bit cache, five query heads to a KV head.
        {"name": "attend_2_long_q4", "op": "attend", "seqs": 2, "longest": 131071, "even": True, "window": 0, "heads": 40,
         "kv_heads": 8, "dim": 128, "page": 64, "cache": "q4_0", "type": "bf16"},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    dim = rng.choice([64, 96, 128, 128, 192, 256])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        heads = kv_heads * group
        room = 16381 * 40 * 128 // ((heads + kv_heads) * dim * (2 if kind == "f32" else 1))
        return {"op": op, "tokens": _spread(rng, 1, min(16381, room)), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]), "type": kind,
                "theta": rng.choice([1e4, 5e5, 1e6]), "scaling": rng.choice(["none", "linear", "banded", "yarn"]),
                "factor": rng.choice([2.0, 4.0, 8.0, 32.0]), "far": rng.choice([2048, 32768, 131072, 1 << 20])}
    cache = rng.choice(["f32", "bf16", "f16", "q8_0", "q8_0", "q4_0", "q4_0"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100])
    if op == "cache":
        room = 65000 * 8 * 128 // (kv_heads * dim * (2 if "f32" in (kind, cache) else 1))
        seqs = _spread(rng, 1, 64)
        new = min(room // 4, _spread(rng, seqs, 8192))
        return {"op": op, "seqs": seqs, "new": max(new, 1), "before": _spread(rng, 1, max(1, room // (2 * seqs))),
                "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache, "type": kind, "read": cache[0] == "q"}
    width = {"f32": 4, "bf16": 2, "f16": 2, "q8_0": 1, "q4_0": 1}[cache]
    room = 64 * 6000 * 8 * 128 // (kv_heads * dim * width)
    seqs = _spread(rng, 1, 96)
    return {"op": op, "seqs": seqs, "longest": _spread(rng, 1, max(1, min(131071, room // seqs))), "even": rng.random() < 0.3,
            "window": rng.choice([0, 0, 0, 512, 4096]), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "page": page, "cache": cache, "type": kind}


# ------------------------------------------------------- shapes of a case --
def _lengths(case):
    """Tokens of each sequence: the case's, not the seed's."""
    rng = random.Random("%d %d" % (case["seqs"], case["longest"]))
    n = [case["longest"] if case["even"] else rng.randint(case["longest"] // 2, case["longest"])
         for _ in range(case["seqs"])]
    if not case["even"] and len(n) > 4:
        n[1], n[3] = 0, 1                     # a slot without a sequence, a sequence just begun
    n[-1] = case["longest"]
    return n


def _chunks(case):
    """(tokens before, new tokens) of each sequence."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["new"], case["before"]))
    cut = sorted(rng.randint(0, case["new"]) for _ in range(case["seqs"] - 1))
    if case["new"] == case["seqs"]:           # a decoding step: one token each
        cut = list(range(1, case["seqs"]))
    new = [b - a for a, b in zip([0] + cut, cut + [case["new"]])]
    before = [rng.randint(0, case["before"]) for _ in range(case["seqs"])]
    before[0] = case["before"]
    return before, new


def _layout(case):
    """(bytes of a row, padded scales of a row, offsets of K rows, V rows, K scales, V scales, bytes of a page and KV head)."""
    dim, page, nb = case["dim"], case["page"], case["dim"] // 32
    row = {"f32": 4 * dim, "bf16": 2 * dim, "f16": 2 * dim, "q8_0": dim, "q4_0": dim // 2}[case["cache"]]
    ns = (2 if nb <= 2 else 4 if nb <= 4 else 8) if case["cache"][0] == "q" else 0
    at = [0, page * row, 2 * page * row, 2 * page * row + 4 * page * ns]
    return row, ns, at, at[3] + 4 * page * ns


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["dim"] * size + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    row, ns, _, _ = _layout(case)
    stored = 2 * case["kv_heads"] * (row + 4 * (case["dim"] // 32 if ns else 0))   # K and V of one token
    if case["op"] == "cache":
        before, new = _chunks(case)
        given = 2 * case["kv_heads"] * case["dim"] * size
        b = case["new"] * (given + stored)
        if case["read"]:
            b += (sum(before) + case["new"]) * (stored + given)
        return {"bytes": b + 4 * (2 * case["seqs"] + 1), "flops": 0}
    seen = [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]
    q = case["seqs"] * case["heads"] * case["dim"]
    return {"bytes": sum(seen) * stored + 2 * q * size + 4 * sum(-(-n // case["page"]) for n in seen) + 4 * case["seqs"],
            "flops": 4 * sum(seen) * case["heads"] * case["dim"]}


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


# ----------------------------------------------------------------- prepare --
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, kind = "cuda", TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    s = {"case": case}
    if case["op"] == "rope":
        n, dim = case["tokens"], case["dim"]
        s["positions"] = torch.randint(0, case["far"], (n,), device=dev, generator=g, dtype=torch.int32)
        s["q"], s["k"] = normal(n, case["heads"], dim).to(kind), normal(n, case["kv_heads"], dim).to(kind)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        return s
    if case["op"] == "cache":
        before, new = _chunks(case)
        total = [a + b for a, b in zip(before, new)]
    else:
        total = _lengths(case)
    pages_of = [-(-max(n, 1) // case["page"]) for n in total]
    width, used = max(pages_of), sum(pages_of)
    order = torch.randperm(used + 3, device=dev, generator=g).to(torch.int32)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32)
    firsts = [sum(pages_of[:i]) for i in range(len(pages_of))]
    order_cpu = order.cpu()
    for i, (a, m) in enumerate(zip(firsts, pages_of)):
        table[i, :m] = order_cpu[a:a + m]
    s["table"] = table.to(dev)
    row, ns, at, chunk = _layout(case)
    s["pages"] = torch.zeros(used + 3, case["kv_heads"] * chunk, dtype=torch.uint8, device=dev)
    # Keys and values as a model writes them: heads with scales of their own, a
    # few channels far larger than the rest in the keys.
    planes = _planes(s["pages"], case)
    loud = 1 + 7 * (torch.rand(case["kv_heads"], 1, case["dim"], device=dev, generator=g) > 0.97).float()
    step = max(1, (1 << 27) // (case["kv_heads"] * case["page"] * case["dim"]))
    for a in range(0, used + 3, step):
        m = min(step, used + 3 - a)
        for j, plane in enumerate(planes[:2]):
            x = normal(m, case["kv_heads"], case["page"], case["dim"])
            if j == 0:
                x *= loud
            if ns:
                codes, d = _codes(x.to(kind), case["cache"])
                plane[a:a + m] = _row_bytes(codes, case["cache"])
                planes[2 + j][a:a + m, ..., :d.shape[-1]] = d
            else:
                plane[a:a + m] = x.to(kind).to(plane.dtype)
            del x
    if case["op"] == "cache":
        n, h, dim = case["new"], case["kv_heads"], case["dim"]
        s["k"], s["v"] = (normal(n, h, dim) * loud[:, 0]).to(kind), normal(n, h, dim).to(kind)
        s["start"] = torch.tensor(before, dtype=torch.int32, device=dev)
        s["cu"] = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device=dev)
        s["cu_all"] = torch.tensor([0] + [sum(total[:i + 1]) for i in range(len(new))], dtype=torch.int32, device=dev)
        if case["read"]:
            s["k_out"] = torch.empty(sum(total), h, dim, dtype=kind, device=dev)
            s["v_out"] = torch.empty_like(s["k_out"])
        return s
    s["q"] = normal(case["seqs"], case["heads"], case["dim"]).to(kind)
    s["out"] = torch.empty_like(s["q"])
    s["lengths"] = torch.tensor(total, dtype=torch.int32, device=dev)
    return s


# --------------------------------------------------------------------- run --
def run(s):
    case = s["case"]
    if own:
        return {"rope": _rope_own, "cache": _cache_own, "attend": _attend_own}[case["op"]](s)
    return {"rope": _rope_plain, "cache": _cache_plain, "attend": _attend_plain}[case["op"]](s)


_kept = {}          # what a program keeps beside its model: the context, and a plan for each kind of rotation


def _context():
    import sapphire_b200 as sp
    if "ctx" not in _kept:
        _kept["ctx"] = sp.Context(num_threads=1)
        _kept["ctx"].set_stream(torch.cuda.current_stream().cuda_stream)
    return _kept["ctx"]


def _rope_own(s):
    from sapphire_b200.attention import Rope
    c = s["case"]
    key = (c["dim"], c["rot"], c["layout"], c["theta"], c["scaling"], c["factor"])
    if key not in _kept:
        _kept[key] = Rope(_context(), c["dim"], rot_dim=c["rot"], layout=c["layout"], theta=c["theta"],
                          scaling=c["scaling"], factor=c["factor"], original_context=8192)
    _kept[key].apply(s["positions"], s["q"], s["k"], q_out=s["q_out"], k_out=s["k_out"])
    return s["q_out"], s["k_out"]


def _handle(s):
    if "handle" not in s:
        from sapphire_b200.attention import KVCache
        c = s["case"]
        s["handle"] = KVCache(_context(), c["cache"], c["page"], c["kv_heads"], c["dim"], s["pages"])
    return s["handle"]


def _cache_own(s):
    c, kv = s["case"], _handle(s)
    kv.write(s["k"], s["v"], s["table"], start=s["start"], cu_tokens=s["cu"])
    if not c["read"]:
        return _planes(s["pages"], c)[:2]
    kv.read(s["k_out"], s["v_out"], s["table"], cu_tokens=s["cu_all"])
    return s["k_out"], s["v_out"]


def _attend_own(s):
    _handle(s).attend(s["q"], s["table"], s["lengths"], s["out"], window=s["case"]["window"])
    return s["out"]


# -------------------------------------------------------------- plain forms --
def _frequencies(c, device):
    """Radians a position of each pair, and the factor on cos and sin, in 64 bits."""
    i = torch.arange(0, c["rot"], 2, dtype=torch.float64, device=device)
    f = c["theta"] ** (-i / c["rot"])
    factor, orig = c["factor"], 8192
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] == "banded":
        # turns over the original context: at least 4 keep their frequency, at most 1 are slowed, between them a blend
        turns = orig * f / (2 * math.pi)
        mix = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * mix + f / factor * (1 - mix), 1.0
    if c["scaling"] == "yarn":
        # the pair at which the original context holds `turns` turns
        pair = [c["rot"] * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(c["theta"])) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), c["rot"] - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rope_plain(s):
    c = s["case"]
    f, m = _frequencies(c, s["q"].device)
    angle = s["positions"].double()[:, None] * f
    cos, sin = (angle.cos() * m).float()[:, None], (angle.sin() * m).float()[:, None]
    return _turn(s["q"], cos, sin, c), _turn(s["k"], cos, sin, c)


def _turn(x, cos, sin, c):
    y, half = x.float().clone(), c["rot"] // 2
    at = (slice(0, half), slice(half, c["rot"])) if c["layout"] == "half" else (slice(0, c["rot"], 2), slice(1, c["rot"], 2))
    a, b = x[..., at[0]].float(), x[..., at[1]].float()
    y[..., at[0]], y[..., at[1]] = a * cos - b * sin, a * sin + b * cos
    return y.to(x.dtype)


def _places(cu, start, table, page, tokens):
    """(page, slot) of each token of ragged sequences."""
    t = torch.arange(tokens, device=cu.device)
    n = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    at = t - cu[n] + (start[n] if start is not None else 0)
    return table[n, at // page].long(), at % page


def _cache_plain(s):
    c = s["case"]
    planes = _planes(s["pages"], c)
    page, slot = _places(s["cu"], s["start"], s["table"], c["page"], c["new"])
    quant = c["cache"][0] == "q"
    for j, x in ((0, s["k"]), (1, s["v"])):
        if quant:
            codes, d = _codes(x, c["cache"])
            planes[j][page, :, slot] = _row_bytes(codes, c["cache"])
            planes[2 + j][:, :, :, :d.shape[-1]][page, :, slot] = d
        else:
            planes[j][page, :, slot] = x.to(planes[j].dtype)
    if not c["read"]:
        return planes[:2]
    page, slot = _places(s["cu_all"], None, s["table"], c["page"], s["k_out"].shape[0])
    return [_row_values(planes[j][page, :, slot], planes[2 + j][page, :, slot], c).to(s["k"].dtype) for j in (0, 1)]


def _attend_plain(s):
    c, q, lengths = s["case"], s["q"], s["lengths"]
    planes = _planes(s["pages"], c)
    pages = s["table"].clamp(min=0).long()
    t = torch.arange(pages.shape[1] * c["page"], device=q.device)
    seen = t < lengths[:, None]
    if c["window"]:
        seen &= t >= lengths[:, None] - c["window"]

    def dense(j):                              # [seqs, kv_heads, tokens, dim]
        x = planes[j][pages]
        x = _row_values(x, planes[2 + j][pages], c) if c["cache"][0] == "q" else x.float()
        return x.transpose(1, 2).flatten(2, 3)

    qs = q.float().unflatten(1, (c["kv_heads"], -1))
    score = qs @ dense(0).transpose(-1, -2) / math.sqrt(c["dim"])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    v = dense(1).masked_fill(~seen[:, None, :, None], 0.0)
    out = p @ v / torch.where(total == 0, 1.0, total)
    return out.flatten(1, 2).to(q.dtype)


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    """The definitions, in 64 bits, sequence by sequence."""
    s = prepare(case, seed)
    if case["op"] == "rope":
        return [_rotated(x, s["positions"], case) for x in (s["q"], s["k"])]
    k, v = (_cache_values(s["pages"], case, j) for j in (0, 1))      # [pages, kv_heads, page, dim] in 64 bits
    if case["op"] == "cache":
        before, new = _chunks(case)
        table = s["table"].tolist()
        outs = []
        for x, dense in ((s["k"], k), (s["v"], v)):
            stored = _stored(x, case["cache"])
            row = 0
            for n, (b, m) in enumerate(zip(before, new)):
                t = torch.arange(b, b + m, device=dense.device)
                page = s["table"][n].long()[t // case["page"]]
                dense[page, :, t % case["page"]] = stored[row:row + m]
                row += m
            if case["read"]:
                parts = []
                for n, (b, m) in enumerate(zip(before, new)):
                    used = -(-(b + m) // case["page"])
                    d = dense[torch.tensor(table[n][:used], device=dense.device).long()]
                    parts.append(d.transpose(1, 2).flatten(0, 1)[:b + m])
                outs.append(torch.cat(parts))
            else:
                outs.append(dense)
        return outs
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for n, length in enumerate(_lengths(case)):
        first = max(0, length - case["window"]) if case["window"] else 0
        if length == first:
            continue
        t = torch.arange(first, length, device="cuda")
        page, slot = s["table"][n].long()[t // case["page"]], t % case["page"]
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            w = torch.softmax(s["q"][n, heads].double() @ k[page, h, slot].T * case["dim"] ** -0.5, -1)
            out[n, heads] = w @ v[page, h, slot]
    return out


def _rotated(x, positions, c):
    """Pairs as complex numbers times m * e^(i * position * frequency)."""
    inv = torch.tensor([c["theta"] ** (-2 * i / c["rot"]) for i in range(c["rot"] // 2)], dtype=torch.float64)
    m = 1.0
    for i in range(c["rot"] // 2):
        slow = float(inv[i]) / c["factor"]
        if c["scaling"] == "linear":
            inv[i] = slow
        elif c["scaling"] == "banded":
            turns = 8192 * float(inv[i]) / (2 * math.pi)
            if turns < 4:
                part = (turns - 1) / 3 if turns > 1 else 0.0
                inv[i] = (1 - part) * slow + part * float(inv[i])
        elif c["scaling"] == "yarn":
            m = 0.1 * math.log(c["factor"]) + 1
            ends = [c["rot"] / 2 * math.log(8192 / (2 * math.pi * r)) / math.log(c["theta"]) for r in (32, 1)]
            a, b = max(0, math.floor(ends[0])), min(c["rot"] - 1, math.ceil(ends[1]))
            part = min(1.0, max(0.0, (i - a) / max(b - a, 1e-3)))
            inv[i] = part * slow + (1 - part) * float(inv[i])
    angle = positions.double()[:, None] * inv.to(x.device)
    turn = torch.polar(torch.full_like(angle, m), angle)[:, None]
    y, half = x.double(), c["rot"] // 2
    r = y[..., :c["rot"]]
    z = torch.complex(r[..., :half], r[..., half:]) if c["layout"] == "half" else torch.complex(r[..., ::2], r[..., 1::2])
    z = z * turn
    r = torch.cat((z.real, z.imag), -1) if c["layout"] == "half" else torch.stack((z.real, z.imag), -1).flatten(-2)
    return torch.cat((r, y[..., c["rot"]:]), -1)


def _stored(x, cache):
    """What the cache holds of x, as numbers: each step of the formulas that rounds to fp32, rounded there."""
    if cache[0] != "q":
        return x.to(TYPES[cache]).double()

    def r(y):
        return y.float().double()

    b = x.double().reshape(*x.shape[:-1], -1, 32)
    if cache == "q8_0":
        d = r(b.abs().max(-1, keepdim=True).values / 127)
        t = r(b * torch.where(d == 0, 0.0, r(1 / d)))
        q = (t.sign() * (t.abs() + 0.5).floor()).clamp(-127, 127)
    else:
        size, place = torch.sort(b.abs(), dim=-1, descending=True, stable=True)
        d = r(torch.take_along_dim(b, place[..., :1], -1) / -8)
        q = r(r(b * torch.where(d == 0, 0.0, r(1 / d))) + 8.5).trunc().clamp(0, 15) - 8
    return (q * d).flatten(-2)


def _cache_values(pages, c, j):
    """The numbers that the K (j = 0) or V (j = 1) rows of every page stand for."""
    row, ns, at, chunk = _layout(c)
    p = pages.reshape(-1, c["kv_heads"], chunk)
    rows = p[:, :, at[j]:at[j] + c["page"] * row].reshape(-1, c["kv_heads"], c["page"], row)
    if not ns:
        return rows.view(TYPES[c["cache"]]).double()
    nb = c["dim"] // 32
    scales = p[:, :, at[2 + j]:at[2 + j] + 4 * ns * c["page"]].contiguous().view(torch.float32)
    scales = scales.reshape(-1, c["kv_heads"], c["page"], ns)[..., :nb].double()
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

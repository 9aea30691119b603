"""Attention of a batch behind a shared prefix against a plain 64-bit form.

Tolerances, before the output's own rounding, with A = sum_t p_t |v_t|.  A score is
off by at most ds, which moves p by a factor of exp(+-ds) and the sum alike, so out
by at most 4 ds A.

fp32 queries: ds = scale sum|q k| 2^-19 and 2^-17 A besides, as attention over one
table (test_attention_gpu).
16-bit queries: products of 16-bit operands are exact and sums fp32, so ds is that
and, where the cache's values become fp16, r scale sum|q k| more: r = 2^-11 of F32, one
rounding, and 2^-10 of Q8_0 and Q4_0, (1 + 2^-11)^2 - 1 to 2^-22, the scale's and the
product's.  A probability is rounded once, by 2^-8 (bf16 operands) or 2^-11 of it (fp16),
a converted value by r.  Small values: an fp16 step is at least 2^-24, and a group's
largest value is at least 2^-4 (a code of 127 times a scale of 2^14, 2^-24 times; 8 times
2^14, 2^-20 times: 2^-3), so half a step of a value or of its offset is 2^-21 of it, and
probabilities below 2^-21 of the largest are off by 2^-32 of it: 2^-20 max|v| together, and
scale sum|q| max|k| 2^-20 of a score.  512 truncating steps of an MMA cost 2^-15 of A.
Together A (4 ds + 2^-14 + p + r) + max|v| 2^-20.
What a sequence has behind the prefix is off as in attend_plain there, over bf16
queries one fp16 rounding of p (2^-12) and of integer queries (max|q| sum|k| 2^-14)
more.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_attention_gpu import CACHES, IO, assert_within, cache_values, dev_ctx, gen, make_cache, ragged  # noqa: E402,F401


def shared_case(ctx, dtype, kind, prefix, lengths, heads, group, dim, page, seed=0, fill=0xFF, loud=1.0, positive=False):
    """A cache with a prefix and what each sequence has behind it; slots that nobody
    holds are 0xFF bytes (NaN in every dense type and in every scale)."""
    g = gen(seed)
    parts = [prefix] + list(lengths)
    need = [-(-n // page) for n in parts]
    pages = sum(need) + 2
    kv = make_cache(ctx, dtype, page, heads, dim, pages, fill=fill)
    order = torch.randperm(pages, device="cuda", generator=g).int().cpu()
    table = torch.full((len(parts), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    table = table.cuda()
    n = sum(parts)
    if n:
        k = torch.randn(n, heads, dim, device="cuda", generator=g)
        k[..., ::17] *= 4 * loud
        v = torch.randn(n, heads, dim, device="cuda", generator=g) * torch.rand(n, heads, 1, device="cuda", generator=g) * loud
        if positive:
            v = v.abs() + 1
        kv.write(k.to(IO[kind]), v.to(IO[kind]), table, cu_tokens=ragged(parts))
    q = torch.randn(len(lengths), heads * group, dim, device="cuda", generator=g).to(IO[kind])
    prefix_table = table[0, :max(1, need[0])].contiguous()
    own = table[1:, :max(1, max(need[1:], default=0))].contiguous()
    return kv, prefix_table, own, q


def shared_plain(kv, q, prefix_table, prefix, table, lengths, page, heads, dim, dtype, scale=None):
    """fp64 out, lse and the error bounds before rounding."""
    k, v = (cache_values(kv.pages, dtype, page, heads, dim, j) for j in (0, 1))
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    lse_bound = torch.zeros_like(lse)
    group, scale = q.shape[1] // heads, dim ** -0.5 if scale is None else scale
    small = q.dtype != torch.float32
    bf16 = dtype == "bf16" and q.dtype == torch.bfloat16
    r = 0.0 if not small else 2.0 ** -10 if dtype in ("q8_0", "q4_0") else 2.0 ** -11 if dtype == "f32" else 0.0
    for s, n in enumerate(lengths):
        if prefix + n == 0:
            continue
        t, u = torch.arange(prefix, device="cuda"), torch.arange(n, device="cuda")
        pg = torch.cat((prefix_table.long()[t // page], table[s].long()[u // page]))
        slot = torch.cat((t % page, u % page))
        for h in range(heads):
            at = slice(h * group, (h + 1) * group)
            x = q[s, at].double()
            ks, vs = k[pg, h, slot], v[pg, h, slot]
            score = x @ ks.T * scale
            ds = (x.abs() @ ks.abs().T * abs(scale)).amax(-1) * (2.0 ** -19 + r)
            if r:
                ds = ds + abs(scale) * x.abs().sum(-1) * ks.abs().max() * 2.0 ** -20
            if n and dtype in ("q8_0", "q4_0") and q.dtype == torch.bfloat16:
                ds = ds + abs(scale) * x.abs().amax(-1) * ks[prefix:].abs().sum(-1).amax() * 2.0 ** -14
            p = torch.softmax(score, -1)
            rel = 2.0 ** -17
            if small:
                rel = 2.0 ** -14 + (2.0 ** -8 if bf16 else 2.0 ** -11) + r + 2.0 ** -12
            out[s, at] = p @ vs
            bound[s, at] = (p @ vs.abs()) * (4 * ds[:, None] + rel) + vs.abs().max() * 2.0 ** -20
            lse[s, at] = torch.logsumexp(score, -1)
            lse_bound[s, at] = 2 * ds + 2.0 ** -15
    return out, bound, lse, lse_bound


def check_shared(ctx, dtype, kind, prefix, lengths, heads, group, dim, page, seed=0, scale=None, loud=1.0, positive=False):
    kv, prefix_table, table, q = shared_case(ctx, dtype, kind, prefix, lengths, heads, group, dim, page, seed, loud=loud, positive=positive)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    m = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    kv.attend_shared(q, prefix_table, m, table, n, out, lse=lse, **({} if scale is None else {"scale": scale}))
    ctx.synchronize()
    want, bound, want_lse, lse_bound = shared_plain(kv, q, prefix_table, prefix, table, lengths, page, heads, dim, dtype, scale)
    assert_within(out, want, bound)
    some = torch.isfinite(want_lse)
    assert torch.equal(lse[~some].double(), want_lse[~some]) and (out[~some] == 0).all()
    assert_within(lse[some], want_lse[some], lse_bound[some])
    return kv, prefix_table, table, q, out


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("dim,heads,group", [(64, 2, 1), (96, 1, 3), (128, 3, 4), (192, 2, 8), (256, 1, 5)])
def test_shared_types_and_heads(dev_ctx, dtype, kind, dim, heads, group):
    check_shared(dev_ctx, dtype, kind, 301, [17, 0, 1, 40], heads, group, dim, 16, seed=dim + group)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "q8_0", "q4_0", "f32"])
@pytest.mark.parametrize("prefix", [0, 1, 15, 63, 64, 65, 127, 128, 129, 256, 1000, 5000])
def test_shared_prefix_lengths(dev_ctx, dtype, prefix):
    check_shared(dev_ctx, dtype, "bf16", prefix, [3, 0, 66], 2, 4, 128, 16, seed=prefix)


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("page", [1, 3, 16, 24, 100, 4096])
def test_shared_pages(dev_ctx, dtype, page):
    check_shared(dev_ctx, dtype, "bf16", 777, [5, 130], 2, 2, 64, page, seed=page)


@pytest.mark.parametrize("dtype", ["bf16", "q8_0", "f16"])
@pytest.mark.parametrize("seqs,group", [(1, 1), (128, 1), (129, 1), (43, 3), (16, 16), (17, 16), (1, 300), (100, 7)])
@pytest.mark.parametrize("dim", [64, 192, 256])
def test_shared_rows(dev_ctx, dtype, seqs, group, dim):
    """One tile of rows, two side by side, sets of them, the last one with one."""
    check_shared(dev_ctx, dtype, "bf16", 333, [(7 * i) % 11 for i in range(seqs)], 2, group, dim, 16, seed=seqs)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "q4_0"])
@pytest.mark.parametrize("heads,seqs,group", [(12, 3, 4), (40, 2, 8), (5, 90, 3), (200, 2, 1)])
def test_shared_blocks_of_several_items(dev_ctx, dtype, heads, seqs, group):
    check_shared(dev_ctx, dtype, "bf16", 2100, [1] * seqs, heads, group, 64, 16, seed=heads)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "q8_0"])
@pytest.mark.parametrize("positive", [False, True])
def test_shared_long_pieces(dev_ctx, dtype, positive):
    """Blocks that take more tokens than O stays in tensor memory for; values of one sign."""
    check_shared(dev_ctx, dtype, "bf16", 30011, [2, 0], 80, 1, 64, 64, seed=4, positive=positive)


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("scale", [0.0078125, 1.5, -0.05])
def test_shared_scale_and_range(dev_ctx, dtype, kind, scale):
    check_shared(dev_ctx, dtype, kind, 400, [30, 7], 2, 5, 128, 16, seed=3, scale=scale, loud=8.0 if abs(scale) < 1 else 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "q8_0", "q4_0"])
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_shared_values_that_grow(dev_ctx, dtype, kind):
    """Keys and values whose size changes by powers of two along the prefix, up and down."""
    prefix, heads, dim, page = 1500, 1, 64, 16
    kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, prefix, [4], heads, 3, dim, page)
    g = gen(8)
    size = torch.exp2(torch.tensor([0, 6, -9, 3, -2, 7, -12, 1], device="cuda", dtype=torch.float32)).repeat_interleave(188)[:prefix, None, None]
    k = torch.randn(prefix, heads, dim, device="cuda", generator=g) * size.clamp(max=4)
    v = torch.randn(prefix, heads, dim, device="cuda", generator=g) * size
    kv.write(k.to(IO[kind]), v.to(IO[kind]), prefix_table[None].contiguous(), cu_tokens=ragged([prefix]))
    out = torch.empty_like(q)
    kv.attend_shared(q, prefix_table, torch.tensor([prefix], dtype=torch.int32, device="cuda"), table,
                     torch.tensor([4], dtype=torch.int32, device="cuda"), out)
    dev_ctx.synchronize()
    want, bound, _, _ = shared_plain(kv, q, prefix_table, prefix, table, [4], page, heads, dim, dtype)
    assert_within(out, want, bound)


def test_shared_query_far_from_one(dev_ctx):
    for kind, dtype in (("bf16", "f16"), ("bf16", "q8_0"), ("bf16", "bf16"), ("f16", "f16")):
        for size in (2.0 ** -12, 2.0 ** 12):
            if kind == "f16" and size > 1:
                size = 8.0
            kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, 300, [5, 5], 1, 4, 128, 16)
            q = (q.float() * size).to(q.dtype)
            out = torch.empty_like(q)
            kv.attend_shared(q, prefix_table, torch.tensor([300], dtype=torch.int32, device="cuda"), table,
                             torch.tensor([5, 5], dtype=torch.int32, device="cuda"), out, scale=0.1 / size)
            dev_ctx.synchronize()
            want, bound, _, _ = shared_plain(kv, q, prefix_table, 300, table, [5, 5], 16, 1, 128, dtype, scale=0.1 / size)
            assert_within(out, want, bound)


def test_shared_strides_and_offset(dev_ctx):
    """Strided and unaligned queries and outputs, lengths behind an offset."""
    for kind, dtype in (("bf16", "bf16"), ("f16", "q8_0"), ("f32", "f32")):
        kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, 200, [9, 30, 1], 2, 3, 64, 16, seed=6)
        n = torch.tensor([9, 30, 1], dtype=torch.int32, device="cuda")
        m = torch.tensor([200], dtype=torch.int32, device="cuda")
        ref = torch.empty_like(q)
        kv.attend_shared(q, prefix_table, m, table, n, ref)
        wide = torch.zeros(3, 7, 71, dtype=q.dtype, device="cuda")
        wide[:, 1:, 5:69] = q
        got = torch.full((3, 6, 67), 5.0, dtype=q.dtype, device="cuda")
        kv.attend_shared(wide[:, 1:, 5:69], prefix_table, m, table, n - 3, got[..., 1:65], length_offset=3)
        dev_ctx.synchronize()
        assert torch.equal(got[..., 1:65], ref)
        assert (got[..., 0] == 5).all() and (got[..., 65:] == 5).all()


def test_shared_is_repeatable_on_either_workspace(dev_ctx):
    for kind, dtype in (("bf16", "bf16"), ("bf16", "q4_0"), ("f32", "f32")):
        kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, 3000, [900, 0, 33, 2], 2, 4, 128, 16, seed=12)
        n, m = torch.tensor([900, 0, 33, 2], dtype=torch.int32, device="cuda"), torch.tensor([3000], dtype=torch.int32, device="cuda")
        ws = torch.full((kv.shared_workspace_bytes(kind, 4, 8),), 0xEE, dtype=torch.uint8, device="cuda")
        first = None
        for i in range(8):
            out = torch.full_like(q, 3.0)
            kv.attend_shared(q, prefix_table, m, table, n, out, workspace=ws if i % 2 else None)
            dev_ctx.synchronize()
            first = out if first is None else first
            assert torch.equal(out, first)


@pytest.mark.parametrize("kind,dtype", [("bf16", "bf16"), ("bf16", "q8_0"), ("f16", "bf16"), ("f32", "q4_0")])
def test_shared_workspace_on_any_sixteen_bytes(dev_ctx, kind, dtype):
    """A workspace that starts on 16 bytes and on no more, of no byte too many."""
    kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, 700, [90, 0, 33], 2, 4, 128, 16, seed=13)
    n, m = torch.tensor([90, 0, 33], dtype=torch.int32, device="cuda"), torch.tensor([700], dtype=torch.int32, device="cuda")
    size = kv.shared_workspace_bytes(kind, 3, 8)
    outs = []
    for shift in (0, 16, 240):
        room = torch.full((size + 512,), 0xEE, dtype=torch.uint8, device="cuda")
        ws, out = room[shift:shift + size], torch.full_like(q, 3.0)
        kv.attend_shared(q, prefix_table, m, table, n, out, workspace=ws)
        dev_ctx.synchronize()
        assert (room[:shift] == 0xEE).all() and (room[shift + size:] == 0xEE).all()
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    with pytest.raises(Exception, match="16-byte"):
        kv.attend_shared(q, prefix_table, m, table, n, outs[0], workspace=room[8:8 + size])


def test_shared_far_offsets(dev_ctx):
    """Prefix pages and summaries behind 4 GB of cache give the bits of near ones."""
    from sapphire_b200.attention import KVCache, kv_page_bytes
    for dtype in ("bf16", "q8_0"):
        per = kv_page_bytes(dtype, 64, 8, 128)
        count = (5 << 30) // per
        far = KVCache(dev_ctx, dtype, 64, 8, 128, torch.empty(count, per, dtype=torch.uint8, device="cuda"))
        near = make_cache(dev_ctx, dtype, 64, 8, 128, 8)
        g = gen(13)
        k, v = (torch.randn(400, 8, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
        q = torch.randn(2, 32, 128, device="cuda", generator=g).bfloat16()
        outs, bounds = [], []
        for kv, pages in ((far, [count - 1, 0, count - 2, count - 5, count - 3, 1, count - 4]), (near, [3, 0, 2, 1, 4, 5, 6])):
            table = torch.tensor([pages], dtype=torch.int32, device="cuda")
            kv.write(k, v, table, cu_tokens=ragged([400]))
            own, prefix = table[:, 5:].expand(2, -1).contiguous(), table[0, :5].contiguous()
            out = torch.empty_like(q)
            kv.attend_shared(q, prefix, torch.tensor([320], dtype=torch.int32, device="cuda"), own,
                             torch.tensor([80, 5], dtype=torch.int32, device="cuda"), out)
            summary = torch.zeros(kv.pages.shape[0], kv.summary_bytes, dtype=torch.uint8, device="cuda")
            kv.summarise(summary, table, tokens=400, cu_tokens=ragged([400]))
            dev_ctx.synchronize()
            outs.append(out)
            bounds.append(summary[table[0].long()])
        assert torch.equal(outs[0], outs[1]) and torch.equal(bounds[0], bounds[1])


def test_shared_two_contexts_at_once(sp):
    """Two contexts on streams of their own, whose calls overlap, give what each gives alone."""
    ctxs = [sp.Context(num_threads=1) for _ in range(2)]
    sets = []
    for i, ctx in enumerate(ctxs):
        kv, prefix_table, table, q = shared_case(ctx, ("bf16", "q4_0")[i], "bf16", 4000, [60, 7], 2, 40, 128, 16, seed=50 + i)
        sets.append((ctx, kv, prefix_table, table, q, torch.tensor([60, 7], dtype=torch.int32, device="cuda"), torch.tensor([4000], dtype=torch.int32, device="cuda")))
        ctx.synchronize()
    torch.cuda.synchronize()
    alone = []
    for ctx, kv, prefix_table, table, q, n, m in sets:
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        kv.attend_shared(q, prefix_table, m, table, n, out)
        ctx.synchronize()
        alone.append(out)
    outs = [[torch.empty_like(s[4]) for _ in range(6)] for s in sets]
    torch.cuda.synchronize()
    for k in range(6):
        for (ctx, kv, prefix_table, table, q, n, m), o in zip(sets, outs):
            kv.attend_shared(q, prefix_table, m, table, n, o[k])
    for ctx in ctxs:
        ctx.synchronize()
    for o, want in zip(outs, alone):
        for x in o:
            assert torch.equal(x, want)
    for ctx in ctxs:
        ctx.close()


def test_shared_growing_and_shrinking_calls(dev_ctx):
    """Calls of many shapes behind one another on the context's workspace."""
    kinds = [("bf16", 40, 2, 1, 64), ("bf16", 900, 60, 8, 128), ("q8_0", 300, 5, 2, 256), ("f16", 2000, 130, 2, 64)]
    cases = [shared_case(dev_ctx, d, "bf16", pre, [3] * s, 2, g, dim, 16, seed=i) for i, (d, pre, s, g, dim) in enumerate(kinds)]
    outs = []
    for (kv, prefix_table, table, q), kind in zip(cases * 2, kinds * 2):
        m = torch.tensor([kind[1]], dtype=torch.int32, device="cuda")
        n = torch.full((q.shape[0],), 3, dtype=torch.int32, device="cuda")
        out = torch.empty_like(q)
        kv.attend_shared(q, prefix_table, m, table, n, out)
        outs.append(out)
    dev_ctx.synchronize()
    for a, b, (kv, prefix_table, table, q), (dtype, prefix, *_) in zip(outs, outs[len(cases):], cases, kinds):
        assert torch.equal(a, b)
        want, bound, _, _ = shared_plain(kv, q, prefix_table, prefix, table, [3] * q.shape[0], 16, 2, q.shape[2], dtype)
        assert_within(a, want, bound)


def test_shared_captured_calls(sp, dev_ctx):
    """Two captured graphs with workspaces of their own, replayed at the same time; new lengths take effect."""
    st = torch.cuda.Stream()
    dev_ctx.set_stream(st.cuda_stream)
    sets = []
    for i, (dtype, kind) in enumerate((("bf16", "bf16"), ("q8_0", "bf16"), ("f32", "f32"))):
        kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, 1500, [90, 9, 40], 2, 4, 128, 16, seed=40 + i)
        n, m = torch.tensor([90, 9, 40], dtype=torch.int32, device="cuda"), torch.tensor([1500], dtype=torch.int32, device="cuda")
        ws = torch.full((kv.shared_workspace_bytes(kind, 3, 8),), 0xEE, dtype=torch.uint8, device="cuda")
        sets.append((dtype, kv, prefix_table, table, q, n, m, torch.empty_like(q), ws))
    dev_ctx.synchronize()
    graphs = []
    for dtype, kv, prefix_table, table, q, n, m, out, ws in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            with pytest.raises(sp.SapphireError, match="workspace"):
                kv.attend_shared(q, prefix_table, m, table, n, out)
            kv.attend_shared(q, prefix_table, m, table, n, out, workspace=ws)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for prefix, lengths in ((1500, [90, 9, 40]), (0, [3, 0, 40]), (129, [0, 0, 0])):
        for *_, n, m, out, ws in sets:
            n.copy_(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
            m.fill_(prefix)
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        dev_ctx.synchronize()
        for dtype, kv, prefix_table, table, q, n, m, out, ws in sets:
            want, bound, _, _ = shared_plain(kv, q, prefix_table, prefix, table, lengths, 16, 2, 128, dtype)
            assert_within(out, want, bound)
    dev_ctx.set_stream(0)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "q8_0", "f32"])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_shared_infinities_and_nan_stay_where_they_are(dev_ctx, dtype, kind):
    """A value that is not finite touches its dims (its block's, quantised); a key that is NaN its head; a query's its row."""
    heads, group, dim, prefix = 2, 2, 64, 200
    kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, prefix, [3, 3, 3], heads, group, dim, 16, fill=0)
    g = gen(1)
    n, m = torch.tensor([3, 0, 3], dtype=torch.int32, device="cuda"), torch.tensor([prefix], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(1, heads, dim, device="cuda", generator=g).to(IO[kind]) for _ in (0, 1))
    start = torch.tensor([77], dtype=torch.int32, device="cuda")

    def run(x):
        out = torch.empty_like(q)
        kv.attend_shared(x, prefix_table, m, table, n, out)
        dev_ctx.synchronize()
        return out

    for bad in (math.nan, math.inf):
        vb = v.clone()
        vb[0, 0, 5] = bad
        kv.write(k, vb, prefix_table[None].contiguous(), start=start)
        out = run(q)
        touched = slice(0, 32) if dtype == "q8_0" else slice(5, 6)
        hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
        hit[:, :group, touched] = True
        if dtype == "q8_0" and bad != bad:         # (a NaN is code 0 of a block that keeps its scale)
            hit[:] = False
        assert torch.isfinite(out[~hit].float()).all() and not torch.isfinite(out[hit].float()).any()
    if dtype != "q8_0":
        kb = k.clone()
        kb[0, 1, 9] = math.nan
        kv.write(kb, v, prefix_table[None].contiguous(), start=start)
        out = run(q)
        assert torch.isfinite(out[:, :group].float()).all() and torch.isnan(out[:, group:].float()).all()
    kv.write(k, v, prefix_table[None].contiguous(), start=start)
    x = q.clone()
    x[1, 2, 7] = math.nan
    out, ref = run(x), run(q)
    assert torch.isnan(out[1, 2].float()).all()
    out[1, 2] = ref[1, 2]
    assert torch.equal(out, ref)


def test_shared_bad_places(sp, dev_ctx):
    """A page outside the cache does not count, a length outside its table counts as its end; both are reported."""
    for kind, dtype in (("bf16", "bf16"), ("bf16", "q4_0"), ("f32", "f32")):
        kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, 320, [20, 20], 1, 4, 64, 16, seed=2)
        n = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
        out = torch.empty_like(q)

        def run(tab, length):
            kv.attend_shared(q, tab, torch.tensor([length], dtype=torch.int32, device="cuda"), table, n, out)

        for place, bad in ((3, 1 << 30), (19, -7)):
            wrong = prefix_table.clone()
            wrong[place] = bad
            run(wrong, 320)
            with pytest.raises(sp.SapphireError, match="outside"):
                dev_ctx.synchronize()
            left = torch.cat((prefix_table[:place], prefix_table[place + 1:]))
            want, bound, _, _ = shared_plain(kv, q, left, 304, table, [20, 20], 16, 1, 64, dtype)
            assert_within(out, want, bound)
        for length, counts in ((321, 320), (-1, 0), (1 << 30, 320)):
            run(prefix_table, length)
            with pytest.raises(sp.SapphireError, match="outside"):
                dev_ctx.synchronize()
            want, bound, _, _ = shared_plain(kv, q, prefix_table, counts, table, [20, 20], 16, 1, 64, dtype)
            assert_within(out, want, bound)
    dev_ctx.synchronize()


def test_shared_refusals(sp, dev_ctx):
    kv, prefix_table, table, q = shared_case(dev_ctx, "bf16", "bf16", 64, [4, 5], 2, 2, 64, 16)
    n, m, out = torch.tensor([4, 5], dtype=torch.int32, device="cuda"), torch.tensor([64], dtype=torch.int32, device="cuda"), torch.empty_like(q)
    small = torch.zeros(64, dtype=torch.uint8, device="cuda")
    good = (q, prefix_table, m, table, n, out)
    for at, bad, kw, match in ((0, q[:, :3], {}, "shape"), (5, out.half(), {}, "one type"), (4, n[:1], {}, "shape"), (3, table[:1], {}, "shape"),
                               (2, m.long(), {}, "int32"), (2, n, {}, "shape"), (1, prefix_table.long(), {}, "int32"),
                               (1, prefix_table[None], {}, "shape"), (1, prefix_table[:0], {}, "prefix_pages"), (0, q.cpu(), {}, "device memory"),
                               (1, prefix_table.cpu(), {}, "device memory"), (2, m.cpu(), {}, "device memory"), (5, out.cpu(), {}, "device memory"),
                               (5, out, {"scale": math.inf}, "scale"), (5, out, {"scale": 3e38}, "scale"), (5, out, {"workspace": small}, "workspace"),
                               (5, out, {"lse": torch.zeros(2, 3, device="cuda")}, "lse")):
        args = list(good)
        args[at] = bad
        if at == 0 and bad.shape[1] == 3:
            args[5] = out[:, :3]
            match = "query heads"
        with pytest.raises(sp.SapphireError, match=match):
            kv.attend_shared(*args, **kw)
    kv.attend_shared(q[:0], prefix_table, m, table[:0], n[:0], out[:0])
    dev_ctx.synchronize()
    for args in (("bf16", 2, 3), ("q8_0", 2, 4), ("bf16", -1, 4), ("bf16", 65535, 4096)):
        with pytest.raises(sp.SapphireError):
            kv.shared_workspace_bytes(*args)


@pytest.mark.parametrize("dtype", ["bf16", "q8_0"])
def test_shared_prefix_then_selected_pages(dev_ctx, dtype):
    """A batch answers behind one prompt, and one sequence goes on over the pages that its bounds select: both beside
    attention over a table that names the prefix's pages for every sequence."""
    heads, group, dim, page, prefix, lengths = 2, 4, 128, 16, 640, [50, 3]
    kv, prefix_table, table, q = shared_case(dev_ctx, dtype, "bf16", prefix, lengths, heads, group, dim, page, seed=21)
    n, m = torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor([prefix], dtype=torch.int32, device="cuda")
    both = torch.cat((prefix_table[None].expand(2, -1), table), 1).contiguous()
    out = [torch.empty_like(q) for _ in range(3)]
    kv.attend_shared(q, prefix_table, m, table, n, out[0])
    kv.attend(q, both, n, out[1], length_offset=prefix)
    summary = torch.zeros(kv.pages.shape[0], kv.summary_bytes, dtype=torch.uint8, device="cuda")
    total = torch.tensor([prefix + x for x in lengths], dtype=torch.int32, device="cuda")
    kv.summarise(summary, both, tokens=int(total.sum()), cu_tokens=ragged([prefix + x for x in lengths]))
    pages = both.shape[1]
    selected, left = torch.empty(2, heads, pages, dtype=torch.int32, device="cuda"), torch.empty_like(n)
    kv.select(q, summary, both, total, selected, left)
    kv.attend(q, selected, left, out[2])           # (every page is within the budget)
    dev_ctx.synchronize()
    want, bound, _, _ = shared_plain(kv, q, prefix_table, prefix, table, lengths, page, heads, dim, dtype)
    for y in out:
        assert_within(y, want, bound)

"""Bounds of pages, the selection of pages by them, and attention over a table
per KV head, against plain forms.

Bounds and selections are whole numbers and fp32 numbers of a definition that
says where it rounds: they are equal, with no tolerance (an fp32 step is a 64-bit
one rounded to fp32, which is exact for one product, sum or quotient).  Attention's
tolerance is that of attention over one table (test_attention_gpu).
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_attention_gpu import (CACHES, IO, assert_within, attend_plain, cache_values, dev_ctx, gen, make_cache,  # noqa: E402,F401
                                make_table, ragged)


def f32(y):
    """y (fp64) rounded to fp32."""
    return y.float().double()


def unit(top):
    """top / 127 and its reciprocal, 0 where the first is below 2^-126."""
    s = f32(top / 127)
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    return s, torch.where(s == 0, 0.0, f32(1 / s))


def bounds_plain(keys):
    """Codes [heads, 2, dim] and scales [heads] of a page's keys [heads, tokens, dim] (fp64)."""
    keys = f32(keys)
    hi, lo = keys.amax(1), keys.amin(1)
    bad = ~torch.isfinite(keys).flatten(1).all(1)
    s, r = unit(torch.maximum(hi.abs(), lo.abs()).amax(-1, keepdim=True))
    codes = torch.stack((f32(hi * r).ceil(), f32(lo * r).floor()), 1).clamp(-127, 127)
    codes[bad] = 0
    s = s[:, 0].clone()
    s[bad] = math.inf
    return codes, s


def bounds_of(kv, summary):
    """Codes [pages, heads, 2, dim] and scales [pages, heads] of a summary."""
    n, d = kv.kv_heads, kv.head_dim
    codes = summary[:, :n * 2 * d].view(torch.int8).reshape(-1, n, 2, d)
    return codes.double(), summary[:, n * 2 * d:n * 2 * d + 4 * n].contiguous().view(torch.float32).double()


def scores_plain(q, codes, scales):
    """Scores [pages] of one KV head: q [group, dim] (fp64), codes [pages, 2, dim], scales [pages]."""
    ok = torch.isfinite(q).all(-1)
    q = torch.where(ok[:, None], q, 0.0)
    t, r = unit(q.abs().amax(-1, keepdim=True))
    x = f32(q * r)
    c = x.sign() * (x.abs() + 0.5).floor()
    n = torch.maximum(c[:, None] * codes[:, 0], c[:, None] * codes[:, 1]).sum(-1)
    score = f32(f32(n * t).amax(0) * scales)
    return torch.where(scales == 0, 0.0, torch.where(scales == math.inf, math.inf, score))


def select_plain(scores, budget, first, last):
    """Places of the selected of len(scores) pages, in order."""
    pages = len(scores)
    if pages <= budget:
        return list(range(pages))
    score = scores.tolist()
    middle = sorted(range(first, pages - last), key=lambda p: (-score[p], p))[:budget - first - last]
    return sorted(list(range(first)) + middle + list(range(pages - last, pages)))


def empty_summary(kv, fill=0xEE):
    return torch.full((kv.pages.shape[0], kv.summary_bytes), fill, dtype=torch.uint8, device="cuda")


def filled(ctx, dtype, kind, lengths, heads, dim, page, seed=0, width=None):
    """A cache of ragged sequences whose pages differ, behind 0xFF bytes, with its summary."""
    g = gen(seed)
    pages = sum(-(-n // page) for n in lengths) + 2
    kv = make_cache(ctx, dtype, page, heads, dim, pages, fill=0xFF)
    table = make_table(lengths, page, pages, g, width)
    n = sum(lengths)
    k = torch.randn(n, heads, dim, device="cuda", generator=g)
    k = k * 0.6 + torch.randn(n // page + 1, heads, dim, device="cuda", generator=g).repeat_interleave(page, 0)[:n]
    k[..., ::17] *= 4
    v = torch.randn(n, heads, dim, device="cuda", generator=g)
    kv.write(k.to(IO[kind]), v.to(IO[kind]), table, cu_tokens=ragged(lengths))
    summary = empty_summary(kv)
    kv.summarise(summary, table, tokens=n, cu_tokens=ragged(lengths))
    return kv, table, summary, g


def check_bounds(kv, summary, table, lengths, dtype):
    keys = cache_values(kv.pages, dtype, kv.page_size, kv.kv_heads, kv.head_dim, 0)
    codes, scales = bounds_of(kv, summary)
    for s, n in enumerate(lengths):
        for i in range(-(-n // kv.page_size)):
            at = int(table[s, i])
            want = bounds_plain(keys[at][:, :min(kv.page_size, n - i * kv.page_size)])
            assert torch.equal(codes[at], want[0]), (s, i)
            assert torch.equal(scales[at], want[1]), (s, i)


# ------------------------------------------------------------------- bounds --
@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("dim,page,heads", [(64, 16, 2), (96, 24, 3), (128, 16, 8), (128, 1, 1), (192, 100, 1), (256, 7, 2)])
def test_bounds(dev_ctx, dtype, dim, page, heads):
    lengths = [3 * page + 1, 0, 1, 2 * page, page - 1 or 1]
    kv, table, summary, _ = filled(dev_ctx, dtype, "f32", lengths, heads, dim, page, seed=dim + page)
    dev_ctx.synchronize()
    check_bounds(kv, summary, table, lengths, dtype)
    used = set(table[table >= 0].tolist())
    for i in set(range(kv.pages.shape[0])) - used:
        assert (summary[i] == 0xEE).all()


@pytest.mark.parametrize("dtype", ["bf16", "q4_0"])
def test_bounds_of_long_pages(dev_ctx, dtype):
    """Pages of several warps' rows."""
    lengths = [4096 * 2 + 700, 33]
    kv, table, summary, _ = filled(dev_ctx, dtype, "bf16", lengths, 2, 64, 4096, seed=5)
    dev_ctx.synchronize()
    check_bounds(kv, summary, table, lengths, dtype)


@pytest.mark.parametrize("dtype", ["f32", "q8_0"])
@pytest.mark.parametrize("page", [1, 8, 16])
def test_bounds_as_a_sequence_grows(dev_ctx, dtype, page):
    """A prompt, chunks and single tokens leave the bounds of the whole; other pages keep theirs."""
    g = gen(page)
    pages, heads, dim = 60, 2, 64
    kv = make_cache(dev_ctx, dtype, page, heads, dim, pages)
    room = 20
    table = torch.randperm(pages, device="cuda", generator=g)[:3 * room].int().view(3, room)
    summary, at = empty_summary(kv), [0, 0, 0]
    for new in ([5, 0, 3], [1, 1, 1], [4, 9, 0], [1, 1, 1], [0, 2, 8]):
        if page == 1 and max(a + b for a, b in zip(at, new)) > room:
            break
        n = sum(new)
        k, v = (torch.randn(n, heads, dim, device="cuda", generator=g) for _ in (0, 1))
        start = torch.tensor(at, dtype=torch.int32, device="cuda")
        one = new == [1, 1, 1]
        kv.write(k, v, table, start=start, cu_tokens=None if one else ragged(new))
        kv.summarise(summary, table, tokens=None if one else n, start=start, cu_tokens=None if one else ragged(new))
        at = [a + b for a, b in zip(at, new)]
        dev_ctx.synchronize()
        check_bounds(kv, summary, table, at, dtype)


def test_bounds_of_extreme_keys(dev_ctx):
    """Zeros, numbers whose unit is no normal number, the largest, infinities and NaN; slots behind the newest token do not count."""
    page, heads, dim = 4, 1, 64
    kv = make_cache(dev_ctx, "f32", page, heads, dim, 8, fill=0xFF)
    rows = [torch.zeros(dim), torch.full((dim,), 1e-37), torch.full((dim,), 3e38), -torch.linspace(0, 1, dim),
            torch.linspace(-3, 5, dim).index_fill(0, torch.tensor([7]), math.inf),
            torch.linspace(-3, 5, dim).index_fill(0, torch.tensor([9]), math.nan),
            torch.linspace(-3, 5, dim).index_fill(0, torch.tensor([60]), -math.inf)]
    n = len(rows)
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous()
    k = torch.stack(rows).cuda()[:, None]
    kv.write(k, torch.zeros_like(k), table)
    summary = empty_summary(kv)
    kv.summarise(summary, table)
    dev_ctx.synchronize()
    check_bounds(kv, summary, table, [1] * n, "f32")
    _, scales = bounds_of(kv, summary)
    assert scales[0, 0] == 0 and scales[1, 0] == 0 and torch.isinf(scales[4:7, 0]).all()


def test_bounds_of_bad_places(sp, dev_ctx):
    """Pages outside the cache and positions outside the table are skipped and reported; the rest is done."""
    kv, table, summary, _ = filled(dev_ctx, "bf16", "bf16", [40, 40], 1, 64, 16, width=4)
    dev_ctx.synchronize()
    for start, bad in (([0, 60], None), ([0, -5], None), ([0, 0], 1 << 20), ([0, 0], -1)):
        wrong = table.clone()
        if bad is not None:
            wrong[1, 1] = bad
        again = empty_summary(kv)
        kv.summarise(again, wrong, tokens=80, start=torch.tensor(start, dtype=torch.int32, device="cuda"), cu_tokens=ragged([40, 40]))
        with pytest.raises(sp.SapphireError, match="outside"):
            dev_ctx.synchronize()
        for i in table[0, :3].tolist():
            assert torch.equal(again[i], summary[i])
    dev_ctx.synchronize()


# ---------------------------------------------------------------- selection --
def check_select(ctx, dtype, kind, lengths, heads, group, dim, page, budget, first=1, last=1, seed=0, width=None, q=None):
    kv, table, summary, g = filled(ctx, dtype, kind, lengths, heads, dim, page, seed, width)
    if q is None:
        q = torch.randn(len(lengths), heads * group, dim, device="cuda", generator=g).to(IO[kind])
    selected = torch.full((len(lengths), heads, budget), 77, dtype=torch.int32, device="cuda")
    n = torch.full((len(lengths),), 77, dtype=torch.int32, device="cuda")
    kv.select(q, summary, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), selected, n, first=first, last=last)
    ctx.synchronize()
    codes, scales = bounds_of(kv, summary)
    want = torch.full_like(selected, -1)
    want_n = torch.zeros_like(n)
    for s, m in enumerate(lengths):
        pages = -(-m // page)
        ids = table[s, :pages].long()
        want_n[s] = m - max(0, pages - budget) * page
        for h in range(heads):
            score = scores_plain(q[s, h * group:(h + 1) * group].double(), codes[ids, h], scales[ids, h])
            chosen = torch.tensor(select_plain(score, budget, first, last), device="cuda", dtype=torch.long)
            want[s, h, :len(chosen)] = ids[chosen].int()
    assert torch.equal(n, want_n)
    assert torch.equal(selected, want)
    return kv, table, summary, q, selected, n


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_select_types(dev_ctx, kind, dim):
    check_select(dev_ctx, "bf16", kind, [900, 0, 1, 333, 16 * 8, 16 * 8 + 1], 2, 4, dim, 16, 8, seed=dim)


@pytest.mark.parametrize("group", [1, 2, 7, 8, 9, 16, 33, 128])
def test_select_groups(dev_ctx, group):
    check_select(dev_ctx, "q8_0", "bf16", [500, 1200], 2, group, 128, 16, 12, seed=group)


@pytest.mark.parametrize("budget,first,last", [(1, 0, 1), (2, 1, 1), (3, 0, 3), (5, 4, 1), (17, 0, 1), (40, 3, 7), (200, 1, 1)])
@pytest.mark.parametrize("page", [1, 24])
def test_select_budgets(dev_ctx, budget, first, last, page):
    check_select(dev_ctx, "f16", "f16", [page * 41, page * 40 - 1 or 1, page * 130 + 1, 3], 2, 3, 64, page, budget, first, last, seed=budget)


@pytest.mark.parametrize("seqs,pages,budget", [(1, 129, 20), (1, 1031, 64), (1, 5000, 300), (2, 2500, 2000), (40, 600, 30), (300, 200, 10)])
def test_select_long_and_many(dev_ctx, seqs, pages, budget):
    """Clusters of 1 to 8 blocks."""
    g = torch.Generator().manual_seed(pages)
    lengths = [pages] + torch.randint(0, pages, (seqs - 1,), generator=g).tolist()
    check_select(dev_ctx, "q4_0", "bf16", lengths, 1, 4, 64, 1, budget, first=2, last=3, seed=pages)


def test_select_table_wider_than_the_sequence(dev_ctx):
    """A table of 2^18 entries, of which a sequence uses few: 32768 keys of a block have room."""
    check_select(dev_ctx, "bf16", "bf16", [700, 65], 1, 2, 64, 4, 16, width=1 << 18)


@pytest.mark.parametrize("dim", [64, 256])
def test_select_the_earlier_of_equal_scores(dev_ctx, dim):
    """Runs of pages with the same bounds: the first ones are in, over blocks of a cluster too."""
    pages, budget = 700, 100
    kv = make_cache(dev_ctx, "f32", 1, 1, dim, pages)
    table = torch.randperm(pages, device="cuda", generator=gen(3)).int()[None].contiguous()
    base = torch.randn(7, dim, device="cuda", generator=gen(4))
    k = base[torch.arange(pages, device="cuda") // 3 % 7][:, None].contiguous()
    kv.write(k, k, table, cu_tokens=ragged([pages]))
    summary = empty_summary(kv)
    kv.summarise(summary, table, tokens=pages, cu_tokens=ragged([pages]))
    q = torch.randn(1, 2, dim, device="cuda", generator=gen(5))
    codes, scales = bounds_of(kv, summary)
    ids = table[0].long()
    score = scores_plain(q[0].double(), codes[ids, 0], scales[ids, 0])
    for zero in (False, True):                     # and where every score is 0
        if zero:
            q.zero_()
            score = torch.zeros_like(score)
        selected, n = torch.zeros(1, 1, budget, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        kv.select(q, summary, table, torch.tensor([pages], dtype=torch.int32, device="cuda"), selected, n)
        dev_ctx.synchronize()
        want = ids[torch.tensor(select_plain(score, budget, 1, 1), device="cuda")].int()
        assert torch.equal(selected[0, 0], want)


def test_select_of_values_that_are_not_finite(dev_ctx):
    """A query head with an infinity or a NaN has no say; a page with one comes first; tiny and huge queries."""
    lengths, heads, group, dim, page, budget = [640], 1, 4, 64, 16, 10
    kv, table, summary, g = filled(dev_ctx, "f32", "f32", lengths, heads, dim, page)
    q0 = torch.randn(1, heads * group, dim, device="cuda", generator=g)
    for change in ("none", "inf", "nan", "all", "tiny", "huge"):
        q = q0.clone()
        if change == "inf":
            q[0, 1, 5] = -math.inf
        elif change == "nan":
            q[0, 2, 63] = math.nan
        elif change == "all":
            q[0, :, 0] = math.nan
        elif change == "tiny":
            q *= 1e-41
        elif change == "huge":
            q *= 1e37
        codes, scales = bounds_of(kv, summary)
        for page_inf in (False, True):
            if page_inf:
                scales = scales.clone()
                at = table[0, 20].long()
                summary[at, 2 * dim:2 * dim + 4] = torch.tensor([math.inf], device="cuda").view(torch.uint8)
                summary[at, :2 * dim] = 0
                codes, scales = bounds_of(kv, summary)
            ids = table[0].long()
            score = scores_plain(q[0].double(), codes[ids, 0], scales[ids, 0])
            selected, n = torch.zeros(1, 1, budget, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
            kv.select(q, summary, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), selected, n)
            dev_ctx.synchronize()
            chosen = select_plain(score, budget, 1, 1)
            assert torch.equal(selected[0, 0], ids[torch.tensor(chosen, device="cuda")].int()), (change, page_inf)
            # (Products of the huge query reach inf themselves, so earlier pages are alike.)
            assert not page_inf or 20 in chosen or (change == "huge" and score[chosen].eq(math.inf).sum() >= budget - 2)


def test_select_strides_offset_and_another_stream(sp):
    """Strided queries, lengths behind an offset, a context's own stream, and a captured call with new lengths."""
    ctx = sp.Context(num_threads=1)
    lengths, heads, group, dim, page, budget = [700, 350], 2, 2, 64, 16, 9
    kv, table, summary, g = filled(ctx, "bf16", "bf16", lengths, heads, dim, page)
    wide = torch.randn(2, heads * group, 2 * dim, device="cuda", generator=g).bfloat16()
    q = wide[..., dim:]
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = [torch.zeros(2, heads, budget, dtype=torch.int32, device="cuda") for _ in range(3)]
    got = [torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    kv.select(q, summary, table, n, out[0], got[0])
    m, q2 = n - 1, q.contiguous()
    torch.cuda.synchronize()
    kv.select(q2, summary, table, m, out[1], got[1], length_offset=1)
    ctx.synchronize()
    assert torch.equal(out[0], out[1]) and torch.equal(got[0], got[1])
    st = torch.cuda.Stream()
    ctx.set_stream(st.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        kv.summarise(summary, table, start=torch.zeros(2, dtype=torch.int32, device="cuda"))
        kv.select(q, summary, table, n, out[2], got[2])
    kv.summarise(summary, table, tokens=1050, cu_tokens=ragged(lengths))
    ctx.synchronize()
    n.copy_(torch.tensor([100, 0]))
    graph.replay()
    torch.cuda.synchronize()
    assert got[2].tolist() == [100, 0]
    assert torch.equal(out[2][0, :, :7], table[0, None, :7].expand(2, -1)) and (out[2][0, :, 7:] == -1).all() and (out[2][1] == -1).all()
    ctx.set_stream(0)
    del graph
    ctx.close()


def test_select_bad_places(sp, dev_ctx):
    """Pages outside the cache come last, lengths outside the table count as its ends; both are reported."""
    lengths, budget = [640, 640], 10
    kv, table, summary, g = filled(dev_ctx, "bf16", "bf16", lengths, 1, 64, 16)
    q = torch.randn(2, 2, 64, device="cuda", generator=g).bfloat16()

    def run(tab, lens):
        sel, n = torch.zeros(2, 1, budget, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        kv.select(q, summary, tab, torch.tensor(lens, dtype=torch.int32, device="cuda"), sel, n)
        return sel, n

    ref, ref_n = run(table, lengths)
    dev_ctx.synchronize()
    wrong = table.clone()
    wrong[1, 7], wrong[1, 8] = 1 << 30, -9
    sel, _ = run(wrong, lengths)
    with pytest.raises(sp.SapphireError, match="outside"):
        dev_ctx.synchronize()
    assert torch.equal(sel[0], ref[0]) and not ((sel[1] == 1 << 30) | (sel[1] == -9)).any()
    sel, n = run(table, [641, -3])
    with pytest.raises(sp.SapphireError, match="outside"):
        dev_ctx.synchronize()
    assert torch.equal(sel[0], ref[0]) and n.tolist() == [int(ref_n[0]), 0] and (sel[1] == -1).all()


# --------------------------------------------------- attention over the pages --
@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("kind,group,dim,page", [("bf16", 4, 128, 16), ("f16", 1, 64, 24), ("f32", 6, 256, 8), ("bf16", 12, 96, 5)])
def test_steps_over_selected_pages(dev_ctx, dtype, kind, group, dim, page):
    """A prompt, then steps that write, summarise, select and attend; each against attention over the selected pages."""
    heads, budget = 2, 6
    lengths = [page * 21 + 3, 1, page * 3, page * 11]
    kv, table, summary, g = filled(dev_ctx, dtype, kind, lengths, heads, dim, page, seed=9, width=30)
    used = set(table[table >= 0].tolist())
    free = [i for i in range(kv.pages.shape[0]) if i not in used]
    selected = torch.zeros(4, heads, budget, dtype=torch.int32, device="cuda")
    n = torch.zeros(4, dtype=torch.int32, device="cuda")
    for step in range(3):
        start = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        for s, m in enumerate(lengths):
            if m % page == 0 and table[s, m // page] < 0:
                if not free:
                    return
                table[s, m // page] = free.pop()
        k, v = (torch.randn(4, heads, dim, device="cuda", generator=g).to(IO[kind]) for _ in (0, 1))
        q = torch.randn(4, heads * group, dim, device="cuda", generator=g).to(IO[kind])
        out, lse = torch.full_like(q, 9.0), torch.empty(4, heads * group, device="cuda")
        kv.write(k, v, table, start=start)
        kv.summarise(summary, table, start=start)
        kv.select(q, summary, table, start, selected, n, first=1, last=2, length_offset=1)
        kv.attend(q, selected, n, out, lse=lse)
        dev_ctx.synchronize()
        lengths = [m + 1 for m in lengths]
        check_bounds(kv, summary, table, lengths, dtype)
        for h in range(heads):
            at = slice(h * group, (h + 1) * group)
            full = q.clone()                       # every KV head against this one's table
            want, bound, want_lse, lse_bound = attend_plain(kv, full, selected[:, h].contiguous(), n.tolist(), page, heads, dim, dtype)
            assert_within(out[:, at], want[:, at], bound[:, at])
            assert_within(lse[:, at], want_lse[:, at], lse_bound[:, at])


def test_tables_of_their_own_that_are_alike(dev_ctx):
    """A table per KV head that repeats one table gives the bits of that table."""
    lengths = [1000, 0, 333, 70]
    for dtype in CACHES:
        kv, table, _, g = filled(dev_ctx, dtype, "bf16", lengths, 3, 128, 16, seed=2)
        q = torch.randn(4, 12, 128, device="cuda", generator=g).bfloat16()
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = [torch.empty_like(q) for _ in (0, 1)]
        kv.attend(q, table, n, out[0], window=300)
        kv.attend(q, table[:, None].expand(-1, 3, -1).contiguous(), n, out[1], window=300)
        dev_ctx.synchronize()
        assert torch.equal(out[0], out[1])


def test_selection_refusals(sp, dev_ctx):
    kv, table, summary, g = filled(dev_ctx, "bf16", "bf16", [64, 64], 2, 64, 16)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    n = torch.tensor([64, 64], dtype=torch.int32, device="cuda")
    sel = torch.zeros(2, 2, 3, dtype=torch.int32, device="cuda")
    got = torch.zeros(2, dtype=torch.int32, device="cuda")
    for args, kw, match in (((q[:, :3], summary, table, n, sel, got), {}, "query heads"),
                            ((q, summary[:, :16], table, n, sel, got), {}, "summary"),
                            ((q, summary.float(), table, n, sel, got), {}, "summary"),
                            ((q, summary, table[:1], n, sel, got), {}, "shape"), ((q, summary, table, n[:1], sel, got), {}, "shape"),
                            ((q, summary, table, n, sel[:, 0], got), {}, "shape"), ((q, summary, table, n, sel[:, :1], got), {}, "shape"),
                            ((q, summary, table, n, sel.long(), got), {}, "int32"), ((q, summary, table, n, sel[..., :2], got), {}, "contiguous"),
                            ((q, summary, table, n, sel, got.long()), {}, "int32"), ((q, summary, table, n, sel, got[:1]), {}, "shape"),
                            ((q, summary, table, n, sel, got), {"first": 3}, "budget"), ((q, summary, table, n, sel, got), {"last": 0}, "budget"),
                            ((q, summary, table, n, sel, got), {"first": -1}, "budget"),
                            ((q.cpu(), summary, table, n, sel, got), {}, "device memory"), ((q, summary.cpu(), table, n, sel, got), {}, "device memory"),
                            ((q, summary, table, n, sel, got.cpu()), {}, "device memory"), ((q.double(), summary, table, n, sel, got), {}, "float32"),
                            ((q.repeat(1, 65, 1), summary, table, n, sel, got), {}, "query heads"),
                            ((q, summary, torch.zeros(2, (1 << 18) + 1, dtype=torch.int32, device="cuda"), n, sel, got), {}, "table_stride")):
        with pytest.raises(sp.SapphireError, match=match):
            kv.select(*args, **kw)
    for kw, match in (({"tokens": 3}, "tokens"), ({"cu_tokens": ragged([1, 1])}, "tokens"), ({"start": n[:1]}, "shape")):
        with pytest.raises(sp.SapphireError, match=match):
            kv.summarise(summary, table, **kw)
    with pytest.raises(sp.SapphireError, match="shape"):
        kv.attend(q, sel[:, :1], got, torch.empty_like(q))
    with pytest.raises(sp.SapphireError, match="contiguous"):
        kv.attend(q, sel[..., :2], got, torch.empty_like(q))
    kv.select(q[:0], summary, table[:0], n[:0], sel[:0], got[:0])
    kv.summarise(summary, table[:0])
    dev_ctx.synchronize()

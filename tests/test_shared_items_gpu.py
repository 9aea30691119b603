"""Attention behind a shared prefix where a block of its product takes several items
(KV heads, or sets of rows) one behind another, each with scores of its own size.

Keys and values are such that nothing but probabilities is rounded: bf16 values in every
dense cache, codes times one power of two in a quantised one.  So the bounds are those of
test_shared_prefix_gpu without what conversion costs there: a score is off by ds = scale
sum|q k| 2^-19, out by A (4 ds + 2^-14 + 2^-8) with A = sum p |v| (probabilities in bf16,
else 2^-11), and lse by 2 ds + 2^-15.  Nothing lies behind the prefix but where a case
says so.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_attention_gpu import IO, assert_within, dev_ctx, gen, layout, make_cache, ragged  # noqa: E402,F401
from test_prefix_ranges_cpu import items_of_blocks  # noqa: E402

DIM, TILE, PAGE, PREFIX = 64, 128, 16, 2100


def write_exact(kv, dtype, kind, table, k, v):
    """k and v [tokens, heads, DIM], bf16 values (codes of -8 .. 7 where quantised), into the cache."""
    tokens, heads = k.shape[:2]
    if dtype in IO:
        kv.write(k.to(IO[kind]), v.to(IO[kind]), table[None].contiguous(), cu_tokens=ragged([tokens]))
        return
    row, ns, at, chunk = layout(dtype, DIM, PAGE)
    pages = kv.pages.view(-1, heads, chunk)
    for j, x in enumerate((k, v)):
        x = x.reshape(-1, PAGE, heads, DIM).transpose(1, 2) if tokens % PAGE == 0 else None
        codes = (x + (128 if dtype == "q8_0" else 8)).to(torch.uint8).unflatten(-1, (DIM // 32, 8, 4)).transpose(-3, -2).flatten(-3)
        if dtype == "q4_0":
            codes = codes[..., ::2] | codes[..., 1::2] << 4
        pages[table.long(), :, at[j]:at[j] + PAGE * row] = codes.flatten(-2)
        scales = torch.ones(*x.shape[:2], PAGE, ns, device="cuda")
        pages[table.long(), :, at[2 + j]:at[2 + j] + 4 * PAGE * ns] = scales.flatten(-2).view(torch.uint8)


def values(g, dtype, tokens, heads):
    """Keys whose first two dims are 0, and values, exact in every type on the way."""
    if dtype in IO:
        k, v = (torch.randn(tokens, heads, DIM, device="cuda", generator=g).bfloat16().float() for _ in (0, 1))
    else:
        lo, hi = (-127, 128) if dtype == "q8_0" else (-8, 8)
        k = torch.randint(-3, 4, (tokens, heads, DIM), device="cuda", generator=g).float()
        v = torch.randint(lo, hi, (tokens, heads, DIM), device="cuda", generator=g).float()
    k[..., :2] = 0
    return k, v


def plain(q, k, v, dtype):
    """fp64 out, its bound, lse and its bound; q [seqs, heads * group, DIM], k and v [tokens, heads, DIM]."""
    heads, group = k.shape[1], q.shape[1] // k.shape[1]
    x = q.double().unflatten(1, (heads, group))
    score = torch.einsum("shgd,thd->shgt", x, k.double()) * DIM ** -0.5
    ds = torch.einsum("shgd,thd->shgt", x.abs(), k.double().abs()).amax(-1) * DIM ** -0.5 * 2.0 ** -19
    p = torch.softmax(score, -1)
    rel = 2.0 ** -14 + (2.0 ** -8 if dtype == "bf16" and q.dtype == torch.bfloat16 else 2.0 ** -11)
    out = torch.einsum("shgt,thd->shgd", p, v.double())
    bound = torch.einsum("shgt,thd->shgd", p, v.double().abs()) * (4 * ds[..., None] + rel)
    return out.flatten(1, 2), bound.flatten(1, 2), torch.logsumexp(score, -1).flatten(1, 2), (2 * ds + 2.0 ** -15).flatten(1, 2)


def attend(ctx, kv, table, q, tokens, own=None, n=None):
    seqs = q.shape[0]
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    own = torch.zeros(seqs, 1, dtype=torch.int32, device="cuda") if own is None else own
    n = torch.zeros(seqs, dtype=torch.int32, device="cuda") if n is None else n
    kv.attend_shared(q, table, torch.tensor([tokens], dtype=torch.int32, device="cuda"), own, n, out, lse=lse)
    ctx.synchronize()
    return out, lse


def neighbours(tmp_path, heads, row_sets, tokens):
    """The pairs of items (KV head, set of rows) that a block takes one behind the other."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    pairs = [(a, b) for x in items_of_blocks(tmp_path, heads * row_sets, tokens, TILE, sms) for a, b in zip(x, x[1:])]
    return {(a // row_sets, b // row_sets) for a, b in pairs}


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("f16", "f16"), ("q8_0", "bf16"), ("f32", "bf16"), ("q4_0", "f16")])
@pytest.mark.parametrize("heads", [100, 200])
@pytest.mark.parametrize("gap", [110, 126, 400])
def test_heads_of_far_apart_scores(dev_ctx, tmp_path, dtype, kind, heads, gap):
    """Every other KV head's scores are 159, 182 or 577 units of log2 e above its neighbours'."""
    pairs = neighbours(tmp_path, heads, 1, PREFIX)
    assert sum(a % 2 == 0 for a, b in pairs) > 20 and sum(a % 2 == 1 for a, b in pairs) > 20
    g = gen(heads + gap)
    tokens = -(-PREFIX // PAGE) * PAGE
    k, v = values(g, dtype, tokens, heads)
    # A score is q k / 8 from the first two dims: q = 64 and so 8 k.
    q = torch.randn(2, heads, DIM, device="cuda", generator=g).to(IO[kind])
    q[..., 0] = q[..., 1] = 64
    for j, part in ((0, gap // 16), (1, gap / 8 - gap // 16)):
        k[:, ::2, j] = part if dtype in IO else 0
    if dtype not in IO:                   # (codes are whole and small: a larger query instead)
        k[:, ::2, 0] = 2
        q[..., 0] = gap * 4
    table = torch.randperm(tokens // PAGE, device="cuda", generator=g).int()
    kv = make_cache(dev_ctx, dtype, PAGE, heads, DIM, tokens // PAGE)
    write_exact(kv, dtype, kind, table, k, v)
    out, lse = attend(dev_ctx, kv, table, q, PREFIX)
    want, bound, want_lse, lse_bound = plain(q, k[:PREFIX], v[:PREFIX], dtype)
    assert (want_lse[:, ::2].amin() - want_lse[:, 1::2].amax()).item() > gap - 30
    assert_within(lse, want_lse, lse_bound)
    assert_within(out, want, bound)


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("f16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("parity", [0, 1])
def test_an_infinite_key_stays_in_its_head(dev_ctx, tmp_path, dtype, kind, parity):
    """A key that is infinite for every other KV head takes nothing from the heads between."""
    heads = 100
    pairs = neighbours(tmp_path, heads, 1, PREFIX)
    assert sum(a % 2 == parity for a, b in pairs) > 20
    g = gen(5)
    tokens = -(-PREFIX // PAGE) * PAGE
    k, v = values(g, dtype, tokens, heads)
    q = torch.randn(1, heads, DIM, device="cuda", generator=g).to(IO[kind])
    q[..., 1] = 1
    table = torch.randperm(tokens // PAGE, device="cuda", generator=g).int()
    kv = make_cache(dev_ctx, dtype, PAGE, heads, DIM, tokens // PAGE)
    k[::7, parity::2, 1] = math.inf
    write_exact(kv, dtype, kind, table, k, v)
    out, lse = attend(dev_ctx, kv, table, q, PREFIX)
    clean = slice(1 - parity, None, 2)
    want, bound, want_lse, lse_bound = plain(q[:, clean], k[:PREFIX, clean], v[:PREFIX, clean], dtype)
    assert_within(lse[:, clean], want_lse, lse_bound)
    assert_within(out[:, clean], want, bound)
    assert not torch.isfinite(out[:, parity::2].float()).any()


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("q8_0", "f16")])
def test_rows_of_far_apart_scores(dev_ctx, tmp_path, dtype, kind):
    """Sets of rows of one KV head whose queries are loud in one set and quiet in the next."""
    heads, seqs = 60, 520                 # three sets of two tiles of rows, the last with 8 rows
    pairs = neighbours(tmp_path, heads, 3, PREFIX)
    assert len(pairs) > 20
    g = gen(9)
    tokens = -(-PREFIX // PAGE) * PAGE
    k, v = values(g, dtype, tokens, heads)
    q = torch.randn(seqs, heads, DIM, device="cuda", generator=g).to(IO[kind])
    q[..., 0] = 0
    k[..., 0] = 2
    loud = [slice(0, 256), slice(256, 512), slice(512, 520)]
    for order in ((1, 0, 1), (0, 1, 0)):
        for rows, on in zip(loud, order):
            q[rows, :, 0] = 600 * on      # 150 in all, 216 units of log2 e
        table = torch.randperm(tokens // PAGE, device="cuda", generator=g).int()
        kv = make_cache(dev_ctx, dtype, PAGE, heads, DIM, tokens // PAGE)
        write_exact(kv, dtype, kind, table, k, v)
        out, lse = attend(dev_ctx, kv, table, q, PREFIX)
        for at in range(0, seqs, 40):
            want, bound, want_lse, lse_bound = plain(q[at:at + 40], k[:PREFIX], v[:PREFIX], dtype)
            assert_within(lse[at:at + 40], want_lse, lse_bound)
            assert_within(out[at:at + 40], want, bound)


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("q8_0", "f16")])
def test_own_tokens_count_beside_a_quiet_second_item(dev_ctx, tmp_path, dtype, kind):
    """What a sequence has behind the prefix keeps its weight beside a prefix read after a louder head's."""
    heads = 100
    assert sum(a % 2 == 0 for a, b in neighbours(tmp_path, heads, 1, PREFIX)) > 20
    g = gen(11)
    tokens = -(-PREFIX // PAGE) * PAGE + PAGE         # the last page is the sequence's own
    k, v = values(g, dtype, tokens, heads)
    k[:, ::2, 0] = 2
    q = torch.randn(1, heads, DIM, device="cuda", generator=g).to(IO[kind])
    q[..., 0] = 440                                   # 110
    table = torch.randperm(tokens // PAGE, device="cuda", generator=g).int()
    kv = make_cache(dev_ctx, dtype, PAGE, heads, DIM, tokens // PAGE)
    write_exact(kv, dtype, kind, table, k, v)
    own = table[-1:].view(1, 1).contiguous()
    n = torch.tensor([5], dtype=torch.int32, device="cuda")
    out, lse = attend(dev_ctx, kv, table[:-1].contiguous(), q, PREFIX, own, n)
    used = torch.cat((torch.arange(PREFIX), torch.arange(tokens - PAGE, tokens - PAGE + 5))).cuda()
    want, bound, want_lse, lse_bound = plain(q, k[used], v[used], dtype)
    assert_within(lse, want_lse, lse_bound)
    assert_within(out, want, bound)

"""Rotary positions, the paged key-value cache and attention of one new token
against plain 64-bit forms.

Tolerances.  A rounding is off by at most half a step, eps(t) / 2 of the value
(fp16 below 2^-14: 2^-25).

rope: the phase is good to 2^-32 of a turn, its fp32 half turns to 2^-25 and
sincospi to 2 ulp, so cos and sin are off by at most pi 2^-25 + 2^-22 < 2^-21.4
(times the amplitude, itself rounded); the products and the sum round three
times.  A turned value is off by at most (|a| + |b|) m 2^-21 before its own
rounding.

attend: q, k and p are held to at least 21 bits, sums in fp32 over at most
2^12 terms per partial sum (tests are smaller), so a score is off by at most
ds = scale sum|q k| 2^-19; p is off by a factor of exp(+-2 ds) (1 + 2^-18) with
the approximate exponential (2^-21), and so out by at most
max|v| (4 ds + 2^-17) before its rounding.

Quantised caches under bf16 queries multiply the query as integers: a value is off
by at most half of max|q| 2^-13, so ds grows by scale max|q| sum|k| 2^-14.  These
and fp16 caches under bf16 queries round a probability to fp16 once, 2^-12 of it,
so out is off by 2^-12 max|v| more.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CACHES = ["f32", "bf16", "f16", "q8_0", "q4_0"]


def half_step(t, y):
    """Half a step of type t at y (fp64)."""
    return y.abs() * (torch.finfo(t).eps / 2) + (2.0 ** -25 if t == torch.float16 else 0.0)


def assert_within(got, want, before, what=""):
    """got (type t) is want (fp64) off by at most `before` and one rounding."""
    tol = before + half_step(got.dtype, want.abs() + before) * (1 if got.dtype != torch.float32 else 1)
    bad = (got.double() - want).abs() - tol
    assert torch.isfinite(got.double()).all(), what
    assert bad.max().item() <= 0, f"{what}: over by {bad.max().item():.3g}, want {want.flatten()[bad.argmax()].item():.6g}"


@pytest.fixture
def dev_ctx(sp):
    """A context on torch's current stream."""
    c = sp.Context(num_threads=1)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# --------------------------------------------------------------------- rope --
def rope_frequencies(rot, theta, scaling, factor, orig=8192):
    i = np.arange(rot // 2, dtype=np.float64)
    f = theta ** (-2 * i / rot)
    m = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "banded":
        r = orig * f / (2 * np.pi)
        s = np.clip((r - 1) / 3, 0, 1)
        f = (1 - s) * f / factor + s * f
    elif scaling == "yarn":
        c = lambda r: rot * math.log(orig / (2 * math.pi * r)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(c(32.0)), 0), min(math.ceil(c(1.0)), rot - 1)
        g = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        f = (1 - g) * f + g * f / factor
        m = 0.1 * math.log(factor) + 1
    return torch.from_numpy(f).cuda(), m


def rope_plain(x, pos, rot, layout, theta=1e4, scaling="none", factor=1.0, inverse=False):
    """fp64 result and the error bound before rounding."""
    f, m = rope_frequencies(rot, theta, scaling, factor)
    a = pos.double()[:, None, None] * f
    if inverse:
        a = -a
    y, e = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    at = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    u, v = y[..., at[0]].clone(), y[..., at[1]].clone()
    y[..., at[0]], y[..., at[1]] = (u * a.cos() - v * a.sin()) * m, (u * a.sin() + v * a.cos()) * m
    e[..., at[0]] = e[..., at[1]] = (u.abs() + v.abs()) * m * 2.0 ** -21
    return y, e


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot,layout,kind,scaling", [
    (1, 4, 1, 256, 256, "half", "f32", "none"),
    (1, 1, 0, 2, 2, "interleaved", "f32", "none"),
    (5, 3, 1, 64, 64, "half", "bf16", "linear"),
    (7, 5, 5, 80, 40, "half", "f16", "none"),
    (7, 5, 5, 80, 40, "interleaved", "f16", "yarn"),
    (33, 32, 8, 128, 128, "half", "bf16", "banded"),
    (33, 32, 8, 128, 64, "interleaved", "bf16", "yarn"),
    (130, 6, 2, 96, 22, "half", "f32", "banded"),
    (130, 6, 2, 96, 22, "interleaved", "f32", "linear"),
    (1000, 2, 1, 512, 512, "half", "f16", "yarn"),
    (601, 40, 0, 18, 18, "interleaved", "bf16", "none"),
])
def test_rope(dev_ctx, tokens, heads, kv_heads, dim, rot, layout, kind, scaling):
    from sapphire_b200.attention import Rope
    g = gen(tokens)
    pos = torch.randint(0, 131072, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    pos[0] = 0 if tokens > 1 else 777
    q = torch.randn(tokens, heads, dim, device="cuda", generator=g).to(IO[kind])
    k = torch.randn(tokens, kv_heads, dim, device="cuda", generator=g).to(IO[kind]) if kv_heads else None
    r = Rope(dev_ctx, dim, rot_dim=rot, layout=layout, theta=5e5, scaling=scaling, factor=4.0, original_context=8192)
    q_out = torch.full_like(q, 9.0)
    k_out = torch.full_like(k, 9.0) if k is not None else None
    r.apply(pos, q, k, q_out, k_out)
    dev_ctx.synchronize()
    for x, y in ((q, q_out), (k, k_out)):
        if x is None:
            continue
        want, e = rope_plain(x, pos, rot, layout, 5e5, scaling, 4.0)
        assert_within(y, want, e)
        assert torch.equal(y[..., rot:], x[..., rot:])
    r.close()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot", [(300, 16, 4, 80, 40), (9, 3, 1, 90, 88), (65, 2, 2, 512, 8),
                                                          (4991, 1, 1, 24, 24), (1, 5, 0, 510, 504)])
def test_rope_halves_of_four(dev_ctx, kind, tokens, heads, kv_heads, dim, rot):
    """Halves of a multiple of 4 values that is none of 8."""
    test_rope(dev_ctx, tokens, heads, kv_heads, dim, rot, "half", kind, "banded")


def test_rope_far_positions(dev_ctx):
    """Every 32-bit position, behind zero too."""
    from sapphire_b200.attention import Rope
    pos = torch.tensor([0, 1, -1, 2 ** 24 + 1, 10 ** 9 + 7, 2 ** 31 - 1, -2 ** 31], device="cuda", dtype=torch.int32)
    q = torch.randn(7, 2, 64, device="cuda", generator=gen(3))
    out = torch.empty_like(q)
    Rope(dev_ctx, 64).apply(pos, q, q_out=out)
    dev_ctx.synchronize()
    # fp64 angles: 2^31 * 2^-53 = 2^-22 rad; the frequency's own rounding of 2^-53 the same again
    want, e = rope_plain(q, pos, 64, "half")
    assert_within(out, want, e + q.abs().max().item() * 2.0 ** -20)


def test_rope_in_place_strided_and_back(dev_ctx):
    from sapphire_b200.attention import Rope
    qkv = torch.randn(9, 10, 128, device="cuda", generator=gen(4)).bfloat16()
    before = qkv.clone()
    pos = torch.arange(9, device="cuda", dtype=torch.int32) * 100
    r = Rope(dev_ctx, 128, rot_dim=64)
    q, k = qkv[:, :6], qkv[:, 6:8]
    r.apply(pos, q, k)
    dev_ctx.synchronize()
    for x, y in ((before[:, :6], q), (before[:, 6:8], k)):
        want, e = rope_plain(x, pos, 64, "half")
        assert_within(y, want, e)
    assert torch.equal(qkv[:, 8:], before[:, 8:])
    # rows that do not start on 16 bytes
    odd = torch.randn(9, 3 * 128 + 5, device="cuda", generator=gen(5)).bfloat16()
    x = odd[:, 1:1 + 3 * 128].unflatten(1, (3, 128))
    y = torch.empty(9, 3, 128, device="cuda", dtype=torch.bfloat16)
    r.apply(pos, q=x, q_out=y)
    dev_ctx.synchronize()
    want, e = rope_plain(x, pos, 64, "half")
    assert_within(y, want, e)
    # the inverse of the turned values, in fp32, gives them back
    f = torch.randn(9, 3, 128, device="cuda", generator=gen(6))
    z = f.clone()
    r.apply(pos, k=z)
    r.apply(pos, k=z, inverse=True)
    dev_ctx.synchronize()
    assert (z - f).abs().max().item() <= 4 * f.abs().max().item() * 2.0 ** -21 * 2


def test_rope_gradient(dev_ctx):
    """The inverse turn is the gradient: against the formula's and against differences."""
    from sapphire_b200.attention import Rope
    g = gen(8)
    pos = torch.randint(0, 5000, (6,), device="cuda", generator=g, dtype=torch.int32)
    x = torch.randn(6, 2, 64, device="cuda", generator=g)
    dy = torch.randn(6, 2, 64, device="cuda", generator=g)
    r = Rope(dev_ctx, 64, rot_dim=48, layout="interleaved", scaling="yarn", factor=4.0, original_context=8192)
    dx = torch.empty_like(x)
    r.apply(pos, q=dy, q_out=dx, inverse=True)
    dev_ctx.synchronize()
    want, e = rope_plain(dy, pos, 48, "interleaved", scaling="yarn", factor=4.0, inverse=True)
    assert_within(dx, want, e)
    u = torch.randn(6, 2, 64, device="cuda", generator=g, dtype=torch.float64)
    f = lambda v: (rope_plain(v, pos, 48, "interleaved", scaling="yarn", factor=4.0)[0] * dy.double()).sum()  # noqa: E731
    diff = (f(x.double() + 1e-3 * u) - f(x.double() - 1e-3 * u)) / 2e-3
    # the turn is linear: differences are exact but for the kernel's own error
    assert abs(diff.item() - (dx.double() * u).sum().item()) <= (e.sum() * u.abs().max()).item() + 1e-6


def test_rope_refusals(sp, dev_ctx):
    from sapphire_b200.attention import Rope
    r = Rope(dev_ctx, 64)
    q = torch.zeros(4, 2, 64, device="cuda")
    pos = torch.zeros(4, device="cuda", dtype=torch.int32)
    with pytest.raises(sp.SapphireError, match="int32"):
        r.apply(pos.long(), q)
    with pytest.raises(sp.SapphireError, match="shape"):
        r.apply(pos[:3], q)
    with pytest.raises(sp.SapphireError, match="float32"):
        r.apply(pos, q.double())
    with pytest.raises(sp.SapphireError, match="one type"):
        r.apply(pos, q, q.bfloat16())
    with pytest.raises(sp.SapphireError, match="shape"):
        r.apply(pos, torch.zeros(4, 2, 32, device="cuda"))
    with pytest.raises(sp.SapphireError, match="contiguous"):
        r.apply(pos, torch.zeros(4, 64, 2, device="cuda").transpose(1, 2))
    with pytest.raises(sp.SapphireError, match="broadcast"):
        r.apply(pos, torch.zeros(1, 2, 64, device="cuda").expand(4, 2, 64))
    with pytest.raises(sp.SapphireError, match="device memory"):
        r.apply(pos, q.cpu())
    with pytest.raises(sp.SapphireError, match="device memory"):
        r.apply(pos.cpu(), q)
    with pytest.raises(sp.SapphireError, match="in place"):
        r.apply(pos, q[:, :1], q_out=torch.as_strided(q, (4, 1, 64), (64, 64, 1)))
    r.apply(pos[:0], q[:0])
    dev_ctx.synchronize()


# -------------------------------------------------------------------- cache --
def layout(dtype, dim, page):
    """(row bytes, padded scales, offsets of K, V, K scales, V scales, chunk bytes)."""
    nb = dim // 32
    row = {"f32": 4 * dim, "bf16": 2 * dim, "f16": 2 * dim, "q8_0": dim, "q4_0": dim // 2}[dtype]
    ns = (2 if nb <= 2 else 4 if nb <= 4 else 8) if dtype[0] == "q" else 0
    at = [0, page * row, 2 * page * row, 2 * page * row + 4 * page * ns]
    return row, ns, at, at[3] + 4 * page * ns


def cache_values(pages, dtype, page, heads, dim, j):
    """fp64 [pages, heads, page, dim] of the K (0) or V (1) rows; quantised rows as code * scale."""
    row, ns, at, chunk = layout(dtype, dim, page)
    p = pages.reshape(-1, heads, chunk)
    rows = p[..., at[j]:at[j] + page * row].reshape(-1, heads, page, row)
    if not ns:
        return rows.contiguous().view(IO[dtype]).double()
    nb = dim // 32
    if dtype == "q4_0":
        rows = torch.stack((rows & 15, rows >> 4), -1).flatten(-2)
    codes = rows.reshape(*rows.shape[:-1], 8, nb, 4).transpose(-3, -2).flatten(-2).double() - (128 if dtype == "q8_0" else 8)
    sc = p[..., at[2 + j]:at[2 + j] + 4 * ns * page].contiguous().view(torch.float32).reshape(-1, heads, page, ns)
    return (codes * sc[..., :nb, None].double()).flatten(-2)


def make_cache(ctx, dtype, page, heads, dim, num_pages, fill=0):
    from sapphire_b200.attention import KVCache, kv_page_bytes
    pages = torch.full((num_pages, kv_page_bytes(dtype, page, heads, dim)), fill, dtype=torch.uint8, device="cuda")
    return KVCache(ctx, dtype, page, heads, dim, pages)


def make_table(lengths, page, num_pages, g, width=None):
    """Random pages for sequences of these lengths; unused entries -1."""
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(num_pages, device="cuda", generator=g)[:sum(need)].cpu().int()
    t = torch.full((len(lengths), width or max(1, max(need))), -1, dtype=torch.int32)
    a = 0
    for i, m in enumerate(need):
        t[i, :m] = order[a:a + m]
        a += m
    return t.cuda()


def ragged(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def expected_store(sp, ctx, x, dtype):
    """fp64 values that the cache should hold of x, quantised by the library's quantiser."""
    if dtype in IO:
        return x.to(IO[dtype]).double()
    code = sp.DTYPE_Q8_0 if dtype == "q8_0" else sp.DTYPE_Q4_0
    flat = np.ascontiguousarray(x.float().cpu().numpy().reshape(-1, x.shape[-1]))
    packed = sp.quantize(ctx, code, flat)
    t = sp.Tensor(code, flat.shape, packed)
    size = 36 if dtype == "q8_0" else 20
    blocks = packed.reshape(-1, size)
    scale = blocks[:, :4].copy().view(np.float32).astype(np.float64)
    body = blocks[:, 4:]
    codes = body.view(np.int8).astype(np.float64) if dtype == "q8_0" else \
        np.stack((body & 15, body >> 4), -1).reshape(len(blocks), 32).astype(np.float64) - 8
    t.release()
    return torch.from_numpy((codes * scale).reshape(x.shape)).cuda()


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("kind,dim,page,heads", [("bf16", 128, 16, 8), ("f32", 256, 7, 1), ("f16", 96, 1, 3),
                                                 ("bf16", 64, 100, 2), ("f32", 192, 24, 5)])
def test_write_and_read(sp, dev_ctx, ctx, dtype, kind, dim, page, heads):
    """Ragged chunks behind what was there, rows that belong to no sequence,
    values stored as the library's quantisers store them, and read back."""
    g = gen(dim + page)
    before, new = [0, 3, 2 * page, 5], [11, 0, page + 1, 2]
    total = [a + b for a, b in zip(before, new)]
    pages = sum(-(-n // page) for n in total) + 2
    kv = make_cache(dev_ctx, dtype, page, heads, dim, pages, fill=0xA5)
    table = make_table(total, page, pages, g)
    rows = sum(new) + 3
    k = torch.randn(rows, heads, dim, device="cuda", generator=g)
    k[1] = 0.0                                            # scale 0
    k[2, :, 3] = -k[2, :, 7].abs().clamp(min=4.0)         # a tie in magnitude, the negative one first
    k[2, :, 7] = -k[2, :, 3]
    k[3] *= 1e-30
    k, v = k.to(IO[kind]), torch.randn(rows, heads, dim, device="cuda", generator=g).to(IO[kind])
    old = kv.pages.clone()
    start = torch.tensor(before, dtype=torch.int32, device="cuda")
    kv.write(k, v, table, start=start, cu_tokens=ragged(new))
    dev_ctx.synchronize()
    # place of every stored token
    where, row = [], 0
    for s, (b, m) in enumerate(zip(before, new)):
        for j in range(m):
            where.append((row, int(table[s, (b + j) // page]), (b + j) % page))
            row += 1
    r, pg, slot = (torch.tensor(c, device="cuda") for c in zip(*where))
    for j, x in ((0, k), (1, v)):
        got = cache_values(kv.pages, dtype, page, heads, dim, j)[pg, :, slot]
        assert torch.equal(got, expected_store(sp, ctx, x, dtype)[r])
    # nothing else changed: put the written slots' old bytes back and compare
    rb, ns, at, chunk = layout(dtype, dim, page)
    a, b = (t.reshape(-1, heads, chunk).clone() for t in (kv.pages, old))
    for _, p_, s_ in where:
        for o, n in ((at[0] + s_ * rb, rb), (at[1] + s_ * rb, rb), (at[2] + 4 * s_ * ns, 4 * (dim // 32) * (ns > 0)),
                     (at[3] + 4 * s_ * ns, 4 * (dim // 32) * (ns > 0))):
            a[p_, :, o:o + n] = 0
            b[p_, :, o:o + n] = 0
    assert torch.equal(a, b)
    # read back: one fp32 product, rounded once
    ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    kv.read(ko, vo, table, start=start, cu_tokens=ragged(new))
    dev_ctx.synchronize()
    for j, out in ((0, ko), (1, vo)):
        want = cache_values(kv.pages, dtype, page, heads, dim, j)[pg, :, slot].float().to(IO[kind])
        assert torch.equal(out[:sum(new)], want)
        assert (out[sum(new):] == 7.0).all()


@pytest.mark.parametrize("dtype", CACHES)
def test_one_token_each_strided(sp, dev_ctx, ctx, dtype):
    """A decoding step out of a fused projection, rows not on 16 bytes."""
    g = gen(5)
    lens, page, heads, dim = [0, 15, 16, 40], 16, 2, 64
    kv = make_cache(dev_ctx, dtype, page, heads, dim, 12)
    table = make_table([n + 1 for n in lens], page, 12, g)
    buf = torch.randn(4, 6 * dim + 3, device="cuda", generator=g).bfloat16()
    k = buf[:, 1:1 + 2 * dim].unflatten(1, (2, dim))
    v = buf[:, 3 + 4 * dim:3 + 6 * dim].unflatten(1, (2, dim))
    start = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kv.write(k, v, table, start=start)
    ko, vo = torch.empty(4, 2, dim, device="cuda"), torch.empty(4, 2, dim, device="cuda")
    kv.read(ko, vo, table, start=start)
    dev_ctx.synchronize()
    assert torch.equal(ko, expected_store(sp, ctx, k, dtype).float())
    assert torch.equal(vo, expected_store(sp, ctx, v, dtype).float())


def test_nan_and_infinity_quantise_as_documented(sp, dev_ctx, ctx):
    for dtype in ("q8_0", "q4_0"):
        x = torch.randn(2, 1, 64, device="cuda", generator=gen(9))
        x[0, 0, 3], x[0, 0, 40], x[1, 0, 5] = math.nan, -math.inf, math.inf
        kv = make_cache(dev_ctx, dtype, 4, 1, 64, 2)
        table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
        kv.write(x, x, table)
        dev_ctx.synchronize()
        got = cache_values(kv.pages, dtype, 4, 1, 64, 0)[:, :, 0]
        want = expected_store(sp, ctx, x, dtype)
        assert torch.equal(torch.nan_to_num(got, 7.0, 8.0, 9.0), torch.nan_to_num(want, 7.0, 8.0, 9.0))


def test_bad_places_are_skipped_and_reported(sp, dev_ctx):
    kv = make_cache(dev_ctx, "bf16", 4, 1, 64, 3, fill=0)
    x = torch.ones(4, 1, 64, device="cuda", dtype=torch.bfloat16)
    table = torch.tensor([[0, 1], [3, 1], [-1, 1], [2, 2]], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 0, 0, 8], dtype=torch.int32, device="cuda")
    kv.write(x, x, table, start=start)
    with pytest.raises(sp.SapphireError, match="paged key-value cache"):
        dev_ctx.synchronize()
    got = cache_values(kv.pages, "bf16", 4, 1, 64, 0)
    assert got[0, 0, 0].eq(1).all() and got.sum().item() == 64
    out = torch.full_like(x, 5.0)
    kv.read(out, out.clone(), table, start=start)
    with pytest.raises(sp.SapphireError, match="paged key-value cache"):
        dev_ctx.synchronize()
    assert out[0].eq(1).all() and out[1:].eq(5).all()
    start[3] = -1
    kv.write(x[3:], x[3:], table[3:], start=start[3:])
    with pytest.raises(sp.SapphireError, match="paged key-value cache"):
        dev_ctx.synchronize()
    kv.write(x[:1], x[:1], table[:1])                # the context works on
    dev_ctx.synchronize()


def test_cache_refusals(sp, dev_ctx):
    from sapphire_b200.attention import KVCache
    kv = make_cache(dev_ctx, "q8_0", 4, 2, 64, 3)
    x = torch.zeros(2, 2, 64, device="cuda")
    table = torch.zeros(2, 1, device="cuda", dtype=torch.int32)
    for bad, match in (((x[:1], x, table), "shape"), ((x, x[..., :32], table), "shape"), ((x, x.half(), table), "one type"),
                       ((x, x, table.long()), "int32"), ((x, x, table[:1]), "without cu_tokens"),
                       ((x.cpu(), x, table), "device memory"), ((x, x, table.cpu()), "device memory")):
        with pytest.raises(sp.SapphireError, match=match):
            kv.write(*bad)
    with pytest.raises(sp.SapphireError, match="shape"):
        kv.write(x, x, table, cu_tokens=torch.zeros(2, device="cuda", dtype=torch.int32))
    with pytest.raises(sp.SapphireError, match="byte tensor"):
        KVCache(dev_ctx, "q8_0", 4, 2, 64, kv.pages[:, :-1])
    with pytest.raises(sp.SapphireError, match="16-byte"):
        flat = torch.zeros(kv.pages.numel() + 16, device="cuda", dtype=torch.uint8)
        KVCache(dev_ctx, "q8_0", 4, 2, 64, flat[8:8 + kv.pages.numel()].view_as(kv.pages)).write(x, x, table)
    kv.write(x[:0], x[:0], table[:0])
    dev_ctx.synchronize()


# ------------------------------------------------------------------- attend --
def attend_plain(kv, q, table, lengths, page, heads, dim, dtype, window=0, scale=None):
    """fp64 out, lse and the error bound before rounding."""
    k, v = (cache_values(kv.pages, dtype, page, heads, dim, j) for j in (0, 1))
    out, bound = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    lse_bound = torch.zeros_like(lse)
    group = q.shape[1] // heads
    scale = dim ** -0.5 if scale is None else scale
    for s, n in enumerate(lengths):
        first = max(0, n - window) if window else 0
        if n <= first:
            continue
        t = torch.arange(first, n, device="cuda")
        pg, slot = table[s].long()[t // page], t % page
        for h in range(heads):
            x = q[s, h * group:(h + 1) * group].double()
            ks, vs = k[pg, h, slot], v[pg, h, slot]
            score = x @ ks.T * scale
            ds = (x.abs() @ ks.abs().T * abs(scale)).amax(-1) * 2.0 ** -19
            one_part = dtype in ("q8_0", "q4_0", "f16") and q.dtype == torch.bfloat16
            if one_part and dtype[0] == "q":
                ds = ds + abs(scale) * x.abs().amax(-1) * ks.abs().sum(-1).amax() * 2.0 ** -14
            out[s, h * group:(h + 1) * group] = torch.softmax(score, -1) @ vs
            bound[s, h * group:(h + 1) * group] = vs.abs().max() * (4 * ds + 2.0 ** -17 + one_part * 2.0 ** -12)[:, None]
            lse[s, h * group:(h + 1) * group] = torch.logsumexp(score, -1)
            lse_bound[s, h * group:(h + 1) * group] = 2 * ds + 2.0 ** -17
    return out, bound, lse, lse_bound


def attend_case(ctx, dtype, kind, lengths, heads, group, dim, page, window=0, seed=0, scale=None, fill=0xFF, loud=1.0):
    """A filled cache; slots that no sequence holds are 0xFF bytes (NaN in every
    dense type and in every scale)."""
    g = gen(seed)
    pages = sum(-(-n // page) for n in lengths) + 2
    kv = make_cache(ctx, dtype, page, heads, dim, pages, fill=fill)
    table = make_table(lengths, page, pages, g)
    n = sum(lengths)
    if n:
        k = torch.randn(n, heads, dim, device="cuda", generator=g)
        k[..., ::17] *= 4 * loud
        v = torch.randn(n, heads, dim, device="cuda", generator=g) * torch.rand(n, heads, 1, device="cuda", generator=g) * loud
        kv.write(k.to(IO[kind]), v.to(IO[kind]), table, cu_tokens=ragged(lengths))
    q = torch.randn(len(lengths), heads * group, dim, device="cuda", generator=g).to(IO[kind])
    return kv, table, q


def check_attend(ctx, dtype, kind, lengths, heads, group, dim, page, window=0, seed=0, scale=None, loud=1.0):
    kv, table, q = attend_case(ctx, dtype, kind, lengths, heads, group, dim, page, window, seed, scale, loud=loud)
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 3.0, device="cuda")
    kv.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), out, window=window, lse=lse,
              scale=0.0 if scale is None else scale)
    ctx.synchronize()
    want, bound, want_lse, lse_bound = attend_plain(kv, q, table, lengths, page, heads, dim, dtype, window, scale)
    assert_within(out, want, bound, f"{dtype} {kind}")
    empty = torch.tensor([n == 0 for n in lengths], device="cuda")
    assert (out[empty] == 0).all() and (lse[empty] == -math.inf).all()
    if (~empty).any():
        assert_within(lse[~empty], want_lse[~empty], lse_bound[~empty], "lse")
    return kv, table, q, out


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,heads,group", [(64, 2, 1), (96, 1, 3), (128, 3, 4), (192, 2, 8), (256, 1, 5)])
def test_attend_types_and_heads(dev_ctx, dtype, kind, dim, heads, group):
    check_attend(dev_ctx, dtype, kind, [37, 0, 1, 200, 16, 65], heads, group, dim, 16, seed=dim)


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("page", [1, 3, 16, 24, 100, 4096])
def test_attend_pages(dev_ctx, dtype, page):
    check_attend(dev_ctx, dtype, "f32", [1, 15, 33, 257, 1000], 2, 4, 128, page, seed=page)


@pytest.mark.parametrize("dtype", ["bf16", "q8_0"])
@pytest.mark.parametrize("window", [1, 16, 100, 513, 5000])
def test_attend_window(dev_ctx, dtype, window):
    check_attend(dev_ctx, dtype, "f32", [0, 1, 16, 99, 100, 101, 700, 1501], 1, 2, 64, 16, window=window, seed=window)


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("group", [2, 6, 7, 9, 12, 16, 33])
def test_attend_groups(dev_ctx, dtype, group):
    check_attend(dev_ctx, dtype, "bf16", [130, 7], 2, group, 128, 16, seed=group)


@pytest.mark.parametrize("group", [12, 24, 40, 72, 88])
def test_attend_head_tiles_side_by_side(dev_ctx, group):
    """2, 3, 5, 9 and 11 tiles of 8 heads: on sides of their own, three of three, or one behind another; few
    sequences (ranges in the middle of them) and many (items of one block each)."""
    check_attend(dev_ctx, "q8_0", "bf16", [5003, 0, 1], 2, group, 64, 16, seed=group)
    check_attend(dev_ctx, "bf16", "f32", [5 * i % 211 for i in range(160)], 2, group, 64, 8, seed=group)


@pytest.mark.parametrize("dtype", CACHES)
def test_attend_long_and_many(dev_ctx, dtype):
    check_attend(dev_ctx, dtype, "f32", [20011], 1, 4, 64, 64, seed=1)
    check_attend(dev_ctx, dtype, "bf16", [3 * i % 97 for i in range(300)], 2, 4, 64, 16, seed=2)


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("scale", [0.0078125, 1.5, -0.05])
def test_attend_scale_and_range(dev_ctx, dtype, scale):
    """Loud keys and values; scores far apart, so single positions win."""
    check_attend(dev_ctx, dtype, "f32", [300, 41], 1, 4, 128, 16, seed=3, scale=scale, loud=30.0)


@pytest.mark.parametrize("dtype", ["q8_0", "q4_0"])
def test_attend_scales_that_grow(dev_ctx, dtype):
    """Values whose block scales rise by many powers of two along the sequence."""
    g = gen(12)
    n, heads, dim, page = 400, 1, 128, 16
    kv = make_cache(dev_ctx, dtype, page, heads, dim, 30)
    table = make_table([n], page, 30, g)
    k = torch.randn(n, heads, dim, device="cuda", generator=g)
    v = torch.randn(n, heads, dim, device="cuda", generator=g) * torch.logspace(-12, 12, n, base=2, device="cuda")[:, None, None]
    kv.write(k, v, table, cu_tokens=ragged([n]))
    q, out = torch.randn(1, 4, dim, device="cuda", generator=g), torch.empty(1, 4, dim, device="cuda")
    kv.attend(q, table, torch.tensor([n], dtype=torch.int32, device="cuda"), out)
    dev_ctx.synchronize()
    want, bound, _, _ = attend_plain(kv, q, table, [n], page, heads, dim, dtype)
    assert_within(out, want, bound)


def test_attend_q_far_from_one(dev_ctx):
    """Queries of large and small magnitude against every cache type."""
    for dtype in CACHES:
        kv, table, q = attend_case(dev_ctx, dtype, "f32", [90, 33], 1, 4, 64, 16, seed=4)
        lengths = torch.tensor([90, 33], dtype=torch.int32, device="cuda")
        for size, scale in ((2.0 ** 40, 2.0 ** -43), (2.0 ** -60, 2.0 ** 57)):
            x, out = q * size, torch.empty_like(q)
            kv.attend(x, table, lengths, out, scale=scale)
            dev_ctx.synchronize()
            want, bound, _, _ = attend_plain(kv, x, table, [90, 33], 16, 1, 64, dtype, scale=scale)
            assert_within(out, want, bound, f"{dtype} {size}")


def test_attend_strides_offset_and_shared_pages(dev_ctx):
    kv, table, _ = attend_case(dev_ctx, "bf16", "f16", [40, 70], 2, 3, 64, 16, seed=5)
    buf = torch.randn(2, 6 * 64 * 2 + 1, device="cuda", generator=gen(6)).half()
    q = buf[:, 1:].unflatten(1, (12, 64))[:, ::2]
    res = torch.full((2, 8, 64), 2.0, device="cuda", dtype=torch.float16)
    out = res[:, 1:7]
    table[1, 0] = table[0, 0]                                  # a prefix both sequences hold
    kv.attend(q, table, torch.tensor([38, 68], dtype=torch.int32, device="cuda"), out, length_offset=2)
    dev_ctx.synchronize()
    want, bound, _, _ = attend_plain(kv, q, table, [40, 70], 16, 2, 64, "bf16")
    assert_within(out, want, bound)
    assert (res[:, 0] == 2).all() and (res[:, 7] == 2).all()


def test_attend_is_repeatable(dev_ctx):
    kv, table, q = attend_case(dev_ctx, "q8_0", "bf16", [3000, 17, 999], 2, 4, 128, 16, seed=7)
    n = torch.tensor([3000, 17, 999], dtype=torch.int32, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(q)
    kv.attend(q, table, n, a)
    for _ in range(5):
        kv.attend(q, table, n, b)
        dev_ctx.synchronize()
        assert torch.equal(a, b)


def test_attend_far_offsets(dev_ctx):
    """Pages behind 4 GB, and rows behind 2^31 elements."""
    from sapphire_b200.attention import KVCache, kv_page_bytes
    per = kv_page_bytes("bf16", 64, 8, 128)
    count = (5 << 30) // per
    kv = KVCache(dev_ctx, "bf16", 64, 8, 128, torch.empty(count, per, dtype=torch.uint8, device="cuda"))
    n = [130, 64]
    table = torch.tensor([[count - 1, 0, count - 2], [count - 3, -1, -1]], dtype=torch.int32, device="cuda")
    g = gen(13)
    k, v = (torch.randn(194, 8, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
    kv.write(k, v, table, cu_tokens=ragged(n))
    q, out = torch.randn(2, 32, 128, device="cuda", generator=g).bfloat16(), torch.empty(2, 32, 128, device="cuda").bfloat16()
    kv.attend(q, table, torch.tensor(n, dtype=torch.int32, device="cuda"), out)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    kv.read(ko, vo, table, cu_tokens=ragged(n))
    dev_ctx.synchronize()
    assert torch.equal(ko, k) and torch.equal(vo, v)
    small = make_cache(dev_ctx, "bf16", 64, 8, 128, 4)
    near = torch.tensor([[3, 0, 2], [1, -1, -1]], dtype=torch.int32, device="cuda")
    small.write(k, v, near, cu_tokens=ragged(n))
    again = torch.empty_like(out)
    small.attend(q, near, torch.tensor(n, dtype=torch.int32, device="cuda"), again)
    dev_ctx.synchronize()
    assert torch.equal(out, again)


def test_attend_bad_places(sp, dev_ctx):
    """A page outside the cache counts as not attended, a length outside the
    table is clamped; both are reported, and the context works on."""
    kv, table, q = attend_case(dev_ctx, "bf16", "f32", [40, 20], 1, 2, 64, 16, seed=8)
    good = table.clone()
    lengths = torch.tensor([40, 20], dtype=torch.int32, device="cuda")
    out, ref = torch.empty_like(q), torch.empty_like(q)
    kv.attend(q, good, lengths, ref)
    dev_ctx.synchronize()
    for bad in (-5, kv.pages.shape[0], 2 ** 31 - 1):
        table[0, 1] = bad
        kv.attend(q, table, lengths, out)
        with pytest.raises(sp.SapphireError, match="paged key-value cache"):
            dev_ctx.synchronize()
        assert torch.equal(out[1], ref[1]) and torch.isfinite(out[0]).all()
    for bad in (-1, 49, 2 ** 31 - 1):
        kv.attend(q, good, torch.tensor([bad, 20], dtype=torch.int32, device="cuda"), out)
        with pytest.raises(sp.SapphireError, match="paged key-value cache"):
            dev_ctx.synchronize()
        assert torch.equal(out[1], ref[1])
        assert bad > 0 or (out[0] == 0).all()
    kv.attend(q, good, lengths, out)
    dev_ctx.synchronize()
    assert torch.equal(out, ref)


def test_attend_refusals(sp, dev_ctx):
    kv, table, q = attend_case(dev_ctx, "f32", "f32", [4, 5], 2, 2, 64, 16)
    n, out = torch.tensor([4, 5], dtype=torch.int32, device="cuda"), torch.empty_like(q)
    for args, kw, match in (((q[:, :3], table, n, out[:, :3]), {}, "query heads"), ((q, table, n, out.half()), {}, "one type"),
                            ((q, table, n[:1], out), {}, "shape"), ((q, table[:1], n, out), {}, "shape"),
                            ((q, table, n.long(), out), {}, "int32"), ((q, table, n, out), {"window": -1}, "window"),
                            ((q, table, n, out), {"scale": math.inf}, "scale"), ((q.cpu(), table, n, out), {}, "device memory"),
                            ((q, table, n, out.cpu()), {}, "device memory"), ((q, table, n.cpu(), out), {}, "device memory"),
                            ((q, table, n, out), {"lse": torch.zeros(2, 3, device="cuda")}, "lse")):
        with pytest.raises(sp.SapphireError, match=match):
            kv.attend(*args, **kw)
    kv.attend(q[:0], table[:0], n[:0], out[:0])
    dev_ctx.synchronize()


# ----------------------------------------------------------------- together --
@pytest.mark.parametrize("dtype", CACHES)
def test_decoding_steps_together(dev_ctx, dtype):
    """rope, write and attend as a serving loop runs them: a ragged prompt, then
    steps of one token each, against the dense 64-bit computation."""
    from sapphire_b200.attention import Rope
    g = gen(21)
    heads, group, dim, page, steps = 2, 3, 64, 8, 5
    prompt = [9, 1, 20]
    total = [n + steps for n in prompt]
    kv = make_cache(dev_ctx, dtype, page, heads, dim, 20, fill=0xFF)
    table = make_table(total, page, 20, g)
    rope = Rope(dev_ctx, dim, theta=1e4)
    pos = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in prompt])
    k, v = (torch.randn(sum(prompt), heads, dim, device="cuda", generator=g) for _ in range(2))
    rope.apply(pos, k=k)
    kv.write(k, v, table, cu_tokens=ragged(prompt))
    lengths = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    for step in range(steps):
        q, k, v = (torch.randn(3, h, dim, device="cuda", generator=g) for h in (heads * group, heads, heads))
        q0, k0 = q.clone(), k.clone()
        rope.apply(lengths, q, k)
        kv.write(k, v, table, start=lengths)
        out = torch.empty_like(q)
        kv.attend(q, table, lengths, out, length_offset=1)
        now = [n + step + 1 for n in prompt]
        dev_ctx.synchronize()
        for x, x0 in ((q, q0), (k, k0)):
            want, e = rope_plain(x0, lengths, dim, "half")
            assert_within(x, want, e)
        want, bound, _, _ = attend_plain(kv, q, table, now, page, heads, dim, dtype)
        assert_within(out, want, bound)
        lengths += 1


def test_another_stream_and_device_guard(sp):
    """Two contexts on streams of their own, each with its cache."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs, runs = [], []
    for i, st in enumerate(streams):
        c = sp.Context(num_threads=1)
        c.set_stream(st.cuda_stream)
        ctxs.append(c)
        with torch.cuda.stream(st):
            lengths = [2500, 0, 300 + i]
            kv, table, q = attend_case(c, "q8_0", "f32", lengths, 2, 4, 64, 16, seed=30 + i)
            runs.append((kv, table, q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.empty_like(q), lengths))
    torch.cuda.synchronize()
    for _ in range(4):
        for kv, table, q, n, out, _ in runs:
            kv.attend(q, table, n, out)
    for c, (kv, table, q, n, out, lengths) in zip(ctxs, runs):
        c.synchronize()
        want, bound, _, _ = attend_plain(kv, q, table, lengths, 16, 2, 64, "q8_0")
        assert_within(out, want, bound)
        c.close()


def test_captured_calls_keep_workspaces_of_their_own(sp, dev_ctx):
    """Two captured graphs replayed at the same time; new lengths take effect."""
    st = torch.cuda.Stream()
    dev_ctx.set_stream(st.cuda_stream)
    sets = []
    for i in range(2):
        kv, table, q = attend_case(dev_ctx, "q8_0", "bf16", [1500, 900, 40], 2, 4, 128, 16, seed=40 + i)
        n = torch.tensor([1500, 900, 40], dtype=torch.int32, device="cuda")
        ws = torch.full((kv.workspace_bytes(3, 8),), 0xEE, dtype=torch.uint8, device="cuda")
        sets.append((kv, table, q, n, torch.empty_like(q), ws))
    dev_ctx.synchronize()
    graphs = []
    for kv, table, q, n, out, ws in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            with pytest.raises(sp.SapphireError, match="workspace"):
                kv.attend(q, table, n, out)
            kv.attend(q, table, n, out, workspace=ws)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for lengths in ([1500, 900, 40], [3, 899, 0], [1400, 1, 40]):
        for *_, n, out, ws in sets:
            n.copy_(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        dev_ctx.synchronize()
        for kv, table, q, n, out, ws in sets:
            want, bound, _, _ = attend_plain(kv, q, table, lengths, 16, 2, 128, "q8_0")
            assert_within(out, want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "q8_0", "q4_0"])
@pytest.mark.parametrize("lengths", [[30001] + [9] * 70, [700, 0, 1, 650], [257] * 40])
def test_pieces_are_joined_in_their_order(dev_ctx, dtype, lengths):
    """Calls on the context's workspace, whose last block joins a sequence's pieces, give the same bits every time;
    so do calls on the caller's."""
    kv, table, q = attend_case(dev_ctx, dtype, "f32", lengths, 2, 4, 64, 16, seed=71)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ws = torch.full((kv.workspace_bytes(len(lengths), 8),), 0xEE, dtype=torch.uint8, device="cuda")
    want, bound, want_lse, lse_bound = attend_plain(kv, q, table, lengths, 16, 2, 64, dtype)
    for workspace in (None, ws):
        first = None
        for _ in range(12):
            out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 3.0, device="cuda")
            kv.attend(q, table, n, out, lse=lse, workspace=workspace)
            dev_ctx.synchronize()
            if first is None:
                first = (out, lse)
                assert_within(out, want, bound)
                some = n > 0
                assert_within(lse[some], want_lse[some], lse_bound[some])
            assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_changing_streams(sp, dev_ctx):
    """A call on the default stream, the next on another at once (both in the
    context's workspace), and a change of streams while one is captured."""
    dev_ctx.set_stream(0)
    kv, table, q = attend_case(dev_ctx, "q8_0", "f32", [9000, 4000, 40], 8, 4, 128, 16, seed=60)
    n = torch.tensor([9000, 4000, 40], dtype=torch.int32, device="cuda")
    outs = [torch.empty_like(q) for _ in range(4)]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    for _ in range(5):
        dev_ctx.set_stream(0)
        for _ in range(4):
            kv.attend(q, table, n, outs[0])
        dev_ctx.set_stream(st.cuda_stream)
        kv.attend(q[:1], table[:1], n[:1], outs[1][:1])
    dev_ctx.set_stream(0)
    ws = torch.empty(kv.workspace_bytes(3, 32), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        dev_ctx.set_stream(st.cuda_stream)
        kv.attend(q, table, n, outs[2], workspace=ws)
        dev_ctx.set_stream(0)
    kv.attend(q, table, n, outs[3])
    graph.replay()
    torch.cuda.synchronize()
    dev_ctx.synchronize()
    want, bound, _, _ = attend_plain(kv, q, table, [9000, 4000, 40], 16, 8, 128, "q8_0")
    for i, o in enumerate(outs):
        rows = 1 if i == 1 else 3
        assert_within(o[:rows], want[:rows], bound[:rows] if torch.is_tensor(bound) else bound, str(i))


def test_workspace_refusals(sp, dev_ctx):
    kv, table, q = attend_case(dev_ctx, "bf16", "bf16", [4], 1, 2, 64, 16)
    n, out = torch.tensor([4], dtype=torch.int32, device="cuda"), torch.empty_like(q)
    need = kv.workspace_bytes(1, 2)
    for ws in (torch.zeros(need - 1, dtype=torch.uint8, device="cuda"), torch.zeros(need + 16, dtype=torch.uint8, device="cuda")[8:]):
        with pytest.raises(sp.SapphireError, match="workspace"):
            kv.attend(q, table, n, out, workspace=ws)
    with pytest.raises(sp.SapphireError, match="device memory"):
        kv.attend(q, table, n, out, workspace=torch.zeros(need, dtype=torch.uint8).contiguous())
    with pytest.raises(sp.SapphireError, match="query heads"):
        kv.workspace_bytes(1, 0)
    kv.attend(q, table, n, out, workspace=torch.zeros(need, dtype=torch.uint8, device="cuda"))
    dev_ctx.synchronize()


@pytest.mark.parametrize("dtype", ["q8_0", "q4_0", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attend_values_beside_infinities(dev_ctx, dtype, kind):
    """An infinite value, and one of 2^40 (2^15 in fp16) at a position whose
    probability is zero, leave the other dims what they are."""
    g = gen(14)
    n, dim, page = 90, 128, 16
    kv = make_cache(dev_ctx, dtype, page, 1, dim, 8)
    table = make_table([n], page, 8, g)
    q = torch.randn(1, 4, dim, device="cuda", generator=g).to(IO[kind])
    k = torch.randn(n, 1, dim, device="cuda", generator=g)
    v = torch.randn(n, 1, dim, device="cuda", generator=g)
    k[50] = -1000 * q[0].float().sign().sum(0).sign()          # far below the others for every head
    q = q.abs() * q.float().sign().sum(1, keepdim=True).sign().to(q.dtype)
    v[50] *= 2.0 ** (12 if dtype == "f16" else 40)
    v[20, 0, 3] = math.inf
    kv.write(k, v, table, cu_tokens=ragged([n]))
    out = torch.empty_like(q)
    kv.attend(q, table, torch.tensor([n], dtype=torch.int32, device="cuda"), out)
    dev_ctx.synchronize()
    clean = v.clone()
    clean[20, 0, 3] = 1.0
    clean[50] = 0.0
    kv.write(k, clean, table, cu_tokens=ragged([n]))
    want, bound, _, _ = attend_plain(kv, q, table, [n], page, 1, dim, dtype)
    hurt = slice(0, 32) if dtype[0] == "q" else slice(3, 4)
    assert not torch.isfinite(out[..., hurt]).any()
    keep = torch.ones(dim, dtype=torch.bool, device="cuda")
    keep[hurt] = False
    assert_within(out[..., keep], want[..., keep], bound[..., keep])


@pytest.mark.parametrize("dtype", ["q8_0", "q4_0"])
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 4), (128, 8), (192, 3), (256, 7)])
@pytest.mark.parametrize("loud", [128.0, 8192.0])
def test_attend_query_with_a_loud_channel(dev_ctx, dtype, dim, group, loud):
    """One channel of a bf16 query 2^15 times the others; its keys are the same in every position, so the others
    decide.  Those are whole multiples of 2^-21 of the loud one, which the query's integers hold exactly; a
    block's sum and the score round fewer than 16 times, 2^-24 each of sum|q k|."""
    g = gen(int(loud) + dim + group)
    lengths, heads, page = [40, 9, 300], 2, 16
    kv = make_cache(dev_ctx, dtype, page, heads, dim, 30, fill=0xFF)
    table = make_table(lengths, page, 30, g)

    def signs(*shape):
        return torch.randint(0, 2, shape, device="cuda", generator=g).float() * 2 - 1

    k = signs(sum(lengths), heads, dim)
    k[..., 0] = 1.0                                       # the first of each block's largest: one scale for all
    v = torch.randn(sum(lengths), heads, dim, device="cuda", generator=g)
    kv.write(k, v, table, cu_tokens=ragged(lengths))
    q = signs(3, heads * group, dim) * loud * 2.0 ** -15
    q[..., 0] = loud * signs(3, heads * group)
    q = q.bfloat16()
    scale = 2.0 ** 11 / loud                              # the others' sum is then about 2^-4 sqrt(dim)
    out, lse = torch.empty_like(q), torch.empty(3, heads * group, device="cuda")
    kv.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), out, scale=scale, lse=lse)
    dev_ctx.synchronize()
    want, bound, want_lse, lse_bound = attend_plain(kv, q, table, lengths, page, heads, dim, dtype, scale=scale)
    ds = (2 ** 11 + dim * 2.0 ** -4) * 2.0 ** -20
    assert_within(out, want, v.abs().max().double() * (4 * ds + 2.0 ** -17 + 2.0 ** -12))
    assert_within(lse, want_lse, torch.tensor(2 * ds + 2.0 ** -17, device="cuda", dtype=torch.float64), "lse")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "q8_0", "q4_0"])
def test_attend_values_of_one_sign_over_a_million_tokens(dev_ctx, dtype):
    """bf16 queries, so many sequences of 2^20 tokens (on the same pages) that one block walks the whole of one, and
    positive values: what every sum loses in the same direction adds up.  A lane adds to its sum of probabilities
    2^15 times and to an output 2^14 times; to nearest, errors of either sign, so at most 4 sqrt(2^15) 2^-24 =
    2^-14.5 and 2^-15 of it.  With scores off by 2^-18 and probabilities rounded to 2^-12 each, either sign: 2^-13."""
    g = gen(70)
    n, dim, page, sequences = 1 << 20, 64, 4096, 600
    kv = make_cache(dev_ctx, dtype, page, 1, dim, n // page)
    table = torch.randperm(n // page, device="cuda", generator=g).int().expand(sequences, -1).contiguous()
    k = torch.randn(n, 1, dim, device="cuda", generator=g)
    v = (torch.rand(dim, device="cuda", generator=g) + 1) * (1 + torch.rand(n, 1, dim, device="cuda", generator=g) / 8)
    kv.write(k.bfloat16(), v.bfloat16(), table[:1], cu_tokens=ragged([n]))
    q = (torch.randn(sequences, 2, dim, device="cuda", generator=g) / 2).bfloat16()
    out = torch.empty_like(q)
    kv.attend(q, table, torch.full((sequences,), n, dtype=torch.int32, device="cuda"), out)
    dev_ctx.synchronize()
    for s in (0, 299, 599):
        want, _, _, _ = attend_plain(kv, q[s:s + 1], table[s:s + 1], [n], page, 1, dim, dtype)
        assert_within(out[s:s + 1], want, want.abs() * 2.0 ** -13, dtype)


def test_set_stream_refuses_what_it_cannot_wait_for(sp, dev_ctx):
    """Work from before a capture began on the context's stream, and work on the default stream while a blocking
    stream is captured, cannot be waited for: the stream stays.  A stream that was set while captured holds no such
    work (test_changing_streams)."""
    st = torch.cuda.Stream()
    dev_ctx.set_stream(st.cuda_stream)
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        x += 1
        with pytest.raises(sp.SapphireError, match="captur"):
            dev_ctx.set_stream(0)
    assert dev_ctx.stream == st.cuda_stream
    graph.replay()                                        # the capture was not ended by it
    torch.cuda.synchronize()
    assert (x == 1).all()
    dev_ctx.set_stream(0)
    assert dev_ctx.stream == 0
    # a capture that was going on when its stream was set, and another behind it
    second, third = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(second, stream=st):
        dev_ctx.set_stream(st.cuda_stream)
        x += 1
    with torch.cuda.graph(third, stream=st):
        x += 1
        with pytest.raises(sp.SapphireError, match="captur"):
            dev_ctx.set_stream(0)
    dev_ctx.set_stream(0)


def test_set_stream_beside_the_capture_of_a_blocking_stream(sp, dev_ctx):
    """The default stream cannot be waited for while a stream that waits for it is captured."""
    cudart = torch.cuda.cudart()
    handle = ctypes.c_void_p()
    assert int(cudart.cudaStreamCreate(ctypes.addressof(handle))) == 0
    blocking, other = torch.cuda.ExternalStream(handle.value), torch.cuda.Stream()
    dev_ctx.set_stream(0)
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=blocking):
        x += 1
        with pytest.raises(sp.SapphireError, match="captur"):
            dev_ctx.set_stream(other.cuda_stream)
        assert dev_ctx.stream == 0
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 1).all()
    dev_ctx.set_stream(other.cuda_stream)
    dev_ctx.set_stream(0)
    del graph
    assert int(cudart.cudaStreamDestroy(handle.value)) == 0


def test_attend_context_workspace_does_not_grow(dev_ctx):
    """The first call without a workspace allocates; a later one of a larger shape neither allocates nor waits for
    what the stream still runs."""
    sets = []
    for dtype, dim, group in (("f32", 256, 1), ("f32", 64, 8), ("q8_0", 256, 8), ("q4_0", 128, 4), ("bf16", 128, 8)):
        kv, table, q = attend_case(dev_ctx, dtype, "f32", [400, 30], 1, group, dim, 16, seed=dim)
        n, out = torch.tensor([400, 30], dtype=torch.int32, device="cuda"), torch.empty_like(q)
        # (once with a workspace, so that the kernels are loaded)
        kv.attend(q, table, n, out, workspace=torch.empty(kv.workspace_bytes(2, group), dtype=torch.uint8, device="cuda"))
        sets.append((kv, table, q, n, out, dtype, dim))
    kv, table, q, n, out, _, _ = sets[0]
    kv.attend(q, table, n, out)
    dev_ctx.synchronize()
    for kv, table, q, n, out, _, _ in sets:
        torch.cuda._sleep(200_000_000)                    # cycles: about 0.1 s
        slept = torch.cuda.Event()
        slept.record()
        kv.attend(q, table, n, out)
        assert not slept.query()
        torch.cuda.synchronize()
    dev_ctx.synchronize()
    for kv, table, q, n, out, dtype, dim in sets:
        want, bound, _, _ = attend_plain(kv, q, table, [400, 30], 16, 1, dim, dtype)
        assert_within(out, want, bound)


def test_rope_of_a_closed_plan_or_context(sp):
    """The plan holds memory of its context: neither is used behind the other's end."""
    from sapphire_b200.attention import Rope
    ctx = sp.Context(num_threads=1)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    a, b = Rope(ctx, 64), Rope(ctx, 64)
    q, pos = torch.zeros(1, 1, 64, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int32)
    a.apply(pos, q)
    a.close()
    with pytest.raises(sp.SapphireError, match="closed"):
        a.apply(pos, q)
    b.apply(pos, q)
    ctx.close()
    with pytest.raises(sp.SapphireError, match="closed"):
        b.apply(pos, q)
    b.close()


@pytest.mark.parametrize("dtype", ["f32", "q8_0", "q4_0"])
def test_attend_lengths_near_2_to_the_31(sp, dev_ctx, dtype):
    """A window at the end of the longest sequence that positions of 31 bits allow, and lengths beyond it."""
    g = gen(31)
    page, dim, longest, window = 4096, 64, 2 ** 31 - 16384, 5000
    kv = make_cache(dev_ctx, dtype, page, 1, dim, 3)
    table = (torch.arange(2 ** 31 // page, device="cuda", dtype=torch.int32) % 3).expand(3, -1).contiguous()
    k, v = (torch.randn(3 * page, 1, dim, device="cuda", generator=g) for _ in range(2))
    kv.write(k, v, table[:1], cu_tokens=ragged([3 * page]))
    q = torch.randn(3, 2, dim, device="cuda", generator=g)
    out = torch.empty_like(q)
    lengths = [longest - 5, 100, longest]
    kv.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), out, window=window)
    dev_ctx.synchronize()
    want, bound, _, _ = attend_plain(kv, q, table, lengths, page, 1, dim, dtype, window)
    assert_within(out, want, bound)
    again = torch.empty_like(q)
    for beyond in (longest + 1, 2 ** 31 - 64, 2 ** 31 - 1):
        kv.attend(q, table, torch.tensor([longest - 5, 100, beyond], dtype=torch.int32, device="cuda"), again, window=window)
        with pytest.raises(sp.SapphireError, match="paged key-value cache"):
            dev_ctx.synchronize()
        assert torch.equal(again, out)


def test_rope_angles_at_the_farthest_positions(dev_ctx):
    """cos and sin against decimals of 50 digits, without slack for the oracle: the phase is good to 2^-32 of a turn
    and its fp32 half turns to 2^-26, so an angle is off by at most 2 pi 2^-25.9 < 2^-23.2, sincospi by one step
    (2^-24) more."""
    from decimal import Decimal, getcontext
    from sapphire_b200.attention import Rope
    getcontext().prec = 50
    turn = 2 * Decimal("3.14159265358979323846264338327950288419716939937510")
    pos = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 77777, 1234567891, 2 ** 30 + 1, 3]
    q = torch.zeros(len(pos), 1, 64, device="cuda")
    q[..., :32] = 1.0
    for theta, factor in ((1e4, 1), (5e5, 1), (1e6, 3)):
        out = torch.empty_like(q)
        Rope(dev_ctx, 64, theta=theta, scaling="linear", factor=factor).apply(
            torch.tensor(pos, device="cuda", dtype=torch.int32), q, q_out=out)
        dev_ctx.synchronize()
        f = [(Decimal(theta).ln() * (Decimal(-2 * i) / 64)).exp() / factor for i in range(32)]
        a = torch.tensor([[float(p * x / turn % 1 * turn) for x in f] for p in pos], dtype=torch.float64, device="cuda")
        want = torch.cat((a.cos(), a.sin()), -1)[:, None]
        assert (out.double() - want).abs().max().item() <= 2.0 ** -23.2 + 2.0 ** -24


# Sizes at which (on 148 SMs) a thread of the rotation walks down tokens (t) or heads (h), and its ends value by
# value do (s).
@pytest.mark.parametrize("kind,tokens,heads,kv_heads,dim,rot,layout,scaling", [
    ("bf16", 9601, 8, 2, 128, 128, "half", "banded"),                # t
    ("f32", 5003, 40, 8, 128, 128, "half", "none"),                  # t, h
    ("f16", 5003, 40, 8, 128, 96, "interleaved", "linear"),          # h
    ("bf16", 9601, 32, 8, 128, 128, "interleaved", "yarn"),          # t, h
    ("f16", 9601, 2, 1, 512, 504, "half", "none"),                   # t, units of 4
    ("f32", 20011, 4, 1, 96, 64, "half", "yarn"),                    # t
    ("bf16", 4001, 64, 32, 256, 256, "half", "banded"),              # h
    ("f32", 9601, 40, 8, 96, 22, "half", "none"),                    # t, h, s
    ("bf16", 9601, 40, 8, 90, 42, "interleaved", "linear"),          # t, h, s
])
def test_rope_threads_that_walk(dev_ctx, kind, tokens, heads, kv_heads, dim, rot, layout, scaling):
    test_rope(dev_ctx, tokens, heads, kv_heads, dim, rot, layout, kind, scaling)


def test_rope_in_place_by_threads_that_walk(dev_ctx):
    from sapphire_b200.attention import Rope
    g = gen(9)
    qkv = torch.randn(9601, 48, 128, device="cuda", generator=g).bfloat16()
    before = qkv.clone()
    pos = torch.randint(0, 131072, (9601,), device="cuda", generator=g, dtype=torch.int32)
    Rope(dev_ctx, 128, rot_dim=96).apply(pos, qkv[:, :32], qkv[:, 32:40])
    dev_ctx.synchronize()
    want, e = rope_plain(before[:, :40], pos, 96, "half")
    assert_within(qkv[:, :40], want, e)
    assert torch.equal(qkv[:, 40:], before[:, 40:]) and torch.equal(qkv[..., 96:], before[..., 96:])


# Sizes at which (on 148 SMs) a thread of the cache kernels walks down four batches of tokens (or two: 96 dims) and
# down the heads, where a block has fewer rows than there are heads of K and V (256 x 5, 128 x 9, 192 x 12).
@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("kind,rows,dim,heads,page", [
    ("bf16", 4801, 128, 8, 16), ("f32", 6001, 256, 5, 7), ("f16", 6001, 128, 9, 64), ("bf16", 4801, 192, 12, 24),
    ("f32", 9001, 96, 3, 16), ("f16", 12001, 64, 2, 100),
])
def test_write_and_read_by_threads_that_walk(sp, dev_ctx, ctx, dtype, kind, rows, dim, heads, page):
    g = gen(dim + heads)
    new = [rows // 3, 0, 1, rows - rows // 3 - 1 - 70]                # 70 rows belong to no sequence
    before = [0, 3, 2 * page, 5]
    total = [a + b for a, b in zip(before, new)]
    pages = sum(-(-n // page) for n in total) + 2
    kv = make_cache(dev_ctx, dtype, page, heads, dim, pages, fill=0xA5)
    table = make_table(total, page, pages, g)
    k, v = (torch.randn(rows, heads, dim, device="cuda", generator=g).to(IO[kind]) for _ in range(2))
    old = kv.pages.clone()
    start = torch.tensor(before, dtype=torch.int32, device="cuda")
    kv.write(k, v, table, start=start, cu_tokens=ragged(new))
    ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    kv.read(ko, vo, table, start=start, cu_tokens=ragged(new))
    dev_ctx.synchronize()
    n = sum(new)
    t = torch.cat([torch.arange(b, b + m, device="cuda") for b, m in zip(before, new)])
    seq = torch.repeat_interleave(torch.arange(4, device="cuda"), torch.tensor(new, device="cuda"))
    pg, slot = table[seq, t // page].long(), t % page
    for j, x, out in ((0, k, ko), (1, v, vo)):
        got = cache_values(kv.pages, dtype, page, heads, dim, j)[pg, :, slot]
        assert torch.equal(got, expected_store(sp, ctx, x, dtype)[:n])
        assert torch.equal(out[:n], got.float().to(IO[kind])) and (out[n:] == 7.0).all()
    # slots that no row went to keep their bytes
    free = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    free[pg, slot] = False
    rb, ns, at, chunk = layout(dtype, dim, page)
    a, b = (x.reshape(pages, heads, chunk) for x in (kv.pages, old))
    for o, size in ((at[0], rb), (at[1], rb), (at[2], 4 * ns), (at[3], 4 * ns)):
        u, w = (x[..., o:o + page * size].reshape(pages, heads, page, size).transpose(1, 2)[free] for x in (a, b))
        assert torch.equal(u, w)


def test_the_first_stream_may_be_set_again(sp):
    """kernel_ctx_get_stream, another stream, and back."""
    ctx = sp.Context(num_threads=1)
    first = ctx.stream
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    kv, table, q = attend_case(ctx, "bf16", "bf16", [40, 3], 1, 2, 64, 16)
    n = torch.tensor([40, 3], dtype=torch.int32, device="cuda")
    outs = [torch.empty_like(q) for _ in range(3)]
    torch.cuda.synchronize()
    kv.attend(q, table, n, outs[0])
    for out in outs[1:]:
        ctx.set_stream(first)
        ctx.set_stream(ctx.stream)
        assert ctx.stream == first
        kv.attend(q, table, n, out)
        ctx.synchronize()
        ctx.set_stream(0)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    ctx.close()


@pytest.mark.parametrize("dtype", ["bf16", "q8_0", "q4_0"])
@pytest.mark.parametrize("page", [16, 24])
def test_attend_pages_before_the_window_may_be_gone(dev_ctx, dtype, page):
    """Table entries of positions before the window are not looked at: freed ones (-1, or of another sequence)
    change nothing and are no error."""
    lengths, window = [1000, 333, 40], 100
    kv, table, q = attend_case(dev_ctx, dtype, "bf16", lengths, 2, 4, 128, page, seed=page)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(q)
    kv.attend(q, table, n, a, window=window)
    gone = table.clone()
    for s, m in enumerate(lengths):
        first = max(0, m - window) // page
        gone[s, :first] = torch.tensor([-1, 2 ** 31 - 1], device="cuda", dtype=torch.int32).repeat(first)[:first]
    kv.attend(q, gone, n, b, window=window)
    dev_ctx.synchronize()
    assert torch.equal(a, b)


def test_attend_most_sequences_and_heads(dev_ctx):
    """65535 sequences of few tokens on shared pages, and 1024 KV heads."""
    g = gen(50)
    kv, held, _ = attend_case(dev_ctx, "q8_0", "bf16", [200], 1, 1, 64, 16, seed=51)
    n = torch.randint(0, 40, (65535,), device="cuda", generator=g, dtype=torch.int32)
    table = held[0, torch.randint(0, 12, (65535, 3), device="cuda", generator=g)]     # full pages of the sequence
    q = torch.randn(65535, 2, 64, device="cuda", generator=g).bfloat16()
    out = torch.full_like(q, 3.0)
    kv.attend(q, table, n, out)
    dev_ctx.synchronize()
    some = torch.cat((torch.arange(40), torch.arange(30000, 30040), torch.arange(65495, 65535))).cuda()
    want, bound, _, _ = attend_plain(kv, q[some], table[some], n[some].tolist(), 16, 1, 64, "q8_0")
    assert_within(out[some], want, bound)
    assert (out[n == 0] == 0).all()
    check_attend(dev_ctx, "f16", "f32", [70, 0, 5], 1024, 1, 64, 16, seed=52)


def test_attend_scales_beyond_fp32_are_refused(sp, dev_ctx):
    """Scores are kept times log2(e), so a scale is refused where that is not finite."""
    kv, table, q = attend_case(dev_ctx, "bf16", "f32", [4], 1, 1, 64, 16)
    n, out = torch.tensor([4], dtype=torch.int32, device="cuda"), torch.empty_like(q)
    for scale in (3e38, -3e38):
        with pytest.raises(sp.SapphireError, match="scale"):
            kv.attend(q, table, n, out, scale=scale)
    kv.attend(q, table, n, out, scale=2e38)
    dev_ctx.synchronize()


@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 4), (256, 3)])
def test_attend_probabilities_of_small_groups_are_not_rounded_to_fp16(dev_ctx, dtype, dim, group):
    """Groups of at most 4 heads under bf16 outputs: with queries so small that the scores' own error vanishes, a
    value is off by the output's rounding and fp32's."""
    lengths, heads, page = [3, 40, 1, 7, 500], 8, 16
    kv, table, q = attend_case(dev_ctx, dtype, "bf16", lengths, heads, group, dim, page, seed=dim)
    q, out = q * 2.0 ** -10, torch.empty_like(q)
    kv.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), out)
    dev_ctx.synchronize()
    want, _, _, _ = attend_plain(kv, q, table, lengths, page, heads, dim, dtype)
    used = torch.cat([table[s, :-(-n // page)] for s, n in enumerate(lengths)]).long()
    k, v = (cache_values(kv.pages, dtype, page, heads, dim, j)[used].nan_to_num(0.0, 0.0, 0.0) for j in (0, 1))
    ds = dim ** -0.5 * q.abs().max().item() * k.abs().sum(-1).max().item() * 2.0 ** -19
    assert ds < 2.0 ** -18
    assert_within(out, want, v.abs().max() * (4 * ds + 2.0 ** -17))

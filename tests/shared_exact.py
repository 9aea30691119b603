"""Caches for attention behind a shared prefix whose keys and values every operand type
holds exactly, so that nothing but probabilities and outputs is rounded: bf16 values in a
dense cache, codes times powers of two in a quantised one.  And their attention in 64 bits,
with bounds.

With ds = scale sum|q k| 2^-19 of a score and u = 2^-8 (bf16 operands: a BF16 cache under
bf16 queries) or 2^-11 (fp16) of a probability:
* out is off by at most A (4 ds + 2^-14 + u), A = sum p |v|, lse by 2 ds + 2^-15, as in
  test_shared_prefix_gpu without what conversion costs there;
* probabilities below 2^-21 of the largest times its group's value lose bits: 2^-20 M, M the
  largest of p_t |v_u| over tokens t and u less than 16 apart;
* roundings of different tokens know nothing of each other, so the norm of out's error is
  about u / sqrt(3) that of S = sqrt(sum (p v)^2).  2 u |S|, and 8 ds |S| for the scores,
  2^-14 |out| for sums that truncate (512 steps of 2^-24, and their like in fp32), 2^-20 |M|
  and the outputs' own half steps are the bound of the norm, whatever the length.  What the
  fewest tokens that a warp brings at a time add to the outputs is more.
"""
from __future__ import annotations

import math

import torch

from test_attention_gpu import IO, gen, half_step, layout, make_cache


def write_rows(kv, dtype, page, table, j, codes, scales):
    """K (j 0) or V (1) rows of a sequence: values (dense) or codes and their scales, [tokens, heads, dim] and
    [tokens, heads, dim / 32], into the pages of `table`."""
    tokens, heads, dim = codes.shape
    row, ns, at, chunk = layout(dtype, dim, page)
    pages = kv.pages.view(-1, heads, chunk)
    t = torch.arange(tokens, device="cuda")
    pg, slot = table.long()[t // page], t % page
    if not ns:
        data = codes.to(IO[dtype]).contiguous().view(torch.uint8)
    else:
        data = (codes + (128 if dtype == "q8_0" else 8)).to(torch.uint8).unflatten(-1, (dim // 32, 8, 4)).transpose(-3, -2).flatten(-3)
        if dtype == "q4_0":
            data = data[..., ::2] | data[..., 1::2] << 4
        padded = torch.zeros(tokens, heads, ns, device="cuda")
        padded[..., :dim // 32] = scales
        rows = pages[..., at[2 + j]:at[2 + j] + 4 * ns * page].unflatten(-1, (page, 4 * ns)).clone()
        rows[pg, :, slot] = padded.view(torch.uint8)
        pages[..., at[2 + j]:at[2 + j] + 4 * ns * page] = rows.flatten(-2)
    rows = pages[..., at[j]:at[j] + page * row].unflatten(-1, (page, row)).clone()
    rows[pg, :, slot] = data
    pages[..., at[j]:at[j] + page * row] = rows.flatten(-2)


def exact_rows(g, dtype, tokens, heads, dim, exponents=None, one_sign=False):
    """(values in fp64, codes, scales) of rows of about unit size, times 2 to `exponents` [tokens]."""
    size = torch.ones(tokens, device="cuda") if exponents is None else torch.exp2(exponents.float())
    if dtype in IO:
        x = torch.randn(tokens, heads, dim, device="cuda", generator=g).bfloat16().float()
        x = (x.abs() + 0.5).bfloat16().float() if one_sign else torch.where(x.abs() < 2.0 ** -7, 0.0, x)      # (fp16 holds 2^-14 in 8 bits)
        x = x * size[:, None, None]
        assert torch.equal(x.to(IO[dtype]).float(), x)
        return x.double(), x, None
    top = 127 if dtype == "q8_0" else 7
    codes = torch.randint(1 if one_sign else -top, top + 1, (tokens, heads, dim), device="cuda", generator=g).float()
    scales = torch.exp2(torch.randint(-7, -4, (tokens, heads, dim // 32), device="cuda", generator=g).float() + (0 if dtype == "q8_0" else 4))
    scales = scales * size[:, None, None]
    return codes.double() * scales.double().repeat_interleave(32, -1), codes, scales


def warp_tokens(dtype, kind, dim):
    """Tokens that a warp of the product brings at a time: a quarter of a tile's where rows are copied as they are, else an eighth."""
    quant = dtype not in IO
    tile = 128 if dim <= 64 else 96 if dim <= 96 else 80 if dim <= 192 else 48 if quant else 64
    return tile // (4 if dtype == "f16" or (dtype == "bf16" and kind == "bf16") else 8)


class Exact:
    """A cache whose sequence of `tokens` is the shared prefix of `seqs` sequences with nothing behind it."""

    def __init__(self, ctx, dtype, kind, tokens, seqs, heads, group, dim, page, seed=0, v_exponents=None, one_sign=False, k_edit=None):
        self.ctx, self.dtype, self.dim, self.heads, self.tokens = ctx, dtype, dim, heads, tokens
        g = gen(seed)
        pages = -(-tokens // page)
        self.table = torch.randperm(pages + 1, device="cuda", generator=g)[:pages].int()
        self.kv = make_cache(ctx, dtype, page, heads, dim, pages + 1, fill=0xFF)
        self.k, codes, scales = exact_rows(g, dtype, tokens, heads, dim)
        if k_edit is not None:                # (one dim's codes, or values)
            codes = k_edit(codes)
            self.k = codes.double() * (1 if scales is None else scales.double().repeat_interleave(32, -1))
        write_rows(self.kv, dtype, page, self.table, 0, codes, scales)
        self.v, codes, scales = exact_rows(g, dtype, tokens, heads, dim, v_exponents, one_sign)
        write_rows(self.kv, dtype, page, self.table, 1, codes, scales)
        self.q = torch.randn(seqs, heads * group, dim, device="cuda", generator=g).to(IO[kind])
        self.u = 2.0 ** -8 if dtype == "bf16" and kind == "bf16" else 2.0 ** -11

    def attend(self):
        seqs, q = self.q.shape[0], self.q
        out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
        self.kv.attend_shared(q, self.table, torch.tensor([self.tokens], dtype=torch.int32, device="cuda"),
                              torch.zeros(seqs, 1, dtype=torch.int32, device="cuda"), torch.zeros(seqs, dtype=torch.int32, device="cuda"), out, lse=lse)
        self.ctx.synchronize()
        return out, lse

    def plain(self, rows):
        """fp64 out, lse, A, S, M and ds of these sequences [n, heads, group, ...]."""
        q = self.q[rows].double().unflatten(1, (self.heads, -1))
        scale = self.dim ** -0.5
        score = torch.einsum("shgd,thd->shgt", q, self.k) * scale
        ds = torch.einsum("shgd,thd->shgt", q.abs(), self.k.abs()).amax(-1, keepdim=True) * scale * 2.0 ** -19
        p = torch.softmax(score, -1)
        big = self.v.abs().amax(-1).T[None, :, None]                           # [1, heads, 1, tokens]
        near = torch.nn.functional.max_pool1d(big.flatten(0, 2), 31, 1, 15).unflatten(0, big.shape[:3])
        M = (p * near).amax(-1, keepdim=True)
        mix = lambda w, v: torch.einsum("shgt,thd->shgd", w, v)               # noqa: E731
        return mix(p, self.v), torch.logsumexp(score, -1), mix(p, self.v.abs()), mix(p * p, self.v * self.v).sqrt(), M, ds, p

    def check(self, out, lse, at_once=4, lost=None):
        """Both bounds; with `lost`, tokens without which the outputs would have to be outside of the second."""
        err2 = tol_u = tol_ds = want2 = half2 = m2 = gone2 = 0.0
        for i in range(0, out.shape[0], at_once):
            want, want_lse, A, S, M, ds, p = self.plain(slice(i, i + at_once))
            got = out[i:i + at_once].double().unflatten(1, (self.heads, -1))
            assert torch.isfinite(got).all()
            before = A * (4 * ds + 2.0 ** -14 + self.u) + M * 2.0 ** -20
            err, half = (got - want).abs(), half_step(out.dtype, want.abs() + before)
            assert (err - before - half).max().item() <= 0, ((err - half) / before).max().item()
            got_lse = lse[i:i + at_once].double().unflatten(1, (self.heads, -1))
            assert ((got_lse - want_lse).abs() - 2 * ds[..., 0] - 2.0 ** -15 - want_lse.abs() * 2.0 ** -24).max().item() <= 0
            err2, want2, half2, m2 = err2 + err.square().sum(), want2 + want.square().sum(), half2 + half.square().sum(), m2 + M.square().sum() * self.dim
            tol_u, tol_ds = tol_u + S.square().sum(), tol_ds + (S * ds).square().sum()
            if lost is not None:
                rest = p.clone()
                rest[..., lost] = 0
                rest = rest / rest.sum(-1, keepdim=True)
                gone2 += (torch.einsum("shgt,thd->shgd", rest, self.v) - want).square().sum()
        root = lambda x: math.sqrt(float(x))                                   # noqa: E731
        tol = 2 * self.u * root(tol_u) + 8 * root(tol_ds) + 2.0 ** -14 * root(want2) + 2.0 ** -20 * root(m2) + root(half2)
        assert root(err2) <= tol, (root(err2), tol)
        if lost is not None:
            assert root(gone2) > 1.25 * tol, (root(gone2), tol)

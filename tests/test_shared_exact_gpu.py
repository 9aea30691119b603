"""Attention behind a shared prefix within bounds that a few lost tokens leave: over rows
that every operand type holds exactly (shared_exact), and over ordinary ones by the norm of
the whole output's error."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from shared_exact import Exact, warp_tokens  # noqa: E402
from test_attention_gpu import CACHES, cache_values, dev_ctx, half_step  # noqa: E402,F401
from test_shared_prefix_gpu import shared_case  # noqa: E402


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("dim,heads,group", [(64, 2, 3), (96, 1, 4), (128, 2, 4), (192, 1, 2), (256, 1, 5)])
def test_exact_rows(dev_ctx, dtype, kind, dim, heads, group):
    """Dropping the tokens that one warp brings at a time (6 to 32) would show."""
    case = Exact(dev_ctx, dtype, kind, 5000, 3, heads, group, dim, 16, seed=dim)
    case.check(*case.attend(), lost=slice(5000 - warp_tokens(dtype, kind, dim), 5000))


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("f16", "f16"), ("q8_0", "bf16"), ("q4_0", "f16"), ("f32", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("one_sign", [False, True])
def test_exact_rows_of_long_pieces(dev_ctx, dtype, kind, one_sign):
    """Blocks that take more tokens than O stays in tensor memory for; values of one sign."""
    case = Exact(dev_ctx, dtype, kind, 30011, 1, 80, 1, 64, 64, seed=4, one_sign=one_sign)
    # Sums of one sign truncate always the same way, by up to 2^-14 of A.
    case.check(*case.attend(), at_once=1, lost=None if one_sign else slice(14000, 14000 + warp_tokens(dtype, kind, 64)))


@pytest.mark.parametrize("dtype", ["q8_0", "q4_0", "f32", "f16"])
@pytest.mark.parametrize("tokens", [1, 5, 6, 7, 10, 47, 48, 49, 63, 64, 65, 79, 80, 81, 96, 127, 128, 129, 640, 641, 1281])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_exact_rows_of_every_length(dev_ctx, dtype, dim, tokens):
    case = Exact(dev_ctx, dtype, "f16", tokens, 2, 1, 3, dim, 24, seed=tokens)
    case.check(*case.attend(), lost=slice(tokens - 1, tokens) if 1 < tokens < 200 else None)


@pytest.mark.parametrize("dtype", ["q8_0", "q4_0", "f32", "f16"])
@pytest.mark.parametrize("seqs,heads,group", [(43, 3, 3), (17, 2, 16), (100, 1, 7), (1, 100, 1), (130, 2, 2)])
def test_exact_rows_of_many_sequences(dev_ctx, dtype, seqs, heads, group):
    case = Exact(dev_ctx, dtype, "bf16", 3000, seqs, heads, group, 128, 16, seed=seqs)
    case.check(*case.attend(), at_once=16, lost=slice(1000, 1000 + warp_tokens(dtype, "bf16", 128)))


@pytest.mark.parametrize("dtype,kind,r", [("q8_0", "bf16", 2.0 ** -10), ("q8_0", "f16", 2.0 ** -10), ("q4_0", "bf16", 2.0 ** -10),
                                          ("f32", "bf16", 2.0 ** -11), ("f32", "f16", 2.0 ** -11)])
@pytest.mark.parametrize("prefix,scale,loud", [(318, None, 1.0), (5000, None, 1.0), (400, 1.5, 1.0), (400, 0.0078125, 8.0)])
def test_ordinary_rows_by_their_norm(dev_ctx, dtype, kind, r, prefix, scale, loud):
    """Rows that are rounded as they become operands.  A value is off by r of it at most, a block's scale and each
    product on their own, so a score by a few times r / sqrt(3) scale sqrt(sum over blocks (q k)^2 + sum (q k)^2): six times
    that for the largest of thousands, in the exponent as it is.  Of different tokens these are as independent as the
    probabilities' roundings (u = 2^-11) and the values' (r), so the norm of out's error is at most 6 / sqrt(3) times
    that of sum over (u, r, the score's) of it times S, S = sqrt(sum (p v)^2); sums as in shared_exact."""
    heads, group, dim, page, seqs = 2, 4, 128, 16, 3
    kv, table, own, q = shared_case(dev_ctx, dtype, kind, prefix, [0] * seqs, heads, group, dim, page, seed=prefix, loud=loud)
    out = torch.empty_like(q)
    kv.attend_shared(q, table, torch.tensor([prefix], dtype=torch.int32, device="cuda"), own,
                     torch.zeros(seqs, dtype=torch.int32, device="cuda"), out, **({} if scale is None else {"scale": scale}))
    dev_ctx.synchronize()
    s = dim ** -0.5 if scale is None else scale
    t = torch.arange(prefix, device="cuda")
    k, v = (cache_values(kv.pages, dtype, page, heads, dim, j)[table.long()[t // page], :, t % page] for j in (0, 1))
    x = q.double().unflatten(1, (heads, group))
    products = torch.einsum("shgd,thd->shgtd", x, k)
    score = products.sum(-1) * s
    p = torch.softmax(score, -1)
    want = torch.einsum("shgt,thd->shgd", p, v).flatten(1, 2)
    off = r * s * (products.square().sum(-1) + products.unflatten(-1, (dim // 32, 32)).sum(-1).square().sum(-1)).sqrt()
    off = off + s * products.abs().sum(-1) * 2.0 ** -19
    S2 = torch.einsum("shgt,thd->shgd", (p * (2.0 ** -11 + r + off)).square(), v.square())
    # (The sum of the probabilities is off by theirs, times out.)
    L2 = (p * (2.0 ** -11 + off)).square().sum(-1)[..., None] * want.unflatten(1, (heads, group)).square()
    tol = 6 / math.sqrt(3) * (math.sqrt(S2.sum().item()) + math.sqrt(L2.sum().item())) + 2.0 ** -14 * want.norm().item()
    tol += half_step(out.dtype, want).norm().item()
    err = (out.double() - want).norm().item()
    assert err <= tol, (err / want.norm().item(), tol / want.norm().item())
    # (Where a few tokens have all the weight their scores' errors are out's: 1.5 times sums of 128 products.)
    assert tol < (0.5 if scale == 1.5 else 0.03) * want.norm().item()

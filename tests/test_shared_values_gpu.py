"""Values of very different size along a shared prefix: what has weight keeps its bits
beside what has none (bounds: shared_exact)."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from shared_exact import Exact  # noqa: E402
from test_attention_gpu import dev_ctx  # noqa: E402,F401

# (cache, queries) whose rows are converted
CONVERTED = [("q8_0", "bf16"), ("q4_0", "bf16"), ("f32", "bf16"), ("bf16", "f16")]


def quiet(loud):
    """Keys whose first dim is 0 but for `loud` tokens, where it is the most that a code can be."""
    def edit(codes):
        codes = codes.clone()
        codes[..., 0] = 0
        codes[loud, :, 0] = 7
        return codes
    return edit


@pytest.mark.parametrize("dtype,kind", CONVERTED)
@pytest.mark.parametrize("size", [12, 26, 30, 60])
@pytest.mark.parametrize("late", [False, True])
def test_a_large_value_without_weight(dev_ctx, dtype, kind, size, late):
    """48 tokens of values 2^size times the others', without weight as the 16 before and behind them."""
    tokens = 1500
    large = slice(1296, 1344) if late else slice(96, 144)
    without = slice(large.start - 16, large.stop + 16)
    exps = torch.zeros(tokens, device="cuda")
    exps[large] = size
    case = Exact(dev_ctx, dtype, kind, tokens, 3, 2, 4, 64, 16, seed=size, v_exponents=exps, k_edit=quiet(without))
    # What a query meets in these tokens: a score of -100 and less (of codes times 2^-7 .. 2^1).
    case.q[..., 0] = -1000 if dtype in ("bf16", "f32") else -4000 if dtype == "q4_0" else -30000
    want, _, _, S, M, _, p = case.plain(slice(0, 3))
    assert p[..., without].amax().item() * 2.0 ** size < 2.0 ** -30 and M.amax().item() < 8
    case.check(*case.attend())


@pytest.mark.parametrize("dtype,kind", CONVERTED)
@pytest.mark.parametrize("size", [-40, 20])
def test_large_values_of_small_weight(dev_ctx, dtype, kind, size):
    """Values 2^size times the others' wherever a token's score is low, both of weight in the end."""
    tokens = 3000
    exps = torch.zeros(tokens, device="cuda")
    some = slice(640, 960)
    exps[some] = size
    case = Exact(dev_ctx, dtype, kind, tokens, 2, 1, 3, 128, 16, seed=7, v_exponents=exps, k_edit=quiet(some))
    case.q[..., 0] = -abs(size) / (1.0 if dtype in ("bf16", "f32") else 8.0 if dtype == "q4_0" else 0.25) if size > 0 else 0.0
    case.check(*case.attend())


@pytest.mark.parametrize("dtype,kind", CONVERTED)
def test_sizes_that_change_along_long_pieces(dev_ctx, dtype, kind):
    """Blocks that take more than O stays in tensor memory for, sizes up and down by up to 2^40 every 160 tokens."""
    tokens = 20011
    steps = torch.tensor([0, 12, -30, 3, -2, 17, -22, 8, 40, -9, 1], device="cuda", dtype=torch.float32)
    exps = steps.repeat_interleave(160).repeat(12)[:tokens] - (36 if kind == "f16" else 0)      # (outputs below 65504)
    case = Exact(dev_ctx, dtype, kind, tokens, 1, 100, 1, 64, 64, seed=8, v_exponents=exps)
    case.check(*case.attend(), at_once=1)

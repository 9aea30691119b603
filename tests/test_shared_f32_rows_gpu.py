"""Attention behind a shared prefix under fp32 queries of many sequences: tiles of 8 rows of
a KV head, side by side and one behind another (bounds: test_shared_prefix_gpu)."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

pytest.importorskip("torch")

from test_attention_gpu import dev_ctx  # noqa: E402,F401
from test_shared_prefix_gpu import check_shared  # noqa: E402


@pytest.mark.parametrize("dtype", ["f32", "bf16", "q8_0"])
@pytest.mark.parametrize("seqs,group", [(22, 4), (26, 4), (75, 4), (37, 8), (1, 300), (131, 1), (64, 4), (9, 5)])
def test_rows_of_many_sequences(dev_ctx, dtype, seqs, group):
    """11, 13, 38, 37, 17, 32 and 6 tiles: numbers with a divisor up to 8 and without one."""
    check_shared(dev_ctx, dtype, "f32", 333, [(7 * i) % 11 for i in range(seqs)], 2, group, 128, 16, seed=seqs)


@pytest.mark.parametrize("dim,heads", [(64, 3), (256, 1)])
def test_rows_behind_a_long_prefix(dev_ctx, dim, heads):
    check_shared(dev_ctx, "f32", "f32", 5000, [3] * 26, heads, 4, dim, 24, seed=dim)

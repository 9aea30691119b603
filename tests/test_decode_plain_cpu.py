"""The 64-bit decode of decode_plain.py against the recorded reference decode (CPU only)."""
from __future__ import annotations

import os

import numpy as np
import pytest

from conftest import GOLDEN

pytest.importorskip("torch")


def test_plain_decode_gives_the_reference_logits():
    """The recorded ids, logits and margins of the grouped-query model, to the reference's fp32 rounding: each of
    six layers adds four fp32 products of at most 512 terms, 6 x 4 x sqrt(512) x 2^-24 of logits around 1."""
    from decode_plain import plain_logits
    from oracle.oracle import Oracle
    from sapphire_b200 import workloads
    golden, oracle, cfg = np.load(os.path.join(GOLDEN, "decode_gqa_tiny_seed3.npz")), Oracle(), workloads.GQA_TINY
    model = workloads.make_decode_model(cfg, lambda a: oracle.quantize(3, a), seed=3)
    assert workloads.model_digest(model) == str(golden["digest"])
    n = len(model["prompt"])
    tokens = np.concatenate([model["prompt"], golden["tokens"]])[:-1]
    logits = plain_logits(cfg, model, tokens, range(n - 1, len(tokens))).numpy()
    assert np.array_equal(logits.argmax(-1), golden["tokens"])
    tol = 6 * 4 * 512 ** 0.5 * 2.0 ** -24
    assert np.abs(logits[0][golden["top_ids"]] - golden["top_logits"]).max() <= tol
    top = np.sort(logits, -1)[:, -2:]
    assert np.abs(top[:, 1] - top[:, 0] - golden["margins"]).max() <= 2 * tol

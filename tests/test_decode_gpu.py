"""Device-resident Gemma-3-270M decode against the reference's own decode.

tests/golden/decode_gemma3_270m_seed0.npz holds the greedy ids the reference
produced (its inference session, layers and Q4_0 kernel_gemv, run by
oracle/decode_ref.c; tests/golden/make_decode_golden.py) for the seeded
random-init model of sapphire_b200.workloads.C3: a 512-token prompt, then 64
greedy tokens.  The GPU decoder must produce the same 64 ids.
"""
from __future__ import annotations

import dataclasses
import os

import numpy as np
import pytest

from conftest import GOLDEN

pytestmark = pytest.mark.gpu

Q4_0 = 3


@pytest.fixture(scope="module")
def golden():
    return np.load(os.path.join(GOLDEN, "decode_gemma3_270m_seed0.npz"))


@pytest.fixture(scope="module")
def decoder(sp, ctx, golden):
    from sapphire_b200 import workloads
    from sapphire_b200.decode import Decoder
    cfg = workloads.C3
    model = workloads.make_decode_model(cfg, lambda a: sp.quantize(ctx, Q4_0, a), seed=0)
    # Same model bytes as the reference run (GPU quantiser == oracle quantiser).
    assert workloads.model_digest(model) == str(golden["digest"])
    dec = Decoder(ctx, cfg, model)
    yield cfg, model, dec
    dec.close()


def test_greedy_tokens_match_reference(decoder, golden):
    cfg, model, dec = decoder
    ids, margins = dec.generate(model["prompt"], cfg.generate)
    ref = golden["tokens"]
    mismatch = np.nonzero(ids != ref)[0]
    assert mismatch.size == 0, (
        f"first mismatch at step {mismatch[0]}: got {ids[mismatch[0]]}, reference {ref[mismatch[0]]}, "
        f"reference margin {golden['margins'][mismatch[0]]:.5f}")
    # The top-1 minus top-2 margins agree with the reference's to rounding.
    assert np.max(np.abs(margins - golden["margins"])) < 2e-3


def test_first_step_logits(decoder, golden):
    cfg, model, dec = decoder
    ids, _ = dec.generate(model["prompt"], 1)
    assert ids[0] == golden["tokens"][0]
    logits = dec.last_logits()
    top = golden["top_ids"]
    # The reference's 64 largest logits, value by value.
    err = np.max(np.abs(logits[top] - golden["top_logits"]))
    assert err < 2e-3 * float(golden["logits0_rms"]) * 10, err
    rms = float(np.sqrt(np.mean(logits.astype(np.float64) ** 2)))
    assert abs(rms - float(golden["logits0_rms"])) < 1e-3 * rms


def test_generate_is_repeatable(decoder):
    cfg, model, dec = decoder
    a, _ = dec.generate(model["prompt"][:40], 8)
    b, _ = dec.generate(model["prompt"][:40], 8)
    assert np.array_equal(a, b)
    assert dec.launches_per_token > 0


def test_generate_rejects_bad_input(sp, decoder):
    cfg, model, dec = decoder
    with pytest.raises(sp.SapphireError):
        dec.generate(np.array([cfg.vocab], dtype=np.int32), 1)
    with pytest.raises(sp.SapphireError):
        dec.generate(model["prompt"], cfg.context)


def test_decoder_from_quantized_safetensors(sp, ctx, decoder, golden, tmp_path):
    """The same model written as a quantized safetensors file (Q4_0
    projections and LM head under the reference's tensor names) loads through
    sapphire_decoder_create_from_safetensors and decodes the reference's ids."""
    from sapphire_b200 import safetensors
    from sapphire_b200.decode import Decoder
    cfg, model, _ = decoder
    path = str(tmp_path / "gemma3_q4_0.safetensors")
    safetensors.save_decode_model(path, cfg, model)
    with safetensors.SafeTensors(path) as st:
        assert st.info("lm_head.weight")[:2] == ("Q4_0", (cfg.vocab, cfg.hidden))
        dec = Decoder.from_safetensors(ctx, cfg, st)
    # The file is closed: everything the decoder uses lives on the GPU.
    os.remove(path)
    try:
        ids, _ = dec.generate(model["prompt"], cfg.generate)
        assert np.array_equal(ids, golden["tokens"])
    finally:
        dec.close()


def test_from_safetensors_rejects_wrong_dtype(sp, ctx, decoder, tmp_path):
    """An LM head stored as BF16 (the reference's tied-embedding layout) is not
    a quantized product here: creation fails with the tensor named."""
    from sapphire_b200 import safetensors
    from sapphire_b200.decode import Decoder
    cfg, model, _ = decoder
    small = dataclasses.replace(cfg, layers=1)
    path = str(tmp_path / "bad.safetensors")
    t = {"model.embed_tokens.weight": ("BF16", (cfg.vocab, cfg.hidden), model["embed"]),
         "lm_head.weight": ("BF16", (cfg.vocab, cfg.hidden), model["embed"])}
    hf = {"q": "self_attn.q_proj", "k": "self_attn.k_proj", "v": "self_attn.v_proj", "o": "self_attn.o_proj",
          "gate": "mlp.gate_proj", "up": "mlp.up_proj", "down": "mlp.down_proj"}
    for name, rows, cols in small.projections():
        t[f"model.layers.0.{hf[name]}.weight"] = ("Q4_0", (rows, cols), model["layers"][0][name])
    safetensors.save(path, t)
    with safetensors.SafeTensors(path) as st:
        with pytest.raises(sp.SapphireError, match="lm_head.weight"):
            Decoder.from_safetensors(ctx, small, st)


def test_stage_per_kernel_path_matches_reference(sp, ctx, decoder, golden, monkeypatch):
    """The one-kernel-per-stage step (SAPPHIRE_DECODE_PERSISTENT=0 at
    creation) gives the reference's ids as well."""
    from sapphire_b200.decode import Decoder
    cfg, model, _ = decoder
    monkeypatch.setenv("SAPPHIRE_DECODE_PERSISTENT", "0")
    dec = Decoder(ctx, cfg, model)
    try:
        assert dec.launches_per_token > 10      # one kernel per stage
        ids, _ = dec.generate(model["prompt"], cfg.generate)
        assert np.array_equal(ids, golden["tokens"])
    finally:
        dec.close()


def test_persistent_step_reports_an_expired_wait(sp, ctx, decoder, golden):
    """A persistent step in which one block never writes its output (a test
    hook: nothing sets the words the others wait for) gives up after its
    bounded wait: creation fails with the expiry reported, no GPU fault, and a
    decoder created afterwards still decodes the reference's ids."""
    from sapphire_b200.decode import Decoder
    cfg, model, dec = decoder
    assert dec.launches_per_token == 3          # persistent step + LM head + argmax
    assert dec.launches_per_prompt_token == 1
    prev = sp.lib.sapphire_test_decode_stall(1)
    try:
        with pytest.raises(sp.SapphireError, match="gave up waiting"):
            Decoder(ctx, cfg, model)
    finally:
        sp.lib.sapphire_test_decode_stall(prev)
    ok = Decoder(ctx, cfg, model)
    try:
        ids, _ = ok.generate(model["prompt"][:64], 8)
        ref, _ = dec.generate(model["prompt"][:64], 8)
        assert np.array_equal(ids, ref)
    finally:
        ok.close()


@pytest.mark.parametrize("persistent", ["1", "0"])
def test_grouped_query_model_matches_reference(sp, ctx, monkeypatch, persistent):
    """A small grouped-query model (two KV heads for four query heads,
    head_dim 64, a global and five local layers, window 32) decodes the
    reference decode's ids through both step implementations
    (tests/golden/decode_gqa_tiny_seed3.npz, tests/golden/make_decode_golden.py)."""
    from sapphire_b200 import workloads
    from sapphire_b200.decode import Decoder
    golden = np.load(os.path.join(GOLDEN, "decode_gqa_tiny_seed3.npz"))
    cfg = workloads.GQA_TINY
    model = workloads.make_decode_model(cfg, lambda a: sp.quantize(ctx, Q4_0, a), seed=3)
    assert workloads.model_digest(model) == str(golden["digest"])
    monkeypatch.setenv("SAPPHIRE_DECODE_PERSISTENT", persistent)
    dec = Decoder(ctx, cfg, model)
    try:
        # 3 launches per generated token for the persistent step, 5 per layer otherwise.
        assert (dec.launches_per_token == 3) == (persistent == "1")
        ids, margins = dec.generate(model["prompt"], cfg.generate)
        assert np.array_equal(ids, golden["tokens"]), (ids, golden["tokens"])
        assert np.max(np.abs(margins - golden["margins"])) < 1e-3
    finally:
        dec.close()


def test_long_prompt_paths_agree(sp, ctx, decoder, monkeypatch):
    """A 1900-token prompt (global layers attend to every position: up to 56
    keys per split over 37 splits per head) gives the same logits through the
    persistent step and through the per-stage path, to fp32 rounding."""
    from sapphire_b200.decode import Decoder
    cfg, model, dec = decoder
    prompt = np.random.default_rng(5).integers(0, cfg.vocab, size=1900).astype(np.int32)
    ids_p, _ = dec.generate(prompt, 1)
    logits_p = dec.last_logits()
    monkeypatch.setenv("SAPPHIRE_DECODE_PERSISTENT", "0")
    ref = Decoder(ctx, cfg, model)
    try:
        ids_s, _ = ref.generate(prompt, 1)
        logits_s = ref.last_logits()
    finally:
        ref.close()
    err = float(np.max(np.abs(logits_p - logits_s)) / np.max(np.abs(logits_s)))
    assert err < 1e-4, err
    top2 = np.sort(logits_s)[-2:]
    if top2[1] - top2[0] > 1e-3:
        assert ids_p[0] == ids_s[0]


# ------------------------------------------------------------- paged cache --
def test_paged_decoder_matches_reference(sp, ctx, decoder, golden):
    """The decoder over fp32 pages (the rope, cache and attention operators in
    place of its own attention) gives the reference's ids."""
    from sapphire_b200.decode import Decoder
    cfg, model, _ = decoder
    for page in (16, 24):
        dec = Decoder(ctx, cfg, model, kv_dtype="f32", kv_page_size=page)
        ids, margins = dec.generate(model["prompt"], cfg.generate)
        assert np.array_equal(ids, golden["tokens"])
        # angles are exact here and fp32 products there: half a step of an angle of up to 575
        assert np.max(np.abs(margins - golden["margins"])) < 2e-3
        assert dec.launches_per_token == 9 * cfg.layers + 4
        dec.close()


@pytest.mark.parametrize("kv", ["bf16", "f16", "q8_0", "q4_0"])
def test_paged_decoder_types(sp, ctx, decoder, golden, kv):
    """Other cache types: the first position attends to itself alone, so its
    logits move by no more than the rounding of its values does; generation
    repeats itself, and the cache is the prompt's alone."""
    from sapphire_b200.decode import Decoder
    cfg, model, ref = decoder
    dec = Decoder(ctx, cfg, model, kv_dtype=kv, kv_page_size=32)
    a, _ = dec.generate(model["prompt"][:40], 8)
    first = dec.last_logits()
    dec.generate(model["prompt"][40:90], 4)
    b, _ = dec.generate(model["prompt"][:40], 8)
    assert np.array_equal(a, b) and np.array_equal(first, dec.last_logits())
    # One token: every attention output is v itself, rounded by the type (half a
    # step relative to the block's largest value).  An RMS norm follows each, so
    # a relative error e of the output of one of 18 layers moves the residual
    # stream by at most e of its own added part, and the sum of 18 parts by 18 e.
    step = {"bf16": 2.0 ** -9, "f16": 2.0 ** -12, "q8_0": 0.5 / 127 * 4, "q4_0": 0.5 / 8 * 4}[kv]
    ref.generate(model["prompt"][:1], 1)
    want = ref.last_logits().astype(np.float64)
    dec.generate(model["prompt"][:1], 1)
    got = dec.last_logits().astype(np.float64)
    assert np.linalg.norm(got - want) <= 18 * step * np.linalg.norm(want)
    dec.close()


def test_paged_decoder_long_context(sp, ctx):
    """A context above the dense cache's 4096: windowed and global layers past it."""
    from sapphire_b200 import workloads
    from sapphire_b200.decode import Decoder
    cfg = dataclasses.replace(workloads.GQA_TINY, context=6000)
    model = workloads.make_decode_model(cfg, lambda a: sp.quantize(ctx, Q4_0, a), seed=3)
    with pytest.raises(sp.SapphireError):
        Decoder(ctx, cfg, model)
    prompt = np.resize(model["prompt"], 4500)
    ids = {}
    for kv, page in (("f32", 64), ("f32", 50)):
        dec = Decoder(ctx, cfg, model, kv_dtype=kv, kv_page_size=page)
        ids[page], _ = dec.generate(prompt, 8)
        with pytest.raises(sp.SapphireError):
            dec.generate(prompt, 1501)
        dec.close()
    assert np.array_equal(ids[64], ids[50])


def test_paged_decoder_refusals(sp, ctx):
    from sapphire_b200 import workloads
    from sapphire_b200.decode import Decoder
    cfg = workloads.GQA_TINY
    model = workloads.make_decode_model(cfg, lambda a: sp.quantize(ctx, Q4_0, a), seed=3)
    for kv, page in (("tq2_0", 16), ("f32", 0), ("q8_0", 5000)):
        with pytest.raises(sp.SapphireError, match="no cache of this type"):
            Decoder(ctx, cfg, model, kv_dtype=kv, kv_page_size=page)


def rounded_store(sp, ctx, kv):
    """What a cache of type kv holds of x [positions, heads, dim], quantised by the library's quantisers."""
    import torch

    def store(x):
        if kv in ("f32", "bf16", "f16"):
            return x.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kv]).double()
        size = 36 if kv == "q8_0" else 20
        flat = np.ascontiguousarray(x.float().cpu().numpy().reshape(-1, x.shape[-1]))
        b = sp.quantize(ctx, sp.DTYPE_Q8_0 if kv == "q8_0" else Q4_0, flat).reshape(-1, size)
        scale = b[:, :4].copy().view(np.float32).astype(np.float64)
        codes = b[:, 4:].view(np.int8) if kv == "q8_0" else \
            np.stack((b[:, 4:] & 15, b[:, 4:] >> 4), -1).reshape(len(b), 32).astype(np.float64) - 8
        return torch.from_numpy((codes * scale).reshape(x.shape)).to(x.device)
    return store


# Each of six layers adds four products to what its logits depend on, and the head one: 25 times the parity bar of
# a product (1e-4) bounds the relative error of the logits.  (A code at the border of two may fall to either side:
# one in 10^5 of them by fp32 rounding.)
LOGITS_RTOL = 25e-4


@pytest.mark.parametrize("kv,page", [("f32", 16), ("bf16", 24), ("f16", 50), ("q8_0", 16), ("q8_0", 7), ("q4_0", 32),
                                     ("q4_0", 5)])
def test_paged_decoder_against_a_plain_decode_of_the_same_cache(sp, ctx, kv, page):
    """Logits at the first positions, inside the window and behind it, against the 64-bit decode whose keys and
    values are rounded as the cache's type rounds them; a decode with others is further away than the tolerance."""
    from decode_plain import plain_logits
    from sapphire_b200 import workloads
    from sapphire_b200.decode import Decoder
    cfg = workloads.GQA_TINY
    model = workloads.make_decode_model(cfg, lambda a: sp.quantize(ctx, Q4_0, a), seed=3)
    tokens = np.random.default_rng(11).integers(0, cfg.vocab, size=120).astype(np.int32)
    lengths = [1, 2, 5, 16, 33, 90, 120]
    want = plain_logits(cfg, model, tokens, [n - 1 for n in lengths], rounded_store(sp, ctx, kv), "cuda").cpu().numpy()
    other = plain_logits(cfg, model, tokens, [n - 1 for n in lengths], rounded_store(sp, ctx, "q4_0" if kv != "q4_0" else "q8_0"),
                         "cuda").cpu().numpy()
    dec = Decoder(ctx, cfg, model, kv_dtype=kv, kv_page_size=page)
    try:
        for n, w, o in zip(lengths, want, other):
            dec.generate(tokens[:n], 1)
            error = np.linalg.norm(dec.last_logits() - w) / np.linalg.norm(w)
            assert error <= LOGITS_RTOL, (n, error)
            assert np.linalg.norm(o - w) > 4 * LOGITS_RTOL * np.linalg.norm(w)
    finally:
        dec.close()


@pytest.mark.parametrize("kv", ["f32", "q8_0", "q4_0"])
def test_paged_decoder_past_the_dense_context(sp, ctx, kv):
    """Logits behind 4096 positions against the 64-bit decode: windows, angles and offsets there."""
    from decode_plain import plain_logits
    from sapphire_b200 import workloads
    from sapphire_b200.decode import Decoder
    cfg = dataclasses.replace(workloads.GQA_TINY, context=6000)
    model = workloads.make_decode_model(cfg, lambda a: sp.quantize(ctx, Q4_0, a), seed=3)
    tokens = np.random.default_rng(12).integers(0, cfg.vocab, size=4500).astype(np.int32)
    lengths = [4097, 4500]
    want = plain_logits(cfg, model, tokens, [n - 1 for n in lengths], rounded_store(sp, ctx, kv), "cuda").cpu().numpy()
    # the same with every token but the last 3000 left out: positions and the global layer's reach count
    near = plain_logits(cfg, model, tokens[-3000:], [2999], rounded_store(sp, ctx, kv), "cuda").cpu().numpy()[0]
    dec = Decoder(ctx, cfg, model, kv_dtype=kv, kv_page_size=64)
    try:
        for n, w in zip(lengths, want):
            dec.generate(tokens[:n], 1)
            error = np.linalg.norm(dec.last_logits() - w) / np.linalg.norm(w)
            assert error <= LOGITS_RTOL, (n, error)
        assert np.linalg.norm(near - want[-1]) > 2 * LOGITS_RTOL * np.linalg.norm(want[-1])
    finally:
        dec.close()


def test_an_expired_wait_is_named_before_a_bad_page(sp, ctx, decoder):
    """Both at the same synchronisation: the message names the wait."""
    import torch
    from sapphire_b200.attention import KVCache, kv_page_bytes
    from sapphire_b200.decode import Decoder
    cfg, model, _ = decoder
    kv = KVCache(ctx, "bf16", 16, 1, 64, torch.zeros(1, kv_page_bytes("bf16", 16, 1, 64), dtype=torch.uint8, device="cuda"))
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    kv.write(x, x, torch.full((1, 1), 7, dtype=torch.int32, device="cuda"))
    prev = sp.lib.sapphire_test_decode_stall(1)
    try:
        with pytest.raises(sp.SapphireError, match="gave up waiting"):
            Decoder(ctx, cfg, model)
    finally:
        sp.lib.sapphire_test_decode_stall(prev)
    ctx.synchronize()
    kv.write(x, x, torch.full((1, 1), 7, dtype=torch.int32, device="cuda"))
    with pytest.raises(sp.SapphireError, match="paged key-value cache"):
        ctx.synchronize()

"""The Gemma-3 decode of sapphire_b200.workloads in 64 bits, all positions at
once: the plain form that decoders are held to where no recorded reference run
reaches (contexts above 4096, caches of other types).

Each step is written from the model's definition; what a cache holds of the
keys and values is the caller's to say (`store`).
"""
from __future__ import annotations

import math

import numpy as np
import torch


def q4_0_values(packed, rows, cols, device):
    """fp64 [rows, cols] of packed Q4_0 rows: 20-byte blocks of an fp32 scale and 32 codes, low nibble first."""
    b = np.asarray(packed).reshape(-1).view(np.uint8).reshape(rows, -1, 20)
    scale = b[..., :4].copy().view(np.float32).astype(np.float64)
    codes = np.stack((b[..., 4:] & 15, b[..., 4:] >> 4), -1).reshape(rows, b.shape[1], 32).astype(np.float64) - 8
    return torch.from_numpy((codes * scale).reshape(rows, -1)[:, :cols]).to(device)


def _norm(x, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt()


def _turn(x, theta):
    """x [positions, heads, dim], pairs (i, i + dim / 2) turned by position theta^(-2i / dim)."""
    n, _, dim = x.shape
    i = torch.arange(dim // 2, dtype=torch.float64, device=x.device)
    a = torch.arange(n, dtype=torch.float64, device=x.device)[:, None, None] * theta ** (-2 * i / dim)
    u, v = x[..., :dim // 2], x[..., dim // 2:]
    return torch.cat((u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()), -1)


def plain_logits(cfg, model, tokens, positions, store=None, device="cpu"):
    """fp64 logits [len(positions), vocab] behind tokens[: p + 1] for each p of positions.  store(x): what the
    cache holds of keys or values x [positions, kv_heads, head_dim] (default: x)."""
    store = store or (lambda x: x)
    eps, n = cfg.rms_eps, len(tokens)
    embed = torch.from_numpy((model["embed"].astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(cfg.vocab, -1))
    h = embed[torch.as_tensor(np.asarray(tokens), dtype=torch.long)].to(device) * math.sqrt(cfg.hidden)
    t = torch.arange(n, device=device)
    group = cfg.heads // cfg.kv_heads
    for l, layer in enumerate(model["layers"]):
        w = {name: q4_0_values(layer[name], rows, cols, device) for name, rows, cols in cfg.projections()}
        x = _norm(h, eps)
        q, k, v = ((x @ w[name].T).unflatten(-1, (-1, cfg.head_dim)) for name in ("q", "k", "v"))
        theta = cfg.rope_theta if cfg.is_global(l) else cfg.rope_local_theta
        q, k = _turn(_norm(q, eps), theta), store(_turn(_norm(k, eps), theta))
        v = store(v)
        seen = t <= t[:, None]
        if not cfg.is_global(l):
            seen &= t > t[:, None] - cfg.sliding_window
        out = torch.empty_like(q)
        for head in range(cfg.heads):
            s = q[:, head] @ k[:, head // group].T / math.sqrt(cfg.query_pre_attn_scalar)
            out[:, head] = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ v[:, head // group]
        h = h + _norm(out.flatten(1) @ w["o"].T, eps)
        x = _norm(h, eps)
        gate, up = x @ w["gate"].T, x @ w["up"].T
        gelu = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
        h = h + _norm((gelu * up) @ w["down"].T, eps)
    return _norm(h[torch.as_tensor(positions)], eps) @ q4_0_values(model["lm_head"], cfg.vocab, cfg.hidden, device).T

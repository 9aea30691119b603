"""Rotary, paged-cache and attention entry points without a GPU: the structs as
C lays them out, page sizes, and refusals that come before any device work."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest

from conftest import ROOT

STRUCTS = {
    "sapphire_rope_config_t": "RopeConfig",
    "sapphire_rope_args_t": "RopeArgs",
    "sapphire_kv_cache_t": "KvCacheStruct",
    "sapphire_kv_args_t": "KvArgs",
    "sapphire_attention_args_t": "AttentionArgs",
}


def test_struct_layout_matches_c(tmp_path, sp):
    from sapphire_b200 import _lib
    lines = ['#include <stdio.h>', '#include "sapphire_attention.h"', "int main(void) {"]
    for c, py in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        for name, _ in getattr(_lib, py)._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {name}));')
    src = tmp_path / "t.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), "-o", str(tmp_path / "t")],
                   check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in STRUCTS.values():
        s = getattr(_lib, py)
        want += [C.sizeof(s)] + [getattr(s, name).offset for name, _ in s._fields_]
    assert got == want


@pytest.mark.parametrize("dtype,dim,page,heads,want", [
    ("f32", 256, 16, 1, 16 * 2 * 1024),
    ("bf16", 128, 16, 8, 8 * 16 * 2 * 256),
    ("f16", 96, 24, 3, 3 * 24 * 2 * 192),
    ("q8_0", 64, 1, 2, 2 * (2 * 64 + 2 * 8)),
    ("q8_0", 96, 7, 1, 7 * (2 * 96 + 2 * 16)),
    ("q4_0", 128, 64, 8, 8 * 64 * (2 * 64 + 2 * 16)),
    ("q4_0", 192, 5, 1, 5 * (2 * 96 + 2 * 32)),
    ("q4_0", 256, 4096, 1, 4096 * (2 * 128 + 2 * 32)),
])
def test_page_bytes(sp, dtype, dim, page, heads, want):
    from sapphire_b200.attention import kv_page_bytes
    assert kv_page_bytes(dtype, page, heads, dim) == want


@pytest.mark.parametrize("dtype,dim,page,heads", [
    ("tq2_0", 128, 16, 8), ("bf16", 80, 16, 8), ("q8_0", 32, 16, 8), ("q8_0", 128, 0, 8), ("q8_0", 128, 4097, 8),
    ("q8_0", 128, -1, 8), ("f32", 128, 16, 0), ("f32", 512, 16, 1),
])
def test_page_shapes_refused(sp, dtype, dim, page, heads):
    from sapphire_b200.attention import kv_page_bytes
    with pytest.raises(sp.SapphireError):
        kv_page_bytes(dtype, page, heads, dim)


@pytest.mark.parametrize("name", ["sapphire_rope_device", "sapphire_kv_write_device", "sapphire_kv_read_device",
                                  "sapphire_attention_device"])
def test_null_arguments(sp, name):
    fn = getattr(sp.lib, name)
    assert fn(*[None] * len(fn.argtypes)) == -1


def test_null_plan_and_workspace(sp):
    assert not sp.lib.sapphire_rope_create(None, None)
    sp.lib.sapphire_rope_destroy(None)
    assert sp.lib.sapphire_kv_page_bytes(None) == 0
    assert sp.lib.sapphire_attention_workspace_bytes(None, None, 1, 1) == 0


def test_uninitialised_context(sp):
    from sapphire_b200 import _lib
    ctx = sp.Context(num_threads=1, init=False)
    cfg = _lib.RopeConfig(128, 0, 0, 0, 1e4, 1.0, 0, 0, 0, 0)
    assert not sp.lib.sapphire_rope_create(ctx.handle, C.byref(cfg))
    assert "not initialized" in ctx.last_error
    kv = _lib.KvCacheStruct(1, 16, 1, 128, 4, 4096)
    for fn, args in ((sp.lib.sapphire_kv_write_device, _lib.KvArgs()), (sp.lib.sapphire_kv_read_device, _lib.KvArgs()),
                     (sp.lib.sapphire_attention_device, _lib.AttentionArgs())):
        assert fn(ctx.handle, C.byref(kv), C.byref(args)) == -1
        assert "not initialized" in ctx.last_error
    ctx.close()


@pytest.mark.parametrize("change,message", [
    ({"head_dim": 127}, "head_dim"), ({"head_dim": 514}, "head_dim"), ({"rot_dim": 130}, "rot_dim"),
    ({"rot_dim": 63}, "rot_dim"), ({"layout": 2}, "layout"), ({"scaling": 4}, "scaling"), ({"theta": 1.0}, "theta"),
    ({"theta": float("nan")}, "theta"), ({"scaling": 1, "factor": 0.5}, "factor"),
    ({"scaling": 2, "factor": 2.0, "original_context": 0}, "original_context"),
    ({"scaling": 3, "factor": 2.0, "original_context": 8192, "turns_slow": 8.0, "turns_fast": 2.0}, "turns"),
    ({"attention_factor": -1.0}, "attention_factor"),
])
def test_rope_configs_refused(sp, change, message):
    from sapphire_b200 import _lib
    ctx = sp.Context(num_threads=1, init=False)
    cfg = _lib.RopeConfig(128, 0, 0, 0, 1e4, 1.0, 0, 0, 0, 0)
    for k, v in change.items():
        setattr(cfg, k, v)
    assert not sp.lib.sapphire_rope_create(ctx.handle, C.byref(cfg))
    assert message in ctx.last_error
    ctx.close()


@pytest.mark.parametrize("bytes_", ["expanded", "strided"])
def test_workspaces_whose_bytes_do_not_lie_together_are_refused(sp, bytes_):
    """Its size is counted from its elements, so they have to be the bytes behind its address."""
    torch = pytest.importorskip("torch")
    from sapphire_b200.attention import KVCache, kv_page_bytes
    ctx = sp.Context(num_threads=1, init=False)
    kv = KVCache(ctx, "bf16", 16, 1, 64, torch.zeros(2, kv_page_bytes("bf16", 16, 1, 64), dtype=torch.uint8))
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.uint8)
    ws = one.expand(1 << 24) if bytes_ == "expanded" else torch.zeros(1 << 12, 2, dtype=torch.uint8)[:, 0]
    with pytest.raises(sp.SapphireError, match="contiguous"):
        kv.attend(q, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.empty_like(q), workspace=ws)
    ctx.close()

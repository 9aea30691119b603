"""Entry points of attention to selected pages without a GPU: the struct as C
lays it out, sizes of summaries, and refusals that come before any device work."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest

from conftest import ROOT


def test_struct_layout_matches_c(tmp_path, sp):
    from sapphire_b200 import _lib
    s = _lib.KvSelectArgs
    lines = ['#include <stdio.h>', '#include "sapphire_attention.h"', "int main(void) {",
             'printf("%zu\\n", sizeof(sapphire_kv_select_args_t));']
    lines += [f'printf("%zu\\n", offsetof(sapphire_kv_select_args_t, {name}));' for name, _ in s._fields_]
    src = tmp_path / "t.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), "-o", str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(s)] + [getattr(s, name).offset for name, _ in s._fields_]


@pytest.mark.parametrize("dtype,dim,page,heads,want", [
    ("f32", 256, 16, 1, 512 + 16), ("bf16", 128, 16, 8, 8 * 256 + 32), ("q4_0", 96, 1, 3, 3 * 192 + 16), ("q8_0", 64, 4096, 5, 5 * 128 + 32),
])
def test_summary_bytes(sp, dtype, dim, page, heads, want):
    from sapphire_b200 import _lib
    from sapphire_b200.attention import _dtype
    assert sp.lib.sapphire_kv_summary_bytes(C.byref(_lib.KvCacheStruct(_dtype(dtype), page, heads, dim, 0, None))) == want


@pytest.mark.parametrize("dtype,dim,page,heads", [(5, 128, 16, 8), (1, 80, 16, 8), (4, 128, 0, 8), (0, 128, 16, 0)])
def test_summary_shapes_refused(sp, dtype, dim, page, heads):
    from sapphire_b200 import _lib
    assert sp.lib.sapphire_kv_summary_bytes(C.byref(_lib.KvCacheStruct(dtype, page, heads, dim, 0, None))) == 0
    assert sp.lib.sapphire_kv_summary_bytes(None) == 0


@pytest.mark.parametrize("name", ["sapphire_kv_summarise_device", "sapphire_kv_select_device", "sapphire_attention_per_head_device"])
def test_null_arguments_and_uninitialised_contexts(sp, name):
    from sapphire_b200 import _lib
    fn = getattr(sp.lib, name)
    assert fn(*[None] * len(fn.argtypes)) == -1
    ctx = sp.Context(num_threads=1, init=False)
    kv = _lib.KvCacheStruct(1, 16, 1, 128, 4, 4096)
    args = {"sapphire_kv_summarise_device": (None, C.byref(_lib.KvArgs())),
            "sapphire_kv_select_device": (C.byref(_lib.KvSelectArgs()),),
            "sapphire_attention_per_head_device": (C.byref(_lib.AttentionArgs()),)}[name]
    assert fn(ctx.handle, C.byref(kv), *args) == -1
    assert "not initialized" in ctx.last_error
    ctx.close()

"""Entry points of attention behind a shared prefix without a GPU: the struct as C
lays it out, and refusals that come before any device work."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest

from conftest import ROOT


def test_struct_layout_matches_c(tmp_path, sp):
    from sapphire_b200 import _lib
    s = _lib.AttentionSharedArgs
    lines = ['#include <stdio.h>', '#include "sapphire_attention.h"', "int main(void) {",
             'printf("%zu\\n", sizeof(sapphire_attention_shared_args_t));']
    lines += [f'printf("%zu\\n", offsetof(sapphire_attention_shared_args_t, {name}));' for name, _ in s._fields_]
    src = tmp_path / "t.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), "-o", str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(s)] + [getattr(s, name).offset for name, _ in s._fields_]


def test_null_arguments_and_uninitialised_contexts(sp):
    from sapphire_b200 import _lib
    fn = sp.lib.sapphire_attention_shared_device
    assert fn(None, None, None) == -1
    assert sp.lib.sapphire_attention_shared_workspace_bytes(None, None, 1, 1, 1) == 0
    ctx = sp.Context(num_threads=1, init=False)
    kv = _lib.KvCacheStruct(1, 16, 1, 128, 4, 4096)
    assert fn(ctx.handle, C.byref(kv), C.byref(_lib.AttentionSharedArgs())) == -1
    assert "not initialized" in ctx.last_error
    ctx.close()


@pytest.mark.parametrize("bytes_", ["expanded", "strided"])
def test_workspaces_whose_bytes_do_not_lie_together_are_refused(sp, bytes_):
    torch = pytest.importorskip("torch")
    from sapphire_b200.attention import KVCache, kv_page_bytes
    ctx = sp.Context(num_threads=1, init=False)
    kv = KVCache(ctx, "bf16", 16, 1, 64, torch.zeros(2, kv_page_bytes("bf16", 16, 1, 64), dtype=torch.uint8))
    q, one = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.uint8)
    ws = one.expand(1 << 24) if bytes_ == "expanded" else torch.zeros(1 << 12, 2, dtype=torch.uint8)[:, 0]
    n = torch.ones(1, dtype=torch.int32)
    with pytest.raises(sp.SapphireError, match="contiguous"):
        kv.attend_shared(q, torch.zeros(1, dtype=torch.int32), n, torch.zeros(1, 1, dtype=torch.int32), n, torch.empty_like(q), workspace=ws)
    ctx.close()

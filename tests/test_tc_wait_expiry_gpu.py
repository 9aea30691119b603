"""Waits of the tensor-core kernels made to run out on purpose, without any GPU fault:
a barrier that a test hook leaves without an arrival, and a limit of 1 ms."""
from __future__ import annotations

import time

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_attention_gpu import dev_ctx  # noqa: E402,F401
from test_shared_prefix_gpu import shared_case  # noqa: E402

Q4_0 = 3


@pytest.fixture
def unarmed(sp):
    """Sets the hook; back to normal at the end whatever happens."""
    yield sp.lib.sapphire_test_tc_unarmed
    sp.lib.sapphire_test_tc_unarmed(0)


@pytest.mark.parametrize("rows,cols,batch", [(256, 64, 16), (2048, 640, 600), (2048, 64, 2560)])
def test_prefill_product_reports_and_recovers(sp, ctx, oracle, unarmed, rows, cols, batch):
    """The first stage of the first block never lands: fewer stages than the ring has, more, several tiles a block."""
    rng = np.random.default_rng(rows + cols)
    packed = oracle.quantize(Q4_0, (rng.standard_normal((rows, cols)) * 0.02).astype(np.float32))
    A = sp.Tensor(Q4_0, (rows, cols), packed)
    X = rng.standard_normal((batch, cols)).astype(np.float32)
    want = sp.gemm(ctx, A, X, batch)
    x, y = torch.from_numpy(X).cuda(), torch.zeros(batch, rows, device="cuda")
    torch.cuda.synchronize()
    unarmed(1)
    assert sp.lib.kernel_gemm_device(ctx.handle, y.data_ptr(), A.handle, x.data_ptr(), batch) == 0
    t0 = time.perf_counter()
    assert sp.lib.kernel_ctx_synchronize(ctx.handle) == -1
    elapsed = time.perf_counter() - t0
    assert "bounded wait expired" in ctx.last_error
    assert elapsed < 0.1, elapsed               # a wait of 1 ms, then one for the copies that never came
    unarmed(0)
    assert sp.lib.kernel_ctx_synchronize(ctx.handle) == 0
    for _ in range(2):
        assert np.array_equal(sp.gemm(ctx, A, X, batch), want)


def test_prefill_product_waits_little_longer_than_its_limit(sp, ctx, oracle, unarmed):
    """Two waits of 1 ms behind one another: 2 ms, and 16 where the timer is read between thousands of tries."""
    rng = np.random.default_rng(1)
    A = sp.Tensor(Q4_0, (256, 640), oracle.quantize(Q4_0, (rng.standard_normal((256, 640)) * 0.02).astype(np.float32)))
    x, y = torch.randn(16, 640, device="cuda"), torch.zeros(16, 256, device="cuda")

    def run():
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        assert sp.lib.kernel_gemm_device(ctx.handle, y.data_ptr(), A.handle, x.data_ptr(), 16) == 0
        return sp.lib.kernel_ctx_synchronize(ctx.handle), time.perf_counter() - t0

    for _ in range(2):
        assert run()[0] == 0
    unarmed(1)
    times = [run() for _ in range(5)]
    assert all(rc == -1 for rc, _ in times)
    assert min(t for _, t in times) < 8e-3, times


@pytest.mark.parametrize("which", [1, 2, 3])
@pytest.mark.parametrize("dtype,kind,seqs,prefix", [("bf16", "bf16", 2, 300), ("bf16", "bf16", 40, 20000), ("f16", "f16", 70, 5000), ("q8_0", "bf16", 40, 5000),
                                                    ("q4_0", "f16", 2, 300), ("f32", "bf16", 40, 2000), ("bf16", "f16", 70, 700)])
def test_shared_prefix_reports_and_recovers(sp, dev_ctx, unarmed, dtype, kind, seqs, prefix, which):
    """A warp of the first block withholds its first queries, probabilities or rows: short pieces and long ones, one tile
    of rows and two, rows that are copied and that are converted."""
    kv, prefix_table, table, q = shared_case(dev_ctx, dtype, kind, prefix, [3] * seqs, 2, 4, 128, 16, seed=seqs)
    n, m = torch.full((seqs,), 3, dtype=torch.int32, device="cuda"), torch.tensor([prefix], dtype=torch.int32, device="cuda")
    ws = torch.zeros(kv.shared_workspace_bytes(kind, seqs, 8), dtype=torch.uint8, device="cuda")

    def run():
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        kv.attend_shared(q, prefix_table, m, table, n, out, workspace=ws)
        try:
            dev_ctx.synchronize()
        finally:
            run.elapsed = time.perf_counter() - t0
        return out

    want = run()
    unarmed(which)
    times = []
    for _ in range(2):
        with pytest.raises(sp.SapphireError, match="bounded wait expired"):
            run()
        times.append(run.elapsed)
    assert min(times) < 0.01, times                 # 1.4 ms, and 32 where the timer is read once in 4096 tries
    unarmed(0)
    dev_ctx.synchronize()
    for _ in range(2):
        assert torch.equal(run(), want)

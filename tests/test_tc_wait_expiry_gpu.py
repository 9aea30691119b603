"""Waits of the tensor-core kernels made to run out on purpose, without any GPU fault:
a barrier that a test hook leaves without an arrival, and a limit of 1 ms."""
from __future__ import annotations

import time

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

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

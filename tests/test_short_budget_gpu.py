"""Norm, its gradient and the grouped products with a wait budget of a nanosecond: a call either finishes (its
values are right) or says which wait gave up, its copies in flight land all the same, and the next
call under the usual budget is right."""
import pytest

import bwgemm

pytestmark = pytest.mark.gpu
USUAL = 2_000_000_000


@pytest.fixture
def short_budget():
    bwgemm.set_wait_budget_ns(1)
    yield
    bwgemm.set_wait_budget_ns(USUAL)


def _try(call, sites):
    """Runs `call` under both budgets, several times in a row (the kernels follow each other without a pause)."""
    import torch

    bwgemm.set_wait_budget_ns(USUAL)
    want = call()
    assert bwgemm.device_status() == 0
    bwgemm.set_wait_budget_ns(1)
    for _ in range(3):
        got = [call() for _ in range(4)]
        status = bwgemm.device_status()
        assert status == 0 or (status >> 8 == bwgemm.BW_ERR_TIMEOUT and status & 255 in sites), hex(status)
        if status == 0:
            assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    bwgemm.set_wait_budget_ns(USUAL)
    got = [call() for _ in range(3)]
    assert bwgemm.device_status() == 0
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


@pytest.mark.parametrize("rows,cols", [(1201, 1088), (1203, 1111), (601, 4097), (150, 16384)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_norm(cuda_dev, short_budget, rows, cols, dtype):
    import torch

    g = torch.Generator(device=cuda_dev).manual_seed(rows)
    x, r = (torch.randn(rows, cols, device=cuda_dev, generator=g).to(getattr(torch, dtype)) for _ in range(2))
    w = torch.ones(cols, device=cuda_dev, dtype=x.dtype)
    _try(lambda: bwgemm.rmsnorm_fp8(x, w, residual=r), {71})


@pytest.mark.parametrize("rows,cols", [(9601, 600), (2371, 4609), (1301, 9000)])
def test_gradient(cuda_dev, short_budget, rows, cols):
    import torch

    g = torch.Generator(device=cuda_dev).manual_seed(rows)
    dy, h, r = (torch.randn(rows, cols, device=cuda_dev, generator=g).bfloat16() for _ in range(3))
    w = torch.ones(cols, device=cuda_dev).bfloat16()
    rstd = h.float().square().mean(1).rsqrt()
    _try(lambda: bwgemm.rmsnorm_backward(dy, h, w, rstd, dresidual=r), {72})


@pytest.mark.parametrize("pair", ["0", "1"])
def test_grouped(cuda_dev, short_budget, monkeypatch, pair):
    import torch

    monkeypatch.setenv("BW_GROUPED_PAIR", pair)
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    off = torch.tensor([0, 300, 301, 1000, 2000], dtype=torch.int32, device=cuda_dev)
    a = torch.randn(2000, 1024, device=cuda_dev, generator=g).bfloat16()
    b = torch.randn(4, 768, 1024, device=cuda_dev, generator=g).bfloat16()
    y = torch.randn(2000, 512, device=cuda_dev, generator=g).bfloat16()
    sites = {61, 62, 63, 64, 65, 66} if pair == "1" else {21, 22, 23, 24, 25, 26}
    _try(lambda: (bwgemm.gemm_grouped(a, b, off, b_transposed=True),), sites)
    _try(lambda: (bwgemm.gemm_grouped_wgrad(a, y, off),), sites)

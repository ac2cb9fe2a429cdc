"""Norm and gradient of 16-bit rows with an FP32 weight on every path: registers, shared memory (many rows), long
rows; whole vectors, rows behind a boundary, and tensors of different alignment. Against the 64-bit formulas."""
import pytest

import bwgemm
from test_norm_gpu import EPS, _check_backward, _check_forward, _check_fp8, _inputs

pytestmark = pytest.mark.gpu

# few rows; many rows through shared memory, aligned and not, two and four vectors a thread; rows too long for registers
SHAPES = [(1, 64), (5, 33), (40, 8192), (4000, 256), (1201, 1088), (1203, 1111), (601, 4097), (9601, 600), (9475, 1023),
          (2401, 4608), (1301, 9000), (150, 16384), (149, 16383), (3, 20000), (3, 20001), (2, 40960)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("residual", [False, True])
def test_fp32_weight(cuda_dev, rows, cols, dtype, residual):
    import torch

    x, r, w = _inputs(cuda_dev, getattr(torch, dtype), rows, cols, residual, wdtype=torch.float32, seed=rows + cols)
    y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, eps=EPS)
    _check_forward(x, r, w, y, h, rstd)
    q, s, h, rstd = bwgemm.rmsnorm_fp8(x, w, residual=r, eps=EPS)
    _check_fp8(x, r, w, q, s, h, rstd)
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    dy = torch.randn(rows, cols, device=cuda_dev, generator=g).to(x.dtype)
    dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd, dresidual=r)
    _check_backward(dy, h, w, rstd, r, dx, dw)
    again, dw2 = bwgemm.rmsnorm_backward(dy, h, w, rstd, dresidual=r)
    assert torch.equal(dx, again) and torch.equal(dw, dw2)
    assert bwgemm.device_status() == 0


@pytest.mark.parametrize("rows,cols", [(9, 300), (9, 9000), (1300, 1500)])
def test_fp32_weight_of_another_alignment(cuda_dev, rows, cols):
    """The weights 4 bytes behind a vector's boundary, the rows on it; and every tensor at a distance of its own."""
    import torch

    x, r, w = _inputs(cuda_dev, torch.bfloat16, rows, cols, True, wdtype=torch.float32, seed=1)
    behind = torch.zeros(cols + 1, device=cuda_dev)
    behind[1:] = w
    other = torch.zeros(rows * cols + 3, dtype=x.dtype, device=cuda_dev)[3:].view(rows, cols)
    other.copy_(x)
    for xs in (x, other):
        y, h, rstd = bwgemm.rmsnorm(xs, behind[1:], residual=r, eps=EPS)
        _check_forward(x, r, w, y, h, rstd)
        q, s, h, rstd = bwgemm.rmsnorm_fp8(xs, behind[1:], residual=r, eps=EPS)
        _check_fp8(x, r, w, q, s, h, rstd)
        dx, dw = bwgemm.rmsnorm_backward(xs, h, behind[1:], rstd, dresidual=r)
        _check_backward(x, h, w, rstd, r, dx, dw)


def test_streams_by_handle(cuda_dev):
    """stream= takes a Stream, its handle as an int, and 0 for the default stream."""
    import torch

    x, r, w = _inputs(cuda_dev, torch.bfloat16, 300, 1024, True)
    off = torch.tensor([0, 100, 300], dtype=torch.int32, device=cuda_dev)
    b = torch.randn(2, 1024, 256, device=cuda_dev).bfloat16()
    want = bwgemm.rmsnorm(x, w, residual=r)[0]
    c = bwgemm.gemm_grouped(want, b, off)
    torch.cuda.synchronize()
    s = torch.cuda.Stream(cuda_dev)
    for stream in (s, s.cuda_stream, 0):
        y, _, _ = bwgemm.rmsnorm(x, w, residual=r, stream=stream)
        d = bwgemm.gemm_grouped(y, b, off, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(d, c)

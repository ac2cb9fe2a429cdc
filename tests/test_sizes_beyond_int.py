"""Sizes that do not fit the C interface's ints are refused, not cut to their low 32 bits (2^32 + 5 rows would be 5).
Expanded tensors: nothing of these sizes is allocated."""
import pytest

import bwgemm

BIG = (1 << 32) + 5


def _wide(rows, cols, dtype=None):
    import torch

    return torch.empty(1, 1, dtype=dtype).expand(rows, cols)


@pytest.mark.parametrize("rows,cols", [(BIG, 1), (1 << 31, 1), (1, BIG)])
def test_norm(rows, cols):
    import torch

    x, w = _wide(rows, cols), torch.empty(1).expand(cols)
    rstd = torch.empty(1).expand(rows)
    for call in (lambda: bwgemm.rmsnorm(x, w), lambda: bwgemm.rmsnorm_fp8(x, w), lambda: bwgemm.rmsnorm_backward(x, x, w, rstd),
                 lambda: bwgemm.rmsnorm_backward_workspace(rows, cols)):
        with pytest.raises(ValueError, match="2147483647"):
            call()
    assert bwgemm.rmsnorm_backward_workspace((1 << 31) - 1, 1) > 0


@pytest.mark.parametrize("rows,n,k", [(BIG, 8, 8), (4, BIG, 8), (4, 8, BIG), (4, 8, 1 << 31)])
def test_grouped(rows, n, k):
    import torch

    one = torch.empty(1, 1, 1, dtype=torch.bfloat16)
    off = torch.zeros(2, dtype=torch.int32)
    a = _wide(rows, k, torch.bfloat16)
    with pytest.raises(ValueError, match="2147483647"):
        bwgemm.gemm_grouped(a, one.expand(1, k, n), off)
    with pytest.raises(ValueError, match="2147483647"):
        bwgemm.gemm_grouped(a, one.expand(1, n, k), off, b_transposed=True)
    with pytest.raises(ValueError, match="2147483647"):
        bwgemm.gemm_grouped_wgrad(a, _wide(rows, n, torch.bfloat16), off)


def test_groups():
    import torch

    off = torch.zeros(1, dtype=torch.int32).expand(BIG)
    a, b = torch.empty(4, 8).bfloat16(), torch.empty(1, 1, 1).bfloat16().expand(BIG - 1, 8, 8)
    with pytest.raises(ValueError, match="2147483647"):
        bwgemm.gemm_grouped(a, b, off)
    with pytest.raises(ValueError, match="2147483647"):
        bwgemm.gemm_grouped_wgrad(a, a, off)

"""Scales of the grouped products whose product leaves FP32 although the result does not."""
import pytest

import bwgemm


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp8", "bfloat16"])
@pytest.mark.parametrize("out", [bwgemm.OUT_F32, bwgemm.OUT_BF16])
@pytest.mark.parametrize("rs,gs,size", [(1e-30, 1e-14, 128.0), (1e-12, 1e-30, 128.0), (3e-38, 1e-3, 16.0), (1e-42, 1e3, 128.0),
                                        (1e25, 1e20, 2.0 ** -9), (2e38, 3.0, 2.0 ** -9), (1e20, 1e-20, 1.0), (0.0, 1e30, 1.0),
                                        (1e-30, -1e-14, 128.0)])
def test_extreme_scales(cuda_dev, kind, out, rs, gs, size):
    """C = (sum * row_scale) * group_scale in 64 bits. Operands are `size` times 0, 1 or 2, so every sum is exact. Two
    FP32 products, or the product of the scales and one (2^-24 each; a factor or result under 2^-126 is a multiple of 2^-149),
    and the output's rounding: half a step, 2^-8 of the value (BF16) where that is a normal number."""
    import torch

    g = torch.Generator(device=cuda_dev).manual_seed(7)
    rows, n, k, offsets = 300, 136, 64, [0, 100, 101, 300]
    a = size * torch.randint(0, 3, (rows, k), device=cuda_dev, generator=g).float()
    b = size * torch.randint(0, 3, (3, n, k), device=cuda_dev, generator=g).float()
    if kind == "bfloat16" and size < 1:  # sums small enough that scales of over 1e38 fit
        a, b = a * 2.0 ** -24, b * 2.0 ** -24
    row = torch.ones(rows, device=cuda_dev)
    row[::2] = rs  # rows of both kinds in every warp
    group = torch.tensor([1.0, gs, gs], device=cuda_dev)
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_dev)
    if kind == "fp8":
        qa, qb = (t.to(torch.float8_e4m3fn) for t in (a, b))
        assert torch.equal(qa.float(), a) and torch.equal(qb.float(), b)
        qa, qb = qa.view(torch.uint8), qb.view(torch.uint8)
    else:
        qa, qb = a.bfloat16(), b.bfloat16()
        assert torch.equal(qa.float(), a) and torch.equal(qb.float(), b)
    C = bwgemm.gemm_grouped(qa, qb, off, b_transposed=True, row_scale=row, group_scale=group, out_dtype=out)
    want = torch.cat([a[i:j].double() @ b[e].double().T * row[i:j, None].double() * group[e].double()
                      for e, (i, j) in enumerate(zip(offsets, offsets[1:]))])
    fits = want.abs() < 3.3e38
    assert bool(torch.isinf(C[want.abs() > 3.5e38]).all())
    rel, least = (3 * 2.0 ** -24, 2.0 ** -148) if out == bwgemm.OUT_F32 else (2.0 ** -8 + 3 * 2.0 ** -24, 2.0 ** -133)
    d = (C.double() - want).abs()
    assert bool((d <= rel * want.abs() + least)[fits].all()), float((d / (want.abs() + least))[fits].max())

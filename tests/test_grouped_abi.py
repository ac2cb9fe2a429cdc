"""Refusals of the grouped products' entry points, before anything touches a GPU."""
import ctypes

import pytest

import bwgemm

INVALID, OK = bwgemm.BW_ERR_INVALID, bwgemm.BW_OK
F16, BF16, FP8 = bwgemm.DTYPE_F16, bwgemm.DTYPE_BF16, bwgemm.DTYPE_FP8


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096)
    p.keep = buf
    return (ctypes.addressof(buf) + 255) & ~255


def _mul(p, **kw):
    a = dict(dtype=F16, A=p, lda=16, B=p, t=0, off=p, groups=2, rs=p, gs=p, C=p, ldc=16, out=1, rows=4, N=16, K=16)
    a.update(kw)
    return bwgemm.lib().bw_gemm_grouped(a["dtype"], a["A"], a["lda"], a["B"], a["t"], a["off"], a["groups"], a["rs"],
                                        a["gs"], a["C"], a["ldc"], a["out"], a["rows"], a["N"], a["K"], None)


@pytest.mark.parametrize("bad", [dict(dtype=bwgemm.DTYPE_F32), dict(dtype=bwgemm.DTYPE_MXFP4), dict(dtype=-1),
                                 dict(dtype=FP8), dict(out=2), dict(rows=-1), dict(N=-1), dict(K=-1), dict(groups=0),
                                 dict(groups=-3), dict(groups=1025), dict(off=None), dict(rows=2 ** 31 - 1),
                                 dict(N=2 ** 31 - 8, ldc=2 ** 31), dict(K=2 ** 31 - 16, lda=2 ** 31), dict(A=None), dict(B=None),
                                 dict(C=None), dict(lda=15), dict(lda=8), dict(lda=20), dict(ldc=15), dict(N=12),
                                 dict(t=1, K=12), dict(t=1, dtype=FP8, K=8, lda=16), dict(t=1, dtype=FP8, lda=24)])
def test_refuses(p, bad):
    assert _mul(p, **bad) == INVALID
    assert bwgemm.lib().bw_last_error_string()


def test_alignment_and_empty(p):
    for k, by in (("A", 8), ("B", 8), ("C", 1), ("off", 2), ("rs", 1), ("gs", 2)):
        assert _mul(p, **{k: p + by}) == INVALID, k
    assert _mul(p, rows=0, A=None, C=None) == OK and _mul(p, N=0, B=None, C=None) == OK


def _wgrad(p, **kw):
    a = dict(dtype=BF16, X=p, ldx=16, Y=p, ldy=16, off=p, groups=2, D=p, out=0, rows=4, M=16, N=16)
    a.update(kw)
    return bwgemm.lib().bw_gemm_grouped_wgrad(a["dtype"], a["X"], a["ldx"], a["Y"], a["ldy"], a["off"], a["groups"],
                                              a["D"], a["out"], a["rows"], a["M"], a["N"], None)


@pytest.mark.parametrize("bad", [dict(dtype=FP8), dict(dtype=bwgemm.DTYPE_F32), dict(out=3), dict(rows=-1), dict(M=-1),
                                 dict(N=-1), dict(groups=0), dict(groups=1025), dict(off=None), dict(X=None),
                                 dict(Y=None), dict(D=None), dict(ldx=15), dict(ldy=8), dict(ldx=20), dict(ldy=17)])
def test_wgrad_refuses(p, bad):
    assert _wgrad(p, **bad) == INVALID


def test_wgrad_alignment_and_empty(p):
    for k, by in (("X", 8), ("Y", 2), ("D", 2), ("off", 1)):
        assert _wgrad(p, **{k: p + by}) == INVALID, k
    assert _wgrad(p, M=0, D=None) == OK and _wgrad(p, N=0, D=None) == OK


def test_sharded_gemm_still_refuses_the_new_types(p):
    s = bwgemm.Shard(0, p, p, None, None, None, None, p, None, None)
    for dt in (BF16, bwgemm.DTYPE_F32):
        assert bwgemm.lib().bw_gemm_sharded(dt, 0, ctypes.byref(s), 1, 8, 8, 8, 0) == INVALID


def test_python_refuses():
    import torch

    A, B, off = torch.ones(4, 16).half(), torch.ones(2, 16, 8).half(), torch.tensor([0, 2, 4], dtype=torch.int32)
    f = bwgemm.gemm_grouped
    with pytest.raises(ValueError, match="CUDA"):
        f(A, B, off)
    for bad, err in [((A.float(), B, off), TypeError), ((A, B.bfloat16(), off), TypeError), ((A, B[0], off), ValueError),
                     ((A, B, off.long()), TypeError), ((A, B, off[:2]), ValueError), ((A, B, off[:1]), ValueError),
                     ((A[:, :8], B, off), ValueError), ((A.t().contiguous().t(), B, off), ValueError),
                     ((A, B.transpose(1, 2), off), ValueError)]:
        with pytest.raises(err):
            f(*bad)
    with pytest.raises(ValueError):
        f(A, B, off, row_scale=torch.ones(3))
    with pytest.raises(TypeError):
        f(A, B, off, group_scale=torch.ones(2).half())
    with pytest.raises(ValueError):
        f(A, B, off, out_dtype=7)
    with pytest.raises(TypeError):
        bwgemm.gemm_grouped_wgrad(A, A.bfloat16(), off)
    with pytest.raises(ValueError):
        bwgemm.gemm_grouped_wgrad(A, A[:3], off)
    with pytest.raises(TypeError):
        bwgemm.gemm_grouped_wgrad(A.view(torch.uint8), A.view(torch.uint8), off)

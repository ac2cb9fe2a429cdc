"""Refusals of the root-mean-square norm's entry points, before anything touches a GPU."""
import ctypes

import pytest

import bwgemm

INVALID, OK = bwgemm.BW_ERR_INVALID, bwgemm.BW_OK
F32, F16, BF16 = bwgemm.DTYPE_F32, bwgemm.DTYPE_F16, bwgemm.DTYPE_BF16


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096)
    p.keep = buf
    return (ctypes.addressof(buf) + 255) & ~255


def _fwd(p, q8=False, **kw):
    a = dict(x=p, ldx=8, res=p, ldr=8, w=p, dtype=F16, wdtype=F16, eps=1e-5, y=p, ldy=8, s=p, h=p, ldh=8, rstd=p, rows=2,
             cols=8)
    a.update(kw)
    L = bwgemm.lib()
    head = (a["x"], a["ldx"], a["res"], a["ldr"], a["w"], a["dtype"], a["wdtype"], a["eps"], a["y"], a["ldy"])
    tail = (a["h"], a["ldh"], a["rstd"], a["rows"], a["cols"], None)
    return L.bw_rmsnorm_fp8(*head, a["s"], *tail) if q8 else L.bw_rmsnorm(*head, *tail)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("bad", [dict(dtype=bwgemm.DTYPE_FP8), dict(dtype=17), dict(wdtype=BF16), dict(rows=-1), dict(cols=-1),
                                 dict(cols=0), dict(eps=-1e-5), dict(eps=float("nan")), dict(eps=float("inf")),
                                 dict(x=None), dict(w=None), dict(y=None), dict(ldx=7), dict(ldr=7), dict(ldy=7),
                                 dict(ldh=7), dict(ldx=0)])
def test_forward_refuses(p, q8, bad):
    assert _fwd(p, q8, **bad) == INVALID
    assert bwgemm.lib().bw_last_error_string()


def test_forward_alignment_and_empty(p):
    for k in ("x", "res", "w", "y", "h"):
        assert _fwd(p, **{k: p + 1}) == INVALID, k
    assert _fwd(p, rstd=p + 2) == INVALID and _fwd(p, True, s=p + 2) == INVALID and _fwd(p, True, s=None) == INVALID
    assert _fwd(p, rows=0, x=None, y=None) == OK  # nothing to do
    assert _fwd(p, rows=0, cols=0) == OK


def _bwd(p, **kw):
    a = dict(dy=p, lddy=8, h=p, ldh=8, w=p, dtype=BF16, wdtype=F32, rstd=p, dres=p, lddr=8, dx=p, lddx=8, dw=p, ws=p,
             nbytes=64, rows=2, cols=8)
    a.update(kw)
    return bwgemm.lib().bw_rmsnorm_backward(a["dy"], a["lddy"], a["h"], a["ldh"], a["w"], a["dtype"], a["wdtype"],
                                            a["rstd"], a["dres"], a["lddr"], a["dx"], a["lddx"], a["dw"], a["ws"],
                                            a["nbytes"], a["rows"], a["cols"], None)


@pytest.mark.parametrize("bad", [dict(dtype=bwgemm.DTYPE_MXFP4), dict(wdtype=F16), dict(rows=-1), dict(cols=0), dict(dy=None),
                                 dict(h=None), dict(w=None), dict(rstd=None), dict(dx=None), dict(dw=None), dict(ws=None),
                                 dict(nbytes=63), dict(lddy=7), dict(ldh=7), dict(lddr=7), dict(lddx=7)])
def test_backward_refuses(p, bad):
    assert _bwd(p, **bad) == INVALID


def test_workspace_size():
    f = bwgemm.lib().bw_rmsnorm_backward_workspace
    assert f(2, 8) == 64 and f(0, 8) == 0 and f(8, 0) == 0 and f(-1, 8) == 0
    assert f(100000, 1 << 20) == f(1000, 1 << 20) == 296 * 4 * (1 << 20)


def test_python_refuses():
    import torch

    x, w = torch.ones(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="CUDA"):
        bwgemm.rmsnorm(x, w)
    with pytest.raises(TypeError):
        bwgemm.rmsnorm(x.double(), w)
    with pytest.raises(TypeError):
        bwgemm.rmsnorm(x, w.half())
    with pytest.raises(TypeError):
        bwgemm.rmsnorm_fp8(x, w, residual=x.half())
    with pytest.raises(ValueError):
        bwgemm.rmsnorm(x, torch.ones(9))
    with pytest.raises(ValueError):
        bwgemm.rmsnorm(x[0], w)
    with pytest.raises(ValueError, match="contiguous"):
        bwgemm.rmsnorm(torch.ones(8, 4).t(), w)
    with pytest.raises(ValueError):
        bwgemm.rmsnorm_fp8(x, w, residual=torch.ones(4, 9))
    with pytest.raises(ValueError):
        bwgemm.rmsnorm_backward(x, x, w, torch.ones(5))
    with pytest.raises(TypeError):
        bwgemm.rmsnorm_backward(x.half(), x, w, torch.ones(4))

"""Root-mean-square norm with outputs over inputs: what is refused, and that an h which is returned is the h
that the gradient needs."""
import ctypes

import pytest

import bwgemm

INVALID = bwgemm.BW_ERR_INVALID
F16 = bwgemm.DTYPE_F16


@pytest.fixture(scope="module")
def at():
    """Addresses of buffers of their own."""
    buf = ctypes.create_string_buffer(1 << 14)
    at.keep = buf
    base = (ctypes.addressof(buf) + 255) & ~255
    return [base + 1024 * i for i in range(10)]


def _fwd(at, q8=False, **kw):
    a = dict(x=at[0], ldx=8, res=at[1], ldr=8, w=at[2], eps=1e-5, y=at[3], ldy=8, s=at[4], h=at[5], ldh=8, rstd=at[6], rows=2)
    a.update(kw)
    head = (a["x"], a["ldx"], a["res"], a["ldr"], a["w"], F16, F16, a["eps"], a["y"], a["ldy"])
    tail = (a["h"], a["ldh"], a["rstd"], a["rows"], 8, None)
    L = bwgemm.lib()
    return L.bw_rmsnorm_fp8(*head, a["s"], *tail) if q8 else L.bw_rmsnorm(*head, *tail)


def test_forward_refuses(at):
    x, r, _, y, _, h = at[:6]
    for q8 in (False, True):
        assert _fwd(at, q8, h=y) == INVALID and b"one buffer" in bwgemm.lib().bw_last_error_string()
        assert _fwd(at, q8, h=x, ldh=16) == INVALID and _fwd(at, q8, h=r, ldr=16) == INVALID
    assert _fwd(at, y=x, h=x) == INVALID and _fwd(at, y=r, h=r) == INVALID
    assert _fwd(at, y=x, ldy=16) == INVALID and _fwd(at, y=r, ldr=16) == INVALID
    assert _fwd(at, True, y=x) == INVALID and _fwd(at, True, y=r) == INVALID
    # one row has no pitch; outputs of their own have any
    assert _fwd(at, h=x, ldh=16, rows=1) != INVALID and _fwd(at, ldh=16, ldy=24) != INVALID


@pytest.mark.parametrize("which", ["dy", "h", "dres"])
def test_backward_refuses(at, which):
    def call(lddx, rows=2):
        a = dict(dy=at[0], h=at[1], dres=at[2])
        L = bwgemm.lib()
        return L.bw_rmsnorm_backward(a["dy"], 8, a["h"], 8, at[3], F16, F16, at[4], a["dres"], 8, a[which], lddx, at[5],
                                     at[6], 64, rows, 8, None)

    assert call(16) == INVALID and b"pitches" in bwgemm.lib().bw_last_error_string()
    assert call(8) != INVALID and call(16, rows=1) != INVALID


def _gradients64(x, w, dy, eps):
    import torch

    xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
    return torch.autograd.grad((xd * (xd.square().mean(1, keepdim=True) + eps).rsqrt() * wd * dy.double()).sum(), (xd, wd))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [24, 1000, 1024, 40000])
def test_gradient_behind_a_norm_in_place(cuda_dev, cols):
    """y over x, over the residual, with and without an h of the caller's: the h returned serves the gradient,
    or there is none."""
    import torch

    g = torch.Generator(device=cuda_dev).manual_seed(cols)
    x0, r0, dy = (torch.randn(6, cols, device=cuda_dev, generator=g) for _ in range(3))
    w = 1 + 0.1 * torch.randn(cols, device=cuda_dev, generator=g)

    def check(h, rstd, h64):
        dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd)
        ref = _gradients64(h64, w, dy, 1e-6)
        for got, want in zip((dx, dw), ref):
            # FP32 sums of `cols` or 6 terms of size 1: far below a thousandth of the gradients' size, and a wrong h is of that size
            assert float((got.double() - want).norm() / want.norm()) < 1e-5

    x = x0.clone()
    y, h, rstd = bwgemm.rmsnorm(x, w, y=x)
    assert y is x and h is None
    x, mine = x0.clone(), torch.empty_like(x0)
    y, h, rstd = bwgemm.rmsnorm(x, w, y=x, h=mine)
    assert h is mine and torch.equal(h, x0)
    check(h, rstd, x0)
    y, h, rstd = bwgemm.rmsnorm(x0, w)
    assert h is x0
    check(h, rstd, x0)
    for over in ("x", "residual"):
        x, r = x0.clone(), r0.clone()
        y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, y=x if over == "x" else r)
        assert torch.equal(h, x0 + r0)
        check(h, rstd, (x0 + r0))
    x = x0.clone()
    with pytest.raises(bwgemm.BwError, match="one buffer"):
        bwgemm.rmsnorm(x, w, y=x, h=x)
    assert torch.equal(x, x0)
    with pytest.raises(bwgemm.BwError, match="different size"):
        bwgemm.rmsnorm_fp8(x, w, q=x.view(torch.uint8)[:, :cols])
    assert torch.equal(x, x0)


@pytest.mark.gpu
def test_no_rows_keep_their_h(cuda_dev):
    import torch

    x, w = torch.empty(0, 16, device=cuda_dev), torch.ones(16, device=cuda_dev)
    for kw in ({}, {"y": x}):
        y, h, rstd = bwgemm.rmsnorm(x, w, **kw)
        dx, dw = bwgemm.rmsnorm_backward(y, h, w, rstd)
        assert dx.shape == (0, 16) and bool((dw == 0).all())

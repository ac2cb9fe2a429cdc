"""Root-mean-square norm (residual, 8-bit output with row scales, gradient) against the formulas in
64 bits.

Tolerances, with u = eps / 2 of the output's type (half a step) and u32 = 2^-24: h is one rounding
of an exact sum. rstd, row_scale: the FP32 sum of cols squares errs by at most (chain) u32, where a
thread adds its own elements one by one and the tree adds log2 more; rstd halves that, and takes a
division, a root and a reciprocal more. y: u of its type, plus rstd's error and two products. A code
q of |v| <= 448 stands within half an E4M3 step, 2^-4 |v| for normal codes and 2^-10 for subnormal
ones, of a v that itself carries those FP32 errors.
"""
import math

import pytest

import bwgemm

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
EPS = 1e-5
DTYPES = ["float32", "float16", "bfloat16"]


def _u(dtype):
    import torch

    return torch.finfo(dtype).eps / 2


def _stat_err(cols):
    # per-thread chain of at most 64 (registers) or cols / 1024 + 16 (long rows) sums, ten tree steps, mean,
    # eps, root, reciprocal, and the product that forms each square
    return (max(64, cols // 1024 + 16) + 10 + 6) * U32


def _inputs(dev, dtype, rows, cols, residual, wdtype=None, seed=0):
    import torch

    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, cols, device=dev, generator=g).to(dtype)
    r = (2 * torch.randn(rows, cols, device=dev, generator=g)).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(cols, device=dev, generator=g)).to(wdtype or dtype)
    return x, r, w


def _forward64(x, r, w, eps=EPS):
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    hd = h.double()
    rstd = (hd.square().mean(1) + eps) ** -0.5
    return h, rstd, hd * w.double() * rstd[:, None]


def _close(got, want, tol):
    d = (got.double() - want).abs()
    bad = d > tol
    assert not bool(bad.any()), f"off by {float((d - tol).max())} over its bound, {int(bad.sum())} values"


def _check_forward(x, r, w, y, h, rstd, eps=EPS):
    import torch

    h64, rstd64, y64 = _forward64(x, r, w, eps)
    assert torch.equal(h, h64)
    e = _stat_err(x.shape[1])
    _close(rstd, rstd64, e * rstd64)
    _close(y, y64, (_u(x.dtype) * 1.01 + e + 3 * U32) * y64.abs() + 2.0 ** -25 * (x.dtype == torch.float16))


def _check_fp8(x, r, w, q, s, h, rstd, eps=EPS):
    import torch

    h64, rstd64, y64 = _forward64(x, r, w, eps)
    assert torch.equal(h, h64)
    e = _stat_err(x.shape[1])
    _close(rstd, rstd64, e * rstd64)
    amax = y64.abs().amax(1)
    s64 = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    _close(s, s64, (e + 6 * U32) * s64)
    v = y64 / s64[:, None]
    _close(q.view(torch.float8_e4m3fn).float(), v, torch.clamp(2.0 ** -4 * v.abs(), min=2.0 ** -10) * (1 + 2.0 ** -10)
           + (e + 8 * U32) * v.abs())


SHAPES = [(1, 1), (3, 7), (5, 33), (1, 8192), (77, 128), (130, 136), (1030, 1000), (9, 2049), (2, 8193), (3, 20000),
          (2, 40960), (1025, 24), (1, 65), (4000, 256)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_forward(cuda_dev, rows, cols, dtype, residual):
    import torch

    x, r, w = _inputs(cuda_dev, getattr(torch, dtype), rows, cols, residual, seed=rows + cols)
    y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, eps=EPS)
    _check_forward(x, r, w, y, h, rstd)
    q, s, h8, rstd8 = bwgemm.rmsnorm_fp8(x, w, residual=r, eps=EPS)
    _check_fp8(x, r, w, q, s, h8, rstd8)
    assert torch.equal(rstd, rstd8)
    # the norm of x with a residual is the norm of the h that it keeps
    if residual:
        y2, _, rstd2 = bwgemm.rmsnorm(h, w, eps=EPS)
        assert torch.equal(y, y2) and torch.equal(rstd, rstd2)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_fp32_weight(cuda_dev, dtype):
    import torch

    x, r, w = _inputs(cuda_dev, getattr(torch, dtype), 33, 520, True, wdtype=torch.float32)
    y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, eps=EPS)
    _check_forward(x, r, w, y, h, rstd)
    q, s, h, rstd = bwgemm.rmsnorm_fp8(x, w, residual=r, eps=EPS)
    _check_fp8(x, r, w, q, s, h, rstd)
    dy = torch.randn_like(x)
    dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd)
    _check_backward(dy, h, w, rstd, None, dx, dw)


@pytest.mark.parametrize("cols,pad,shift", [(512, 8, 0), (512, 16, 8), (500, 12, 0), (512, 3, 1), (513, 0, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pitches_and_alignment(cuda_dev, cols, pad, shift, dtype):
    """Rows inside wider buffers, at every alignment; what lies around them stays as it was."""
    import torch

    dt, rows = getattr(torch, dtype), 37

    def window(kind, fill):
        whole = torch.full(((rows + 1) * (cols + pad) + 64,), fill, dtype=kind, device=cuda_dev)
        return whole, whole[16 + shift:16 + shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]

    x, r, w = _inputs(cuda_dev, dt, rows, cols, True)
    (_, xw), (_, rw), (by, yw), (bh, hw) = window(dt, 0), window(dt, 0), window(dt, 7), window(dt, 7)
    bq, qw = window(torch.uint8, 0x5A)
    xw.copy_(x), rw.copy_(r)
    y, h, rstd = bwgemm.rmsnorm(xw, w, residual=rw, eps=EPS, y=yw, h=hw)
    _check_forward(x, r, w, y, h, rstd)
    q, s, h, rstd = bwgemm.rmsnorm_fp8(xw, w, residual=rw, eps=EPS, q=qw, h=hw)
    _check_fp8(x, r, w, q, s, h, rstd)
    bd, dxw = window(dt, 7)
    dy = torch.randn_like(x)
    dx, dw = bwgemm.rmsnorm_backward(dy, hw, w, rstd, dresidual=rw, dx=dxw)
    _check_backward(dy, h, w, rstd, r, dx, dw)
    for whole, view, fill in ((by, yw, 7), (bh, hw, 7), (bq, qw, 0x5A), (bd, dxw, 7)):
        view.fill_(fill)
        assert bool((whole == fill).all())


@pytest.mark.parametrize("cols", [1, 5, 16, 300, 1500, 5000, 9000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tensors_of_different_alignment(cuda_dev, cols, dtype):
    """Each tensor at a distance of its own from a vector's boundary: element by element."""
    import torch

    dt, rows = getattr(torch, dtype), 9

    def place(src, shift, pad):
        whole = torch.zeros(rows * (cols + pad) + 32, dtype=src.dtype, device=cuda_dev)
        view = whole[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        view.copy_(src)
        return view

    x, r, w = _inputs(cuda_dev, dt, rows, cols, True)
    wide = torch.zeros(cols + 3, dtype=dt, device=cuda_dev)
    wide[3:] = w
    xs, rs = place(x, 1, 3), place(r, 2, 1)
    ys, hs, qs = place(x, 5, 0), place(x, 0, 8), place(x.to(torch.uint8), 3, 2)
    y, h, rstd = bwgemm.rmsnorm(xs, wide[3:], residual=rs, eps=EPS, y=ys, h=hs)
    _check_forward(x, r, w, y, h, rstd)
    q, s, h, rstd = bwgemm.rmsnorm_fp8(xs, wide[3:], residual=rs, eps=EPS, q=qs, h=hs)
    _check_fp8(x, r, w, q, s, h, rstd)
    dx, dw = bwgemm.rmsnorm_backward(place(x, 7, 0), h, wide[3:], rstd, dresidual=rs, dx=place(x, 2, 5))
    _check_backward(x, h, w, rstd, r, dx, dw)
    # one alignment for all rows, the weights at another
    y, h, rstd = bwgemm.rmsnorm(x, wide[3:], residual=r, eps=EPS)
    _check_forward(x, r, w, y, h, rstd)


def test_in_place(cuda_dev):
    """y over x, h over the residual, dx over dy: registers and long rows alike."""
    import torch

    for cols in (1000, 1024, 70001):
        x, r, w = _inputs(cuda_dev, torch.bfloat16, 5, cols, True)
        x0, r0 = x.clone(), r.clone()
        y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, eps=EPS, y=x, h=r)
        assert y is x and h is r
        _check_forward(x0, r0, w, y, h, rstd)
        dy = torch.randn_like(x)
        dy0 = dy.clone()
        dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd, dx=dy)
        _check_backward(dy0, h, w, rstd, None, dx, dw)
        y2, _, rstd2 = bwgemm.rmsnorm(r, w, eps=EPS, y=r)
        _check_forward(h.clone() if h is not r else (x0.double() + r0.double()).to(x.dtype), None, w, y2,
                       (x0.double() + r0.double()).to(x.dtype), rstd2)


def test_special_rows(cuda_dev):
    """All zeros, one NaN, one infinity, overflowing squares, a maximum too small to invert."""
    import torch

    x = torch.ones(6, 64, device=cuda_dev)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3] = 1e30
    x[4] = 1e-38
    w = torch.ones(64, device=cuda_dev)
    w[9] = 0
    q, s, h, rstd = bwgemm.rmsnorm_fp8(x, w, eps=1e-5)
    y, _, rstd_y = bwgemm.rmsnorm(x, w, eps=1e-5)
    f = q.view(torch.float8_e4m3fn).float()
    assert torch.equal(rstd.isnan(), rstd_y.isnan())
    assert bool((f[0] == 0).all()) and float(s[0]) == 1.0 and bool((y[0] == 0).all())
    assert bool(f[1].isnan().all()) and float(s[1]) == 1.0 and bool(y[1].isnan().all())
    assert float(rstd[2]) == 0 and float(s[2]) == 1.0 and bool(f[2, 5].isnan()) and bool(y[2, 5].isnan())
    assert int(f[2].isnan().sum()) == 1 and float(f[2].nan_to_num(0).abs().max()) == 0
    assert float(rstd[3]) == 0 and bool((y[3] == 0).all()) and bool((f[3] == 0).all())
    assert bool(torch.isfinite(f[4]).all()) and bool(torch.isfinite(s[4]))
    assert float(f[5].max()) == 448 and float(f[5, 9]) == 0
    tiny = torch.full((1, 64), 1e-40, device=cuda_dev)
    q, s, _, _ = bwgemm.rmsnorm_fp8(tiny, w, eps=1.0)
    assert float(s[0]) == 1.0 and bool((q == 0).all())


# ------------------------------------------------------------------ gradient
def _check_backward(dy, h, w, rstd, dres, dx, dw):
    """dx within u |dx| plus the FP32 errors of its terms; dw within the FP32 error of a chain over
    rows: at most rows / min(rows, 296) + 32 sums in one thread, slabs / 32 + 5 after it."""
    import torch

    rows, cols = h.shape
    n = h.double() * rstd.double()[:, None]
    g = dy.double() * w.double()
    mean = (g * n).mean(1, keepdim=True)
    want = rstd.double()[:, None] * (g - n * mean)
    mags = rstd.double()[:, None] * (g.abs() + n.abs() * (g * n).abs().mean(1, keepdim=True))
    if dres is not None:
        want = want + dres.double()
        mags = mags + dres.double().abs()
    _close(dx, want, _u(h.dtype) * 1.01 * want.abs() + (_stat_err(cols) + 8 * U32) * mags
           + 2.0 ** -25 * (h.dtype == torch.float16))
    t = dy.double() * n
    chain = rows / min(max(rows, 1), 296) + 32 + 296 / 32 + 5 + 8
    _close(dw, t.sum(0), chain * 4 * U32 * t.abs().sum(0))


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dres", [False, True])
def test_backward(cuda_dev, rows, cols, dtype, dres):
    import torch

    dt = getattr(torch, dtype)
    x, r, w = _inputs(cuda_dev, dt, rows, cols, dres, seed=rows * 3 + cols)
    _, h, rstd = bwgemm.rmsnorm(x, w, eps=EPS)
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    dy = torch.randn(rows, cols, device=cuda_dev, generator=g).to(dt)
    dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd, dresidual=r)
    _check_backward(dy, h, w, rstd, r, dx, dw)
    # the same bits again, from a workspace with other contents
    ws = torch.full((bwgemm.lib().bw_rmsnorm_backward_workspace(rows, cols),), 0xFF, dtype=torch.uint8, device=cuda_dev)
    dx2, dw2 = bwgemm.rmsnorm_backward(dy, h, w, rstd, dresidual=r, workspace=ws)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


def test_backward_against_differences(cuda_dev):
    """dx and dweight against central differences of the 64-bit forward formula."""
    import torch

    x, r, w = _inputs(cuda_dev, torch.float32, 3, 40, True)
    y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, eps=EPS)
    g = torch.Generator(device=cuda_dev).manual_seed(6)
    dy = torch.randn(3, 40, device=cuda_dev, generator=g)
    dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd)
    hd, wd = h.double(), w.double()

    def loss(hh, ww):
        return (dy.double() * hh * ww * ((hh.square().mean(1, keepdim=True) + EPS) ** -0.5)).sum()

    step = 1e-5
    for i, j in [(0, 0), (1, 17), (2, 39)]:
        e = torch.zeros_like(hd)
        e[i, j] = step
        num = (loss(hd + e, wd) - loss(hd - e, wd)) / (2 * step)
        assert abs(float(num) - float(dx[i, j])) <= 1e-5 * (1 + abs(float(num)))
        num = (loss(hd, wd + e[i]) - loss(hd, wd - e[i])) / (2 * step)
        assert abs(float(num) - float(dw[j])) <= 1e-5 * (1 + abs(float(num)))


@pytest.mark.parametrize("size", [1e-15, 1e-6, 1e6, 1e15])
def test_magnitudes(cuda_dev, size):
    """Rows of very small and very large values: no intermediate power of rstd leaves FP32."""
    import torch

    for cols in (64, 1001, 20000):
        x, r, w = _inputs(cuda_dev, torch.float32, 3, cols, True)
        x, r = x * size, r * size
        y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, eps=0.0)
        _check_forward(x, r, w, y, h, rstd, eps=0.0)
        q, s, h, rstd = bwgemm.rmsnorm_fp8(x, w, residual=r, eps=0.0)
        _check_fp8(x, r, w, q, s, h, rstd, eps=0.0)
        g = torch.Generator(device=cuda_dev).manual_seed(8)
        dy = torch.randn(3, cols, device=cuda_dev, generator=g)
        dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd)
        _check_backward(dy, h, w, rstd, None, dx, dw)


def test_zero_row_without_eps(cuda_dev):
    """0 / 0: NaN in the row, not in its neighbours."""
    import torch

    x = torch.ones(3, 40, device=cuda_dev)
    x[1] = 0
    w = torch.ones(40, device=cuda_dev)
    y, _, _ = bwgemm.rmsnorm(x, w, eps=0.0)
    q, s, _, _ = bwgemm.rmsnorm_fp8(x, w, eps=0.0)
    assert bool(y[1].isnan().all()) and bool((q[1] & 0x7F == 0x7F).all()) and float(s[1]) == 1.0
    assert bool((y[[0, 2]] == 1).all()) and bool((s[[0, 2]] == torch.tensor(1.0) / 448).all())


def test_capture_with_fork_and_join(cuda_dev):
    """Captured behind a copy, a memset and another stream's kernels: full dependencies are kept."""
    import torch

    w = torch.ones(512, device=cuda_dev, dtype=torch.bfloat16)
    src, res, dy = (torch.randn(300, 512, device=cuda_dev).bfloat16() for _ in range(3))
    x, r, g = torch.zeros_like(src), torch.zeros_like(src), torch.zeros_like(src)
    side = torch.cuda.Stream(cuda_dev)

    def work():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        x.copy_(src)
        with torch.cuda.stream(side):
            r.zero_()
            r.add_(res)
            g.copy_(dy)
        main.wait_stream(side)
        y, h, rstd = bwgemm.rmsnorm(x, w, residual=r)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            dx, dw = bwgemm.rmsnorm_backward(g, h, w, rstd)
        q, s, _, _ = bwgemm.rmsnorm_fp8(y, w)
        main.wait_stream(side)
        return y, dx, dw, q, s

    want = work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for _ in range(4):
        x.zero_(), r.fill_(5), g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_empty(cuda_dev):
    import torch

    x = torch.empty(0, 16, device=cuda_dev)
    w = torch.ones(16, device=cuda_dev)
    y, h, rstd = bwgemm.rmsnorm(x, w)
    assert y.shape == (0, 16) and rstd.shape == (0,)
    dw = torch.full((16,), 3.0, device=cuda_dev)
    bwgemm.rmsnorm_backward(x, x, w, rstd, dweight=dw)
    assert bool((dw == 0).all())


def test_graph_and_streams(cuda_dev):
    """Two captured graphs of the gradient, replayed on two streams at once, and an eager call."""
    import torch

    w = torch.ones(1024, device=cuda_dev, dtype=torch.bfloat16)
    sets, graphs = [], []
    for k in range(2):
        x, r, _ = _inputs(cuda_dev, torch.bfloat16, 700, 1024, True, seed=k)
        dy = torch.randn_like(x)
        s = torch.cuda.Stream(cuda_dev)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _, h, rstd = bwgemm.rmsnorm(x, w, residual=r)
            want = bwgemm.rmsnorm_backward(dy, h, w, rstd)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            _, hg, rg = bwgemm.rmsnorm(x, w, residual=r)
            got = bwgemm.rmsnorm_backward(dy, hg, w, rg)
        sets.append((s, want, got, (x, r, dy)))  # a graph reads its inputs at every replay
        graphs.append(g)
    for _ in range(5):
        for g, (s, *_) in zip(graphs, sets):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, want, got, _ in sets:
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    # stream= runs there, without a stream context of the caller's
    s = sets[0][0]
    x, r, _ = _inputs(cuda_dev, torch.bfloat16, 300, 1024, True, seed=9)
    torch.cuda.synchronize()
    y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, eps=EPS, stream=s)
    s.synchronize()
    _check_forward(x, r, w, y, h, rstd)


def test_large_offsets(cuda_dev):
    """Rows behind 2^31 elements."""
    import torch

    rows, cols = 3, 64
    pitch = 1_100_000_000
    buf = torch.zeros(2 * pitch + cols, dtype=torch.bfloat16, device=cuda_dev)
    x = buf.as_strided((rows, cols), (pitch, 1))
    src, _, w = _inputs(cuda_dev, torch.bfloat16, rows, cols, False)
    x.copy_(src)
    y, h, rstd = bwgemm.rmsnorm(x, w, eps=EPS)
    _check_forward(src, None, w, y, h, rstd)
    bwgemm.rmsnorm(x, w, eps=EPS, y=x)
    assert torch.equal(x, y)


# rows enough that a block takes several, out of its shared memory: whole vectors or not, 2 to 16 warps a row,
# one or more slots a block
@pytest.mark.parametrize("rows,cols", [(1201, 1088), (1203, 1111), (700, 2498), (601, 4097), (333, 9553), (150, 16384),
                                       (149, 16383), (2401, 520)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_many_rows(cuda_dev, rows, cols, dtype, residual):
    import torch

    x, r, w = _inputs(cuda_dev, getattr(torch, dtype), rows, cols, residual, seed=rows + cols)
    y, h, rstd = bwgemm.rmsnorm(x, w, residual=r, eps=EPS)
    _check_forward(x, r, w, y, h, rstd)
    q, s, h8, rstd8 = bwgemm.rmsnorm_fp8(x, w, residual=r, eps=EPS)
    _check_fp8(x, r, w, q, s, h8, rstd8)
    if residual:  # outputs over the inputs
        xi, ri = x.clone(), r.clone()
        yi, hi, rstdi = bwgemm.rmsnorm(xi, w, residual=ri, eps=EPS, y=xi, h=ri)
        assert torch.equal(yi, y) and torch.equal(hi, h) and torch.equal(rstdi, rstd)
    assert bwgemm.device_status() == 0


@pytest.mark.parametrize("rows,cols", [(9601, 600), (9475, 1023), (2401, 4608), (2371, 4609), (1301, 9000), (1190, 16384),
                                       (1185, 8191)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dres", [False, True])
def test_backward_many_rows(cuda_dev, rows, cols, dtype, dres):
    import torch

    dt = getattr(torch, dtype)
    h, res, w = _inputs(cuda_dev, dt, rows, cols, dres, seed=rows + cols)
    dy = torch.randn(rows, cols, device=cuda_dev).to(dt)
    rstd = (h.double().square().mean(1) + EPS).rsqrt().float()
    dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd, dresidual=res)
    _check_backward(dy, h, w, rstd, res, dx, dw)
    again, dw2 = bwgemm.rmsnorm_backward(dy, h, w, rstd, dresidual=res)
    assert torch.equal(dx, again) and torch.equal(dw, dw2)
    over, dw3 = bwgemm.rmsnorm_backward(dy.clone(), h, w, rstd, dresidual=None if res is None else res, dx=h.clone())
    assert torch.equal(over, dx) and torch.equal(dw3, dw)
    own = dy.clone()
    inplace, dw4 = bwgemm.rmsnorm_backward(own, h, w, rstd, dresidual=res, dx=own)
    assert torch.equal(inplace, dx) and torch.equal(dw4, dw)
    assert bwgemm.device_status() == 0


def test_many_rows_of_a_pitch(cuda_dev):
    """Rows inside wider buffers that start behind a vector's boundary, read through shared memory; what
    lies around the outputs stays as it was."""
    import torch

    rows, cols, pad, shift = 1203, 1500, 13, 3
    x, r, w = _inputs(cuda_dev, torch.bfloat16, rows, cols, True, seed=5)

    def window(src, kind, fill):
        whole = torch.full((rows * (cols + pad) + 64,), fill, dtype=kind, device=cuda_dev)
        view = whole[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        if src is not None:
            view.copy_(src)
        return whole, view

    xs, rs = window(x, x.dtype, 7.0)[1], window(r, x.dtype, 7.0)[1]
    hw, h = window(None, x.dtype, 5.0)
    qw, q = window(None, torch.uint8, 77)
    q, s, h, rstd = bwgemm.rmsnorm_fp8(xs, w, residual=rs, eps=EPS, q=q, h=h)
    _check_fp8(x, r, w, q.contiguous(), s, h, rstd)
    h.fill_(5.0)
    q.fill_(77)
    assert bool((hw == 5.0).all()) and bool((qw == 77).all())


def test_workspace_shared_by_captured_graphs(cuda_dev):
    """Two graphs over one workspace, replayed one after the other on one stream."""
    import torch

    rows, cols = 2401, 4608
    h, _, w = _inputs(cuda_dev, torch.bfloat16, rows, cols, False, seed=9)
    rstd = (h.double().square().mean(1) + EPS).rsqrt().float()
    dys = [torch.randn(rows, cols, device=cuda_dev).bfloat16() for _ in range(2)]
    want = [bwgemm.rmsnorm_backward(dy, h, w, rstd) for dy in dys]
    ws = torch.empty(bwgemm.rmsnorm_backward_workspace(rows, cols), dtype=torch.uint8, device=cuda_dev)
    outs = [(torch.empty_like(h), torch.empty(cols, device=cuda_dev)) for _ in dys]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graphs = []
    for dy, (dx, dw) in zip(dys, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            bwgemm.rmsnorm_backward(dy, h, w, rstd, dx=dx, dweight=dw, workspace=ws)
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (dx, dw), (dx0, dw0) in zip(outs, want):
        assert torch.equal(dx, dx0) and torch.equal(dw, dw0)

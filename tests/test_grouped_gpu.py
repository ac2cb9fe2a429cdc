"""Products grouped by expert (forward, input gradient, weight gradient) against 64-bit products.

Tolerance of one output: the tensor core adds K / 16 (E4M3: K / 32) k-steps into an FP32
accumulator, each of which may lose up to one last place (2^-23, it truncates) of a value that
never exceeds sum |a||b|, and as much again inside a step; then two scale products (2^-24 each) and the
rounding to the output's type (BF16: 2^-8 of the value).
"""
import pytest

import bwgemm

pytestmark = pytest.mark.gpu

F32, BF16 = bwgemm.OUT_F32, bwgemm.OUT_BF16
KINDS = ["float16", "bfloat16", "fp8"]


def _close(got, want, mag, ksteps, out):
    u = 2.0 ** -8 if out == BF16 else 0.0
    tol = 1.01 * u * want.abs() + ((2 * ksteps + 8) * 2.0 ** -23) * mag
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((d - tol).max())} over its bound"


def bounds_of(offsets, rows):
    """The rows that the kernel takes for each group: clamped to 0..rows, never decreasing."""
    out, high = [], 0
    for v in offsets:
        high = max(high, min(max(int(v), 0), rows))
        out.append(high)
    return out


def _make(dev, kind, layout, groups, rows, n, k, seed=0, pad=0):
    import torch

    g = torch.Generator(device=dev).manual_seed(seed)
    a = torch.randn(rows, k + pad, device=dev, generator=g)
    shape = (groups, n, k) if layout == "nk" else (groups, k, n)
    b = torch.randn(*shape, device=dev, generator=g)
    if kind == "fp8":
        rs = torch.rand(rows, device=dev, generator=g) + 0.5
        gs = torch.rand(groups, device=dev, generator=g) + 0.5
        a8, b8 = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
        return a8.view(torch.uint8)[:, :k], b8.view(torch.uint8), rs, gs, a8.double()[:, :k], b8.double()
    dt = getattr(torch, kind)
    a, b = a.to(dt), b.to(dt)
    return a[:, :k], b, None, None, a.double()[:, :k], b.double()


def _product(a, b, layout, bnd, rs, gs):
    """(value, sum of magnitudes), NaN outside every group."""
    import torch

    n = b.shape[1] if layout == "nk" else b.shape[2]
    want = torch.full((a.shape[0], n), float("nan"), dtype=torch.float64, device=a.device)
    mag = want.clone()
    for e in range(len(bnd) - 1):
        i, j = bnd[e], bnd[e + 1]
        m = b[e].T if layout == "nk" else b[e]
        s = (rs[i:j, None].double() if rs is not None else 1.0) * (gs[e].double() if gs is not None else 1.0)
        want[i:j] = a[i:j] @ m * s
        mag[i:j] = a[i:j].abs() @ m.abs() * s
    return want, mag


def _steps(kind, k):
    return -(-k // (32 if kind == "fp8" else 16))


def _check_rows(dev, kind, layout, offsets, rows, n, k, out, seed=0, pad=0, C=None):
    import torch

    groups = len(offsets) - 1
    a, b, rs, gs, ad, bd = _make(dev, kind, layout, groups, rows, n, k, seed, pad)
    off = torch.tensor(offsets, dtype=torch.int32, device=dev)
    if C is None:
        C = torch.full((rows, n), -77.0, dtype=torch.bfloat16 if out == BF16 else torch.float32, device=dev)
    bwgemm.gemm_grouped(a, b, off, C, b_transposed=layout == "nk", row_scale=rs, group_scale=gs, out_dtype=out)
    torch.cuda.synchronize()
    assert bwgemm.device_status() == 0
    bnd = bounds_of(offsets, rows)
    want, mag = _product(ad, bd, layout, bnd, rs, gs)
    inside = torch.zeros(rows, dtype=torch.bool, device=dev)
    inside[bnd[0]:bnd[-1]] = True
    _close(C[inside], want[inside], mag[inside], _steps(kind, k), out)
    assert bool((C[~inside] == -77.0).all())
    return C


ROWS = [
    ([0, 1], 1, 8, 16),                                        # one row
    ([0, 0, 1, 1, 1], 1, 4096, 512),                           # one token of several experts' batch
    ([0, 1, 2, 3, 4, 5, 6, 7, 8], 8, 520, 1040),
    ([0, 5, 5, 40, 40, 41, 169, 300], 300, 264, 96),           # empty groups, ragged, tiles that end inside
    ([3, 10, 130, 131, 390], 400, 640, 208),                   # rows before the first and behind the last group
    ([0, 128, 256, 512], 512, 256, 128),                       # everything even
    ([0, 1000, 1000, 2100], 2100, 1032, 528),
    ([0, 0, 0, 0], 64, 64, 64),                                # no rows at all
    ([7, 7, 63], 64, 8, 2048),
]


@pytest.mark.parametrize("offsets,rows,n,k", ROWS, ids=range(len(ROWS)))
@pytest.mark.parametrize("kind,layout", [("float16", "nk"), ("float16", "kn"), ("bfloat16", "nk"), ("bfloat16", "kn"),
                                         ("fp8", "nk")])
@pytest.mark.parametrize("out", [F32, BF16])
def test_rows(cuda_dev, offsets, rows, n, k, kind, layout, out):
    _check_rows(cuda_dev, kind, layout, offsets, rows, n, k, out, seed=rows + n)


VARIANTS = [{"BW_GROUPED_PAIR": "1"}, {"BW_GROUPED_PAIR": "0", "BW_GROUPED_W": "64"},
            {"BW_GROUPED_PAIR": "0", "BW_GROUPED_W": "128"}, {"BW_GROUPED_PAIR": "0", "BW_GROUPED_W": "256"},
            {"BW_GROUPED_PAIR": "0", "BW_GROUPED_W": "176"}]


@pytest.mark.parametrize("env", VARIANTS, ids=["pair", "w64", "w128", "w256", "w176"])
@pytest.mark.parametrize("case", [1, 3, 4, 6])
def test_every_tile_shape(cuda_dev, monkeypatch, env, case):
    """The kernels and tile widths that the sizes would not choose by themselves, forward and gradients."""
    import torch

    for k, v in env.items():
        monkeypatch.setenv(k, v)
    offsets, rows, n, k = ROWS[case]
    for kind, layout in (("float16", "kn"), ("bfloat16", "nk"), ("fp8", "nk")):
        for out in (F32, BF16):
            _check_rows(cuda_dev, kind, layout, offsets, rows, n, k, out, seed=case)
    g = torch.Generator(device=cuda_dev).manual_seed(case)
    x = torch.randn(rows, k, device=cuda_dev, generator=g).bfloat16()
    y = torch.randn(rows, n, device=cuda_dev, generator=g).bfloat16()
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_dev)
    for out in (F32, BF16):
        _check_wgrad(x, y, offsets, bwgemm.gemm_grouped_wgrad(x, y, off, out_dtype=out), out)
    assert bwgemm.device_status() == 0


@pytest.mark.parametrize("n", [1, 3, 17, 65, 127, 250, 257, 511])
@pytest.mark.parametrize("out", [F32, BF16])
def test_odd_columns(cuda_dev, n, out):
    """Any N for a K-contiguous B: stores element by element at the edge, nothing beside."""
    for kind in KINDS:
        _check_rows(cuda_dev, kind, "nk", [0, 3, 140], 140, n, 80, out, seed=n)


@pytest.mark.parametrize("k", [1, 5, 63, 65, 100])
def test_odd_depth(cuda_dev, k):
    """Any K for an N-contiguous B (A needs its pitch): the slab behind K reads zeros."""
    _check_rows(cuda_dev, "bfloat16", "kn", [0, 3, 140], 140, 72, k, F32, seed=k, pad=-k % 8 + 8)


def test_next_matrix_and_padding_may_be_anything(cuda_dev):
    """NaN and infinities in other groups' rows and matrices and in A's padding do not spread."""
    import torch

    for layout in ("nk", "kn"):
        a, b, _, _, ad, bd = _make(cuda_dev, "bfloat16", layout, 3, 90, 72, 72, pad=56)
        off = torch.tensor([0, 30, 60, 90], dtype=torch.int32, device=cuda_dev)
        want, mag = _product(ad, bd, layout, [0, 30, 60, 90], None, None)
        a[30:60] = float("nan")
        b[1] = float("inf")
        whole = a._base if a._base is not None else a
        whole[:, 72:] = float("nan")
        C = bwgemm.gemm_grouped(a, b, off, b_transposed=layout == "nk", out_dtype=F32)
        keep = [i for i in range(90) if not 30 <= i < 60]
        _close(C[keep], want[keep], mag[keep], _steps("bf16", 72), F32)
        assert bool(C[30:60].isnan().all())


@pytest.mark.parametrize("offsets", [[-5, 10, 4, 500, 20], [40, 30, 20, 10, 0], [2 ** 31 - 1, 0, 5, 6, 7],
                                     [-2 ** 31, -1, 0, 33, 2 ** 31 - 1]])
def test_bad_offsets_stay_inside(cuda_dev, offsets):
    """Offsets that are out of range or fall count as documented; nothing outside is touched."""
    import torch

    _check_rows(cuda_dev, "float16", "kn", offsets, 64, 64, 64, F32)
    x, y = torch.randn(64, 64, device=cuda_dev).half(), torch.randn(64, 72, device=cuda_dev).half()
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_dev)
    D = bwgemm.gemm_grouped_wgrad(x, y, off)
    _check_wgrad(x, y, bounds_of(offsets, 64), D, F32)


@pytest.mark.parametrize("kind", KINDS)
def test_pitches(cuda_dev, kind):
    """A and C inside wider buffers, C at every store width."""
    import torch

    rows, n, k = 150, 264, 144
    for out, dt in ((F32, torch.float32), (BF16, torch.bfloat16)):
        for pad, shift in ((56, 0), (24, 16), (8, 4), (1, 1)):
            whole = torch.full((rows * (n + pad) + 64,), -77.0, dtype=dt, device=cuda_dev)
            C = whole[shift:shift + rows * (n + pad)].view(rows, n + pad)[:, :n]
            _check_rows(cuda_dev, kind, "nk", [1, 20, 149], rows, n, k, out, pad=32, C=C)
            C.fill_(-77.0)
            assert bool((whole == -77.0).all())


def test_exact_integers(cuda_dev):
    """Small integers: every sum is exact, so forward and gradients equal the 64-bit product bit for bit."""
    import torch

    g = torch.Generator(device=cuda_dev).manual_seed(3)
    offsets = [0, 700, 701, 701, 1500, 3000]
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_dev)
    a = torch.randint(-4, 5, (3000, 1024), device=cuda_dev, generator=g).double()
    b = torch.randint(-4, 5, (5, 1024, 768), device=cuda_dev, generator=g).double()
    want, _ = _product(a, b, "kn", offsets, None, None)
    for dt in (torch.float16, torch.bfloat16):
        assert torch.equal(bwgemm.gemm_grouped(a.to(dt), b.to(dt), off, out_dtype=F32).double(), want)
        bt = b.to(dt).transpose(1, 2).contiguous()
        assert torch.equal(bwgemm.gemm_grouped(a.to(dt), bt, off, b_transposed=True, out_dtype=F32).double(), want)
        y = torch.randint(-4, 5, (3000, 768), device=cuda_dev, generator=g).double()
        D = bwgemm.gemm_grouped_wgrad(a.to(dt), y.to(dt), off)
        for e in range(5):
            i, j = offsets[e], offsets[e + 1]
            assert torch.equal(D[e].double(), a[i:j].T @ y[i:j])
    f8 = lambda t: t.to(torch.float8_e4m3fn).view(torch.uint8)  # noqa: E731
    C = bwgemm.gemm_grouped(f8(a), f8(b.transpose(1, 2).contiguous()), off, b_transposed=True, out_dtype=F32)
    assert torch.equal(C.double(), want)


@pytest.mark.parametrize("which", ["rows", "groups", "both"])
def test_scales_of_16_bit_products(cuda_dev, which):
    """Row and group scales are taken with every operand type, each alone too."""
    import torch

    offsets = [0, 40, 40, 300]
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_dev)
    a, b, _, _, ad, bd = _make(cuda_dev, "bfloat16", "kn", 3, 300, 264, 136)
    rs = torch.rand(300, device=cuda_dev) + 0.5 if which != "groups" else None
    gs = torch.rand(3, device=cuda_dev) + 0.5 if which != "rows" else None
    C = bwgemm.gemm_grouped(a, b, off, row_scale=rs, group_scale=gs, out_dtype=F32)
    want, mag = _product(ad, bd, "kn", offsets, rs, gs)
    _close(C, want, mag, _steps("bf16", 136), F32)


def test_dependent_calls_in_a_row(cuda_dev):
    """Each call reads what the one before it wrote, and writes what that one read, without a pause:
    the same bits as with a synchronisation after every call."""
    import torch

    offsets = [0, 130, 131, 400, 700]
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_dev)
    g = torch.Generator(device=cuda_dev).manual_seed(2)
    a0 = torch.randn(700, 512, device=cuda_dev, generator=g).bfloat16()
    b = (torch.randn(4, 512, 512, device=cuda_dev, generator=g) * 512 ** -0.5).bfloat16()
    w = torch.ones(512, device=cuda_dev).bfloat16()

    def chain(pause):
        one, two = a0.clone(), torch.empty_like(a0)
        grads = torch.zeros(4, 512, 512, device=cuda_dev)
        for i in range(20):
            for x, y in ((one, two), (two, one)):
                bwgemm.gemm_grouped(x, b, off, y, b_transposed=bool(i % 2))
                pause()
                bwgemm.gemm_grouped_wgrad(x, y, off, grads)
                pause()
                bwgemm.rmsnorm(y, w, y=y)
                pause()
                off.copy_(torch.roll(off, 0))
        return one, two, grads

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        got = chain(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_many_groups(cuda_dev):
    """1024 groups, most of them empty or of one row."""
    import torch

    g = torch.Generator().manual_seed(1)
    counts = torch.randint(0, 3, (1024,), generator=g)
    offsets = [0] + counts.cumsum(0).tolist()
    _check_rows(cuda_dev, "float16", "nk", offsets, offsets[-1], 72, 64, F32)


def test_k_zero_and_empty(cuda_dev):
    import torch

    off = torch.tensor([1, 3, 5], dtype=torch.int32, device=cuda_dev)
    for layout in (True, False):
        C = torch.full((7, 24), 5.0, device=cuda_dev)
        A = torch.empty(7, 0, dtype=torch.float16, device=cuda_dev)
        B = torch.empty((2, 24, 0) if layout else (2, 0, 24), dtype=torch.float16, device=cuda_dev)
        nan = torch.full((2,), float("nan"), device=cuda_dev)
        bwgemm.gemm_grouped(A, B, off, C, b_transposed=layout, group_scale=nan, out_dtype=F32)
        assert bool((C[1:5] == 0).all()) and bool((C[:1] == 5).all()) and bool((C[5:] == 5).all())
    e = torch.empty(0, 24, dtype=torch.float16, device=cuda_dev)
    assert bwgemm.gemm_grouped(e, torch.ones(2, 24, 24, dtype=torch.float16, device=cuda_dev), off).shape == (0, 24)
    D = torch.full((2, 24, 24), 5.0, device=cuda_dev)
    bwgemm.gemm_grouped_wgrad(e, e, off, D)
    assert bool((D == 0).all())


# ------------------------------------------------------------------ weight gradient
def _check_wgrad(x, y, bnd, D, out):
    xd, yd = x.double(), y.double()
    for e in range(len(bnd) - 1):
        i, j = bnd[e], bnd[e + 1]
        want, mag = xd[i:j].T @ yd[i:j], xd[i:j].abs().T @ yd[i:j].abs()
        _close(D[e], want, mag, _steps("f16", max(1, j - i)), out)
        if i == j:
            assert bool((D[e] == 0).all())


WGRAD = [
    ([0, 1], 1, 8, 8),
    ([0, 16, 16, 31, 64], 64, 64, 72),
    ([0, 5, 5, 69, 197, 198, 400], 400, 264, 520),
    ([3, 130, 131, 131, 390], 400, 1032, 128),
    ([0, 1000, 2049], 2049, 136, 264),
    ([0, 0, 0], 9, 64, 64),
]


@pytest.mark.parametrize("offsets,rows,m,n", WGRAD, ids=range(len(WGRAD)))
@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("out", [F32, BF16])
def test_wgrad(cuda_dev, offsets, rows, m, n, kind, out):
    import torch

    g = torch.Generator(device=cuda_dev).manual_seed(rows)
    x = torch.randn(rows, m, device=cuda_dev, generator=g).to(getattr(torch, kind))
    y = torch.randn(rows, n, device=cuda_dev, generator=g).to(getattr(torch, kind))
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_dev)
    D = torch.full((len(offsets) - 1, m, n), -77.0, device=cuda_dev, dtype=torch.bfloat16 if out == BF16 else torch.float32)
    bwgemm.gemm_grouped_wgrad(x, y, off, D, out_dtype=out)
    torch.cuda.synchronize()
    assert bwgemm.device_status() == 0
    _check_wgrad(x, y, offsets, D, out)


@pytest.mark.parametrize("m,n", [(1, 1), (5, 130), (100, 7), (257, 65)])
def test_wgrad_odd_sizes(cuda_dev, m, n):
    """Any M and N, given operand pitches of 16 bytes."""
    import torch

    x = torch.randn(100, m + 8 + -m % 8, device=cuda_dev).half()[:, :m]
    y = torch.randn(100, n + 8 + -n % 8, device=cuda_dev).half()[:, :n]
    off = torch.tensor([0, 33, 100], dtype=torch.int32, device=cuda_dev)
    _check_wgrad(x, y, [0, 33, 100], bwgemm.gemm_grouped_wgrad(x, y, off), F32)


@pytest.mark.parametrize("cut", [1, 7, 15, 16, 17, 47, 63, 64, 65])
def test_wgrad_rows_behind_a_group_may_be_anything(cuda_dev, cut):
    """The rows behind a group's end (another group's, or nobody's) hold NaN and infinities."""
    import torch

    x = torch.randn(200, 192, device=cuda_dev).bfloat16()
    y = torch.randn(200, 320, device=cuda_dev).bfloat16()
    for bad in (float("nan"), float("inf")):
        x[cut:150] = bad
        y[cut:150] = bad
        off = torch.tensor([0, cut, 150, 200], dtype=torch.int32, device=cuda_dev)
        D = bwgemm.gemm_grouped_wgrad(x, y, off)
        torch.cuda.synchronize()
        assert bwgemm.device_status() == 0
        _check_wgrad(x[:cut], y[:cut], [0, cut], D[:1], F32)
        _check_wgrad(x[150:], y[150:], [0, 50], D[2:], F32)
        assert not bool(D[1].isfinite().any())                    # inf * inf = inf, nan * nan = nan


def test_gradients_against_differences(cuda_dev):
    """dA (the other layout of the same B) and dB against differences of the 64-bit product."""
    import torch

    offsets = [0, 3, 3, 8]
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_dev)
    a, b, _, _, ad, bd = _make(cuda_dev, "bfloat16", "nk", 3, 8, 24, 32, seed=4)
    dc = torch.randn(8, 24, device=cuda_dev).bfloat16()
    da = bwgemm.gemm_grouped(dc, b, off, out_dtype=F32)           # groups x N x K read as contraction x outputs
    db = bwgemm.gemm_grouped_wgrad(dc, a, off)                    # groups x N x K
    loss = lambda x, w: torch.nansum(_product(x, w, "nk", offsets, None, None)[0] * dc.double())  # noqa: E731
    for r, k in ((0, 0), (2, 31), (7, 5)):
        e = torch.zeros_like(ad)
        e[r, k] = 0.5                                             # the product is linear: any step is exact
        num = float(loss(ad + e, bd) - loss(ad - e, bd))
        assert abs(num - float(da[r, k])) <= 1e-5 * (1 + abs(num))
    for g, n, k in ((0, 0, 0), (1, 3, 4), (2, 23, 31)):
        e = torch.zeros_like(bd)
        e[g, n, k] = 0.5
        num = float(loss(ad, bd + e) - loss(ad, bd - e))
        assert abs(num - float(db[g, n, k])) <= 1e-5 * (1 + abs(num))


# ------------------------------------------------------------------ use
def test_graph_replays_with_new_sizes(cuda_dev):
    """One captured graph serves other offsets and data; two graphs on two streams share nothing."""
    import torch

    graphs = []
    for k in range(2):
        a, b, rs, gs, _, _ = _make(cuda_dev, "fp8", "nk", 6, 300, 264, 256, seed=k)
        x, y = torch.randn(300, 136, device=cuda_dev).bfloat16(), torch.randn(300, 72, device=cuda_dev).bfloat16()
        off = torch.tensor([0, 50, 100, 150, 200, 250, 300], dtype=torch.int32, device=cuda_dev)
        C = torch.zeros(300, 264, dtype=torch.bfloat16, device=cuda_dev)
        D = torch.zeros(6, 136, 72, device=cuda_dev)
        s = torch.cuda.Stream(cuda_dev)
        g = torch.cuda.CUDAGraph()
        bwgemm.gemm_grouped(a, b, off, C, b_transposed=True, row_scale=rs, group_scale=gs)
        bwgemm.gemm_grouped_wgrad(x, y, off, D)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            bwgemm.gemm_grouped(a, b, off, C, b_transposed=True, row_scale=rs, group_scale=gs)
            bwgemm.gemm_grouped_wgrad(x, y, off, D)
        graphs.append((g, s, a, b, rs, gs, x, y, off, C, D))
    for new in ([0, 0, 7, 150, 150, 299, 300], [0, 300, 300, 300, 300, 300, 300]):
        for g, s, a, b, rs, gs, x, y, off, C, D in graphs:
            off.copy_(torch.tensor(new, dtype=torch.int32))
            C.zero_(), D.zero_()
        torch.cuda.synchronize()
        for g, s, *_ in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert bwgemm.device_status() == 0
        for g, s, a, b, rs, gs, x, y, off, C, D in graphs:
            f8 = lambda t: t.view(torch.float8_e4m3fn).double()  # noqa: E731
            want, mag = _product(f8(a), f8(b), "nk", new, rs, gs)
            _close(C, want, mag, _steps("fp8", 256), BF16)
            _check_wgrad(x, y, new, D, F32)


def test_capture_with_fork_and_join(cuda_dev):
    """Captured behind a copy, a memset and another stream's kernels: full dependencies are kept."""
    import torch

    a, b, rs, gs, _, _ = _make(cuda_dev, "fp8", "nk", 4, 500, 264, 256)
    A, off = torch.zeros_like(a.contiguous()), torch.zeros(5, dtype=torch.int32, device=cuda_dev)
    true = torch.tensor([0, 100, 100, 330, 500], dtype=torch.int32, device=cuda_dev)
    y = torch.randn(500, 72, device=cuda_dev).bfloat16()
    side = torch.cuda.Stream(cuda_dev)

    def work():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        A.copy_(a)
        with torch.cuda.stream(side):
            off.zero_()
            off.add_(true)
        main.wait_stream(side)
        C = bwgemm.gemm_grouped(A, b, off, b_transposed=True, row_scale=rs, group_scale=gs)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            D = bwgemm.gemm_grouped_wgrad(C, y, off)
        E = C * 2
        main.wait_stream(side)
        return C, D, E

    want = work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for _ in range(4):
        A.zero_(), off.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert bwgemm.device_status() == 0
        assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_repeatable(cuda_dev):
    """The same call twice gives the same bits."""
    import torch

    off = torch.tensor([0, 100, 600, 601, 1500], dtype=torch.int32, device=cuda_dev)
    a, b, rs, gs, _, _ = _make(cuda_dev, "fp8", "nk", 4, 1500, 512, 1024)
    one = bwgemm.gemm_grouped(a, b, off, b_transposed=True, row_scale=rs, group_scale=gs, out_dtype=F32)
    x = torch.randn(1500, 256, device=cuda_dev).half()
    w1 = bwgemm.gemm_grouped_wgrad(x, x, off)
    for _ in range(3):
        assert torch.equal(one, bwgemm.gemm_grouped(a, b, off, b_transposed=True, row_scale=rs, group_scale=gs, out_dtype=F32))
        assert torch.equal(w1, bwgemm.gemm_grouped_wgrad(x, x, off))


def test_large_offsets(cuda_dev):
    """B and C beyond 2^31 elements, rows beyond 2^31 bytes."""
    import torch

    groups, n, k = 5, 16384, 32768                                # 2.7e9 elements of B
    b = torch.zeros(groups, n, k, dtype=torch.uint8, device=cuda_dev)
    b[-1, -8:] = torch.randint(0, 120, (8, k), dtype=torch.uint8, device=cuda_dev)
    a = torch.randint(0, 120, (3, k), dtype=torch.uint8, device=cuda_dev)
    off = torch.tensor([0, 0, 1, 1, 2, 3], dtype=torch.int32, device=cuda_dev)
    pitch = 1_200_000_000
    C = torch.empty(2 * pitch + n, device=cuda_dev, dtype=torch.bfloat16).as_strided((3, n), (pitch, 1))
    bwgemm.gemm_grouped(a, b, off, C, b_transposed=True)
    f8 = lambda t: t.view(torch.float8_e4m3fn).double()  # noqa: E731
    want = f8(a[2:]) @ f8(b[-1, -8:]).T
    _close(C[2:, -8:], want, want.abs(), _steps("fp8", k), BF16)  # codes below 128 are positive
    assert bool((C[:2] == 0).all()) and bool((C[2, :-8] == 0).all())


def test_expert_layer(cuda_dev):
    """The operators in a row: norm of the residual stream to E4M3 with row scales, rows sent to
    their experts, grouped E4M3 product, back; and the BF16 training step of the same layer."""
    import torch

    g = torch.Generator(device=cuda_dev).manual_seed(11)
    T, E, K, N, top = 200, 7, 512, 384, 2
    rnd = lambda *s: torch.randn(*s, device=cuda_dev, generator=g)  # noqa: E731
    x, res, w = rnd(T, K).bfloat16(), rnd(T, K).bfloat16(), (1 + 0.1 * rnd(K)).bfloat16()
    W = rnd(E, N, K) * K ** -0.5
    qw = torch.empty(E, N, K, dtype=torch.uint8, device=cuda_dev)
    sw = torch.empty(E, device=cuda_dev)
    for e in range(E):
        bwgemm.quantize_fp8(W[e], False, bwgemm.SCALE_AMAX, dst=qw[e], scale_out=sw[e:e + 1])
    choice = rnd(T, E).topk(top, dim=1).indices.reshape(-1)
    order = choice.argsort(stable=True)
    off = torch.cat([torch.zeros(1, dtype=torch.int64, device=cuda_dev), choice.bincount(minlength=E).cumsum(0)]).int()
    token = order // top
    # serving
    q, s, h, rstd = bwgemm.rmsnorm_fp8(x, w, residual=res)
    c = bwgemm.gemm_grouped(q[token], qw, off, b_transposed=True, row_scale=s[token], group_scale=sw, out_dtype=F32)
    f8 = lambda t: t.view(torch.float8_e4m3fn).double()  # noqa: E731
    want, mag = _product(f8(q[token]), f8(qw), "nk", off.tolist(), s[token], sw)
    _close(c, want, mag, _steps("fp8", K), F32)
    # the 8-bit product is the unquantised one to E4M3's precision: 2^-4 of each factor, over K random terms
    h64 = (x.double() + res.double()).bfloat16().double()
    y64 = h64 * (h64.square().mean(1, keepdim=True) + 1e-6) ** -0.5 * w.double()
    full, full_mag = _product(y64[token], W.double(), "nk", off.tolist(), None, None)
    assert bool(((c.double() - full).abs() <= (2 * 2.0 ** -4 + 2.0 ** -8) * full_mag).all())
    # training
    wb = W.bfloat16()
    y, h, rstd = bwgemm.rmsnorm(x, w, residual=res)
    yt = y[token]
    c = bwgemm.gemm_grouped(yt, wb, off, b_transposed=True)
    dc = rnd(T * top, N).bfloat16()
    dW = bwgemm.gemm_grouped_wgrad(dc, yt, off)
    dyt = bwgemm.gemm_grouped(dc, wb, off, out_dtype=F32)
    dy = torch.zeros(T, K, device=cuda_dev).index_add_(0, token, dyt).bfloat16()
    dx, dw = bwgemm.rmsnorm_backward(dy, h, w, rstd)
    xr = h.double().requires_grad_()
    wr, Wr = w.double().requires_grad_(), wb.double().requires_grad_()
    yr = xr * (xr.square().mean(1, keepdim=True) + 1e-6) ** -0.5 * wr
    expert = torch.searchsorted(off[1:].long(), torch.arange(T * top, device=cuda_dev), right=True)
    loss = (torch.einsum("rk,rnk->rn", yr[token], Wr[expert]) * dc.double()).sum()
    loss.backward()
    rel = lambda got, ref: float((got.double() - ref).norm() / ref.norm())  # noqa: E731
    # each gradient carries a few BF16 roundings (y, c or dy: 2^-8 each at most)
    assert rel(dW, Wr.grad) <= 2 * 2.0 ** -8
    assert rel(dx, xr.grad) <= 4 * 2.0 ** -8
    assert rel(dw, wr.grad) <= 4 * 2.0 ** -8

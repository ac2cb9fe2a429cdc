"""Grouped products whose waits run out in the middle: every load that was issued lands before the CTA
ends, the status word says where, and the next call is right.

Ring of the forms below: 4 stages of 64 summed elements (single CTA, tiles 256 wide), 3 of 128 (pairs).
"""
import ctypes

import pytest

import bwgemm

FAR = 2 ** 31 - 1
BUDGET = 5_000_000  # ns


def _call(pair, wgrad, A, B, off, C, rows, N, K, stall, stops, landed, budget=BUDGET):
    return bwgemm.lib().bw_selftest_grouped_wait(pair, wgrad, A, B, off, 1, C, rows, N, K, stall, *stops, budget, landed, None)


@pytest.mark.parametrize("bad", [dict(A=None), dict(B=None), dict(C=None), dict(off=None), dict(landed=None), dict(rows=0),
                                 dict(K=0), dict(K=12), dict(stall=-1), dict(stops=(-1, 0)), dict(stops=(0, -1)),
                                 dict(budget=0), dict(budget=1_000_000_001)])
def test_selftest_refuses(bad):
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) & ~255
    a = dict(pair=0, wgrad=0, A=p, B=p, off=p, C=p, rows=4, N=8, K=8, stall=0, stops=(0, 0), landed=p)
    a.update(bad)
    assert _call(**a) == bwgemm.BW_ERR_INVALID


def _run(dev, monkeypatch, pair, wgrad, summed, rows, stall, stops):
    """Value of `landed` for one group and one tile: 256 columns, `rows` output rows, `summed` elements a sum."""
    import torch

    monkeypatch.setenv("BW_GROUPED_W", "256")
    g = torch.Generator(device=dev).manual_seed(summed + rows)
    r, n, k = (summed, rows, 256) if wgrad else (rows, 256, summed)
    a = torch.randn(r, n if wgrad else k, device=dev, generator=g).bfloat16()
    b = torch.randn(*((r, k) if wgrad else (1, n, k)), device=dev, generator=g).bfloat16()
    off = torch.tensor([0, r], dtype=torch.int32, device=dev)
    c = torch.zeros((1, n, k) if wgrad else (r, n), dtype=torch.bfloat16, device=dev)
    landed = torch.zeros(1, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    rc = _call(pair, wgrad, a.data_ptr(), b.data_ptr(), off.data_ptr(), c.data_ptr(), r, n, k, stall, stops, landed.data_ptr())
    assert rc == bwgemm.BW_ERR_TIMEOUT, bwgemm.lib().bw_last_error_string()
    assert bwgemm.device_status() == 0
    # the same operands again, by the call that a user makes: small integers, so every sum is exact
    a, b = a.clamp(-3, 3).round(), b.clamp(-3, 3).round()
    monkeypatch.setenv("BW_GROUPED_PAIR", str(pair))
    if wgrad:
        got, want = bwgemm.gemm_grouped_wgrad(a, b, off)[0], a.double().T @ b.double()
    else:
        got, want = bwgemm.gemm_grouped(a, b, off, b_transposed=True, out_dtype=bwgemm.OUT_F32), a.double() @ b[0].double().T
    assert torch.equal(got.double(), want) and bwgemm.device_status() == 0
    return int(landed)


# slabs of the tile, slab that the MMA thread gives up at, slab that the producer gives up at, stages filled
SINGLE = [(1, 0, FAR, 1), (2, 0, FAR, 2), (4, 0, FAR, 4), (12, 0, FAR, 4), (12, 5, FAR, 4), (12, 11, FAR, 4), (12, FAR, 3, 3),
          (12, FAR, 6, 4), (12, FAR, 0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("slabs,stall,stop,stages", SINGLE)
@pytest.mark.parametrize("wgrad", [0, 1])
@pytest.mark.parametrize("cut", [0, 3])
def test_single(cuda_dev, monkeypatch, slabs, stall, stop, stages, wgrad, cut):
    summed = 64 * slabs - (8 * cut if not wgrad else cut)  # wgrad: the last slab ends inside a k-step of 16
    for rows in (24, 96):
        assert _run(cuda_dev, monkeypatch, 0, wgrad, summed, rows, stall, (stop, 0)) == stages


# ..., slabs that the leader's and the peer's producer give up at
PAIR = [(1, 0, FAR, FAR), (2, 0, FAR, FAR), (3, 0, FAR, FAR), (12, 0, FAR, FAR), (12, 5, FAR, FAR), (12, 11, FAR, FAR),
        (12, FAR, 4, FAR), (12, FAR, FAR, 4), (12, FAR, 1, FAR), (12, FAR, FAR, 1), (12, FAR, 0, FAR), (12, FAR, FAR, 0),
        (12, FAR, 0, 0), (12, FAR, 5, 6), (12, FAR, 6, 5), (3, FAR, 2, FAR), (3, FAR, FAR, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("slabs,stall,leader,peer", PAIR)
@pytest.mark.parametrize("wgrad", [0, 1])
def test_pair(cuda_dev, monkeypatch, slabs, stall, leader, peer, wgrad):
    done = min(stall, leader, peer, slabs)  # slabs that were multiplied
    issued = [min(slabs, done + 3, stop) for stop in (leader, peer)]
    stages = 256 * min(3, max(issued))
    for rows in (48, 136, 256):
        for cut in (0, 3):
            summed = 128 * slabs - (8 * cut if not wgrad else cut)
            ends = sum(n == slabs for n in issued) if wgrad and cut else 0
            got = _run(cuda_dev, monkeypatch, 1, wgrad, summed, rows, stall, (leader, peer))
            assert got == stages + ends, (rows, cut, got, stages, ends)

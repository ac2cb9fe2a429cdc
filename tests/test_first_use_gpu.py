"""The first calls of a process: captured into a graph before any eager one, and from several threads at once. Each in a
process of its own (the library keeps what it learns of its kernels)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

COMMON = """
import sys, threading
sys.path.insert(0, {pkg!r})
import torch
import bwgemm
bwgemm.init(0)
dev = torch.device("cuda:0")
g = torch.Generator(device=dev).manual_seed(1)
rnd = lambda *s: torch.randn(*s, device=dev, generator=g).bfloat16()
few, many, long, odd = rnd(37, 512), rnd(2500, 1600), rnd(3, 20000), rnd(1300, 1111)
offs = torch.tensor([0, 10, 10, 37], dtype=torch.int32, device=dev)
offm = torch.tensor([0, 1000, 1001, 2500], dtype=torch.int32, device=dev)
b = rnd(3, 512, 256)
bm = rnd(3, 1600, 512)
w = {{x.shape[1]: rnd(x.shape[1]) for x in (few, many, long, odd)}}

def work():
    out = []
    for x in (few, many, long, odd):
        y, h, rstd = bwgemm.rmsnorm(x, w[x.shape[1]])
        q, s, _, _ = bwgemm.rmsnorm_fp8(x, w[x.shape[1]], residual=x)
        out += [y, rstd, q, s, *bwgemm.rmsnorm_backward(y, h, w[x.shape[1]], rstd)]
    for x, o, m in ((few, offs, b), (many, offm, bm)):
        c = bwgemm.gemm_grouped(x, m, o)
        out += [c, bwgemm.gemm_grouped_wgrad(x, c, o), bwgemm.gemm_grouped(c, m, o, b_transposed=True)]
    return out
"""

CAPTURED = """
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = work()
graph.replay()
torch.cuda.synchronize()
want = work()
assert bwgemm.device_status() == 0
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""

THREADS = """
torch.cuda.synchronize()
streams = [torch.cuda.Stream() for _ in range(4)]
got, errors = [None] * 4, []
def one(i):
    try:
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                got[i] = work()
    except Exception as e:
        errors.append(e)
ts = [threading.Thread(target=one, args=(i,)) for i in range(4)]
[t.start() for t in ts]
[t.join() for t in ts]
torch.cuda.synchronize()
assert not errors, errors
want = work()
assert bwgemm.device_status() == 0
assert all(torch.equal(a, b) for mine in got for a, b in zip(mine, want))
print("same")
"""


@pytest.mark.parametrize("how", ["captured", "threads"])
def test_first_use(cuda_dev, how):
    import bwgemm

    code = COMMON.format(pkg=os.path.dirname(os.path.abspath(bwgemm.__file__))) + {"captured": CAPTURED, "threads": THREADS}[how]
    r = subprocess.run([sys.executable, "-c", code], cwd=HERE, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stdout[-500:] + r.stderr[-1500:]

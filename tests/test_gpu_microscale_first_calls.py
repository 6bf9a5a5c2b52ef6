"""The first calls of a process: in any order, and from many threads at once, the results are those of any other call."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = r"""
import hashlib, sys, threading
import torch
from trellis_b200 import microscale as ms
order, threads = sys.argv[1], int(sys.argv[2])
g = torch.Generator(device="cuda").manual_seed(0)
calls = {}
for fmt in ("mxfp4", "nvfp4"):
    w = ms.quantize(torch.randn(1300, 2304, generator=g, device="cuda"), fmt)
    for m in (1, 6, 30, 100, 300):
        x = torch.randn(m, 2304, generator=g, device="cuda")
        q = ms.quantize(x, fmt)
        calls[fmt, m, "matmul"] = lambda q=q, w=w: ms.matmul(q, w)
        for t in (torch.float32, torch.float16, torch.bfloat16):
            calls[fmt, m, t] = lambda x=x.to(t), w=w: ms.linear(x, w)
names = list(calls)
if order == "back":
    names.reverse()
out, failed = {}, []
start = threading.Barrier(threads)
def run(mine):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for n in mine:
                out[n] = calls[n]()
            torch.cuda.current_stream().synchronize()
    except BaseException as e:
        failed.append(repr(e))
torch.cuda.synchronize()
ts = [threading.Thread(target=run, args=(names[i::threads],)) for i in range(threads)]
[t.start() for t in ts]
[t.join() for t in ts]
assert not failed, failed
h = hashlib.sha256()
for n in calls:
    h.update(out[n].cpu().contiguous().view(torch.uint8).numpy().tobytes())
print(h.hexdigest())
"""


def test_results_do_not_depend_on_which_call_is_first():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=os.path.join(root, "trellis-everywhere_b200"))
    got = [subprocess.run([sys.executable, "-c", CHILD, order, threads], env=env, capture_output=True, text=True, timeout=120)
           for order, threads in (("forth", "1"), ("back", "1"), ("forth", "8"), ("back", "5"))]
    for r in got:
        assert r.returncode == 0, r.stderr[-2000:]
    assert len({r.stdout for r in got}) == 1


CAPTURED = r"""
import torch
from trellis_b200 import microscale as ms
k = 2304
gen = torch.Generator().manual_seed(0)
for fmt in ("mxfp4", "nvfp4"):
    codes, scales = torch.randint(0, 256, (1300, k // 2), generator=gen), torch.randint(50, 60, (1300, k // ms.BLOCKS[fmt]), generator=gen)
    w = ms.from_blocks(codes.to(torch.uint8).cuda(), scales.to(torch.uint8).cuda(), None if fmt == "mxfp4" else 1.0, k, fmt)
    for m in (1, 30, 300):
        for t in (torch.bfloat16, torch.float16, torch.float32):
            x = torch.randn(m, k, generator=gen).to(t).cuda()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = ms.linear(x, w), ms.matmul(ms.quantize(x, fmt), w, t), ms.dequantize(w, t)
            graph.replay()
            torch.cuda.synchronize()
            want = ms.linear(x, w), ms.matmul(ms.quantize(x, fmt), w, t), ms.dequantize(w, t)
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (fmt, m, t)
print("ok")
"""


def test_first_calls_may_be_captured():
    """Nothing in a process has been called before: what a call sets up for its kernel is set up while a stream is captured."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURED], env=dict(os.environ, PYTHONPATH=os.path.join(root, "trellis-everywhere_b200")), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]

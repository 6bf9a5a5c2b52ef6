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

"""The products' bounded waits: loads that never come end in NaN, from the first missing one on, and in nothing else.

Every CTA stops loading after a few pieces of 256 columns.  A wait for the others runs out (about a quarter of a second) and the kernel ends by
itself.  A result is then NaN or what it is in an ordinary call, which these whole numbers make exact; never the sums of an earlier tile.
"""
import time

import pytest
import torch

from ms_cases import whole_matrix, whole_tokens

pytestmark = pytest.mark.gpu
CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check(call, want, done):
    """``call(loads limit or None, y)``; the first ``done`` x ``done`` results are of a tile that gets all of its loads."""
    y = torch.full_like(want, 5.0)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    assert call(True, y) == 0
    torch.cuda.synchronize()
    assert time.perf_counter() - t0 < 1.5
    lost = torch.isnan(y)
    assert torch.equal(torch.where(lost, want, y), want), "neither NaN nor the result"
    assert lost[-1, -1] and (lost.all() if not done else not lost[:done, :done].any())
    assert call(False, y) == 0
    assert torch.equal(y, want)


# Two or more tiles a CTA: the first turn is whole, the second misses its last piece, and nothing comes after it.  Then columns shared by clusters.
@pytest.mark.parametrize("fmt,dtype,m,n,k,loads,done", (
    ("nvfp4", torch.bfloat16, 3, 151552, 512, 3, 3), ("mxfp4", torch.float32, 2, 151552, 512, 3, 2), ("mxfp4", torch.float16, 8, 151552, 1024, 6, 8),
    ("nvfp4", torch.bfloat16, 1, 40900, 1100, 6, 1), ("nvfp4", torch.bfloat16, 16, 113664, 1024, 6, 16), ("mxfp4", torch.float16, 12, 113664, 1024, 5, 12),
    ("nvfp4", torch.bfloat16, 700, 19000, 1024, 5, 128), ("mxfp4", torch.float16, 700, 19000, 1024, 7, 128), ("nvfp4", torch.float32, 40, 40000, 1024, 6, 21),
    ("nvfp4", torch.bfloat16, 1, 300, 4096, 1, 0), ("mxfp4", torch.float32, 5, 300, 4096, 0, 0), ("mxfp4", torch.bfloat16, 60, 300, 4096, 1, 0),
    ("nvfp4", torch.float16, 100, 300, 4096, 1, 0), ("mxfp4", torch.float32, 30, 200, 4096, 1, 0)))
def test_linear_whose_loads_do_not_come(fmt, dtype, m, n, k, loads, done):
    from trellis_b200 import _lib, microscale as ms
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    w, wv = whole_matrix(n, k, fmt, n + k)
    x = whole_tokens(m, k, dtype, m)
    want = (x.double() @ wv.t()).to(dtype)
    f = ms.FORMATS[fmt]
    ws = torch.empty(lib.tcq_ms_linear_workspace_bytes(m, n, k, CODE[dtype], f), dtype=torch.uint8, device="cuda")
    args = (x.data_ptr(), CODE[dtype], m, k, w.codes.data_ptr(), w.scales.data_ptr(), _ptr(w.row_scale), n, k, f)

    def call(short, y):
        rest = (y.data_ptr(), n, ws.data_ptr(), ws.numel(), stream)
        return lib.tcq_selftest_ms_linear_waits(loads, *args, *rest) if short else lib.tcq_ms_linear(*args, *rest)

    _check(call, want, done)


@pytest.mark.parametrize("fmt,dtype,m,n,k,loads,done", (
    ("nvfp4", torch.bfloat16, 5, 75776, 512, 3, 5), ("mxfp4", torch.float32, 40, 75776, 512, 3, 40), ("mxfp4", torch.float16, 100, 75776, 600, 5, 100),
    ("nvfp4", torch.float32, 300, 9700, 512, 3, 128), ("mxfp4", torch.bfloat16, 2100, 12200, 512, 3, 128), ("nvfp4", torch.float16, 2100, 12200, 1024, 5, 128),
    ("nvfp4", torch.bfloat16, 1, 1024, 4096, 1, 0), ("mxfp4", torch.float32, 20, 500, 4096, 1, 0), ("nvfp4", torch.float16, 100, 400, 8200, 0, 0)))
def test_matmul_whose_loads_do_not_come(fmt, dtype, m, n, k, loads, done):
    from trellis_b200 import _lib, microscale as ms
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    w, wv = whole_matrix(n, k, fmt, n + k)
    x, xv = whole_matrix(m, k, fmt, m)
    want = (xv @ wv.t()).to(dtype)
    args = (x.codes.data_ptr(), x.scales.data_ptr(), _ptr(x.row_scale), m, w.codes.data_ptr(), w.scales.data_ptr(), _ptr(w.row_scale), n, k, ms.FORMATS[fmt])

    def call(short, y):
        rest = (y.data_ptr(), CODE[dtype], n, stream)
        return lib.tcq_selftest_ms_matmul_waits(loads, *args, *rest) if short else lib.tcq_ms_matmul(*args, *rest)

    _check(call, want, done)

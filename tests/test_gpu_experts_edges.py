"""Calls of the operators around experts at which something could go wrong that sizes between do not show."""
import ms_cases
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k", [(1, 64), (2, 64), (1, 700), (2, 512)])
def test_many_items_of_the_same_rows(m, k, fmt):
    """One or two rows through a matrix of more than three times 128 rows for every SM: a CTA's items share what x was cut into.  Whole numbers, bit for bit, call after call."""
    from trellis_b200 import microscale as ms
    n = 128 * 148 * 4 - 77
    w, wv = ms_cases.whole_matrix(n, k, fmt, 1)
    x = ms_cases.whole_tokens(m, k, torch.bfloat16, 2)
    want = (x.double() @ wv.t()).to(torch.bfloat16)
    b = torch.zeros(n, device=DEV)
    got = [ms.linear(x, w, bias=b) for _ in range(20)]
    assert all(torch.equal(y, want) for y in got)

"""dW of no rows is zeros, for rows of W up to the longest (whose last columns are
past 2^32 bytes) and many short ones; what lies beside them stays."""
import pytest
import torch

import bwpp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,rows,cols,pad", [
    (torch.bfloat16, 1, 8, 0), (torch.bfloat16, 3, 1001, 5), (torch.float32, 5000, 7, 2), (torch.float32, 2, 1 << 20, 1),
    (torch.bfloat16, 1, 2 ** 31 - 1, 0), (torch.float32, 1, 2 ** 31 - 1, 0), (torch.bfloat16, 2, 2 ** 31 - 100, 3)])
def test_zeros(be, dtype, rows, cols, pad):
    buf = torch.full((rows * (cols + pad) + 8,), 7.0, device="cuda", dtype=dtype)
    w = torch.zeros(8, device="cuda")
    t = torch.zeros(1, device="cuda", dtype=torch.int32)
    p = bwpp.LinearXentParams(rows=0, vocab=rows, dim=cols, trans_w=1, lddw=cols + pad, dtype=int(dtype == torch.bfloat16))
    be.dispatch_linear_xent_grad(w, w, t, w, None, None, buf, p)
    dw = buf[:rows * (cols + pad)].reshape(rows, cols + pad)
    for i in range(0, cols, 1 << 28):
        assert not bool(dw[:, i:min(i + (1 << 28), cols)].any())
    assert bool((dw[:, cols:] == 7.0).all()) and bool((buf[rows * (cols + pad):] == 7.0).all())

"""dx between the rows of W, and dW between those of x, as column blocks of one
buffer (no element of one is another's): the bits of a call into other buffers."""
import pytest
import torch

import bwpp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,T,V", [(torch.float32, 40, 700), (torch.float32, 100, 33000), (torch.float32, 1200, 4000),
                                       (torch.bfloat16, 40, 700), (torch.bfloat16, 600, 4000), (torch.bfloat16, 3, 5)])
def test_column_blocks(be, dtype, T, V):
    D = 256
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    w0, x0 = rand(V, D) * 0.1, rand(T, D)
    t = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
    t[1] = -1
    one = torch.full((max(T, V), 2 * D), 7.0, device="cuda", dtype=dtype)  # [W | dx]
    two = torch.full((max(T, V), 2 * D), 7.0, device="cuda", dtype=dtype)  # [dW | x]
    w, dx, dw, x = one[:V, :D], one[:T, D:], two[:V, :D], two[:T, D:]
    w.copy_(w0)
    x.copy_(x0)
    lse, lse0 = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    dx0, dw0 = torch.empty(T, 2 * D, device="cuda", dtype=dtype)[:, :D], torch.empty(V, 2 * D, device="cuda", dtype=dtype)[:, :D]
    ws, xs = torch.empty(V, 2 * D, device="cuda", dtype=dtype)[:, :D], torch.empty(T, 2 * D, device="cuda", dtype=dtype)[:, :D]
    ws.copy_(w0)
    xs.copy_(x0)
    p = bwpp.LinearXentParams(rows=T, vocab=V, dim=D, ldx=2 * D, ldw=2 * D, lddx=2 * D, lddw=2 * D, trans_w=1,
                              dtype=int(dtype == torch.bfloat16))
    be.dispatch_linear_xent(xs, ws, t, None, lse0, None, p)
    be.dispatch_linear_xent_grad(xs, ws, t, lse0, None, dx0, dw0, p)
    be.dispatch_linear_xent(x, w, t, None, lse, None, p)
    be.dispatch_linear_xent_grad(x, w, t, lse, None, dx, dw, p)
    assert torch.equal(lse, lse0) and torch.equal(dx, dx0) and torch.equal(dw, dw0)
    assert torch.equal(w, w0) and torch.equal(x, x0)
    assert bool((one[T:, D:] == 7.0).all()) and bool((two[V:, :D] == 7.0).all())

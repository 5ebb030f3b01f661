"""Empty tensors (whose address is NULL) through the operators around a block: no
error, weight gradients and sums 0, nothing else written."""
import pytest
import torch

import bwpp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_empty_tensors(be, dtype):
    D, V, dt = 64, 100, int(dtype == torch.bfloat16)
    e = lambda *s, t=dtype: torch.empty(*s, device="cuda", dtype=t)
    x, i = e(0, D), e(0, t=torch.int32)
    assert x.data_ptr() == 0
    rp = bwpp.RotaryParams(tokens=0, q_heads=2, k_heads=1, dim=32, dtype=dt)
    be.dispatch_rotary(x, x, i, x, x, rp)
    be.dispatch_rotary_grad(x, x, None, x, x, rp)
    w = lambda: torch.full((D,), 7.0, device="cuda", dtype=dtype)
    for gate_rows in (0, 4):
        gate, dgate = e(0 if gate_rows else 1, D), torch.full((1, D), 7.0, device="cuda", dtype=dtype)
        np_ = bwpp.ResidualNormParams(rows=0, cols=D, eps=1e-6, post_norm=1, gate_rows=gate_rows, dtype=dt)
        be.dispatch_residual_norm(x, x, w(), gate, w(), x, x, np_)
        dpost, dpre = w(), w()
        be.dispatch_residual_norm_grad(x, x, w(), gate, w(), x, x, x, x, dpost, dgate, dpre, np_)
        assert not bool(dpost.any()) and not bool(dpre.any())
        assert bool((dgate == (7.0 if gate_rows else 0.0)).all())  # (no gate row for no rows)
    xp = bwpp.LinearXentParams(rows=0, vocab=V, dim=D, trans_w=1, dtype=dt)
    wv, dw, f = e(V, D), torch.full((V, D), 7.0, device="cuda", dtype=dtype), e(0, t=torch.float32)
    sums = torch.full((2,), 7.0, device="cuda")
    be.dispatch_linear_xent(x, wv, i, f, f, sums, xp)
    be.dispatch_linear_xent(x, wv, i, f, f, None, xp)
    be.dispatch_linear_xent_grad(x, wv, i, f, f, x, dw, xp)
    be.dispatch_linear_xent_grad(x, wv, i, f, None, x, None, xp)
    assert not bool(sums.any()) and not bool(dw.any())

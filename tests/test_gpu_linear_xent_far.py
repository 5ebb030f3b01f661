"""Hidden states and weights of more than 2^32 elements: rows at both ends and in
the middle against 64 bits.  In norm, bf16 dx and dW are off by at most half a step
of their own and, relative to the sums of magnitudes, half a step of dz, which
adds with random signs: two half steps together; fp32 ones by (D + 2) 2^-24 of
each logit's terms and the sums' own roundings.
A wrong row or column is off by its whole size."""
import pytest
import torch

import bwpp

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype,wide,T,D,V", [(BF16, "vd", 64, 4096, 1200000), (BF16, "dv", 300, 4096, 1100000),
                                              (BF16, "vd", 1200000, 4096, 64), (F32, "dv", 16, 4096, 1100001),
                                              (F32, "vd", 1100000, 4096, 40)])
def test_past_32_bits(be, dtype, wide, T, D, V):
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty((V, D) if wide == "vd" else (D, V), device="cuda", dtype=dtype)
    for i in range(0, w.shape[0], 1 << 16):
        w[i:i + (1 << 16)].normal_(0, 1.5 / D ** 0.5, generator=g)
    x = torch.empty(T, D, device="cuda", dtype=dtype).normal_(generator=g)
    t = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
    t[0], t[-1] = 0, V - 1
    lse, dx, dw = torch.empty(T, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    p = bwpp.LinearXentParams(rows=T, vocab=V, dim=D, trans_w=int(wide == "vd"), dtype=int(dtype == BF16))
    be.dispatch_linear_xent(x, w, t, None, lse, None, p)
    be.dispatch_linear_xent_grad(x, w, t, lse, None, dx, dw, p)
    part = lambda lo, hi: (w[lo:hi] if wide == "vd" else w[:, lo:hi].t()).double().contiguous()
    ends = lambda n: torch.tensor([0, 1, n // 2, n - 2, n - 1], device="cuda")
    rows, cols = ends(T), ends(V)
    total, want = torch.zeros(5, device="cuda", dtype=torch.float64), torch.zeros(5, D, device="cuda", dtype=torch.float64)
    for i in range(0, V, 1 << 15):
        wc = part(i, i + (1 << 15))
        q = torch.exp(x[rows].double() @ wc.t().contiguous() - lse[rows].double()[:, None])
        total += q.sum(dim=1)
        at = t[rows].long() - i
        here = (at >= 0) & (at < wc.shape[0])
        q[here.nonzero()[:, 0], at[here]] -= 1.0
        want += q @ wc
    u = 2.0 ** -24
    logit = (D + 2) * u * 1.5 * D ** 0.5  # sum of |x w|: D terms of 2 / pi 1.5 / sqrt(D) on average
    assert float(total.log().abs().max()) <= logit + (V / 64 + 48) * u + u * float(lse.abs().max())
    step = 2 * 2.0 ** -8 if dtype == BF16 else 2 * logit + (V / 64 + 64) * u
    assert float((dx[rows].double() - want).norm() / want.norm()) <= step
    wc = torch.cat([part(int(c), int(c) + 1) for c in cols])
    want = torch.zeros(5, D, device="cuda", dtype=torch.float64)
    for i in range(0, T, 1 << 16):
        xc = x[i:i + (1 << 16)].double()
        q = torch.exp(xc @ wc.t().contiguous() - lse[i:i + (1 << 16)].double()[:, None])
        q -= (t[i:i + (1 << 16), None] == cols[None, :]).double()
        want += q.t().contiguous() @ xc
    got = torch.cat([(dw[int(c):int(c) + 1] if wide == "vd" else dw[:, int(c):int(c) + 1].t()).double() for c in cols])
    assert float((got - want).norm() / want.norm()) <= step

"""dW of few tiles (from many tokens K in ranges, summed in planes): the targets'
dz counts with what its rounding to bf16 left, as in dW of many tiles.

A log-sum-exp 7 above the logits' leaves p small, so that a half step of the
targets' p - 1 alone would pass the elements' bound: each other dz is off by
rel, its exp's error, and a half step; a target's by rel of p, and by two half
steps of p - 1 one after the other (its remainder is rounded to bf16) and fp32's
own; sums add (terms + planes) 2^-24 of the terms' magnitudes, the result half a
step of itself."""
import pytest
import torch

from lm64 import HALF_STEP, strided, untouched
from test_gpu_linear_xent import BF16, U, _case, _logit_error, _params, _vd

pytestmark = pytest.mark.gpu
H = HALF_STEP[BF16]


@pytest.mark.parametrize("wide,T,D,V,targets,pads", [
    ("vd", 2, 8, 1000, "any", (0, 0)), ("vd", 17, 320, 768, "any", (0, 0)), ("dv", 64, 1000, 1024, "any", (1, 1)),
    ("dv", 256, 512, 512, "few", (0, 0)), ("vd", 257, 8, 9, "any", (0, 0)), ("dv", 257, 9, 8, "any", (0, 0)),
    ("vd", 300, 72, 2001, "any", (3, 1)), ("dv", 300, 72, 2000, "any", (3, 1)),
    ("vd", 1505, 1024, 3144, "any", (0, 0)), ("dv", 1505, 1024, 3144, "any", (0, 5)),
    ("vd", 4500, 130, 515, "one", (0, 0)), ("dv", 4500, 130, 515, "one", (0, 0)), ("vd", 9000, 512, 16400, "any", (0, 0)),
    ("dv", 9000, 520, 16400, "few", (0, 0)), ("vd", 8191, 264, 300, "few", (8, 8))])
def test_targets_keep_their_bits(be, wide, T, D, V, targets, pads):
    g = torch.Generator(device="cuda").manual_seed(77)
    x, w, t = _case(T, D, V, BF16, wide, 21, lean=0.0)
    if targets == "one":  # every token's
        t[:] = V - 1
    if targets == "few":
        t %= 7
    t[::11] = -1
    wv, live = _vd(w, wide), t >= 0
    z = x.double() @ wv.double().t().contiguous()
    lse = (torch.logsumexp(z, dim=1) + 7.0).float()
    up = torch.rand(T, device="cuda", generator=g) + 0.5
    p = torch.exp(z - lse.double()[:, None]) * torch.where(live, up.double(), 0.0)[:, None]
    rel = (_logit_error(x, wv, 1.0) + 20 * U)[:, None]
    rows = torch.arange(T, device="cuda")[live]
    cols = t[live].long()
    dz, err = p.clone(), p * (rel + H)
    dz[rows, cols] -= up.double()[live]
    err[rows, cols] = p[rows, cols] * rel[live, 0] + dz[rows, cols].abs() * (H ** 2 + 4 * U)
    x64 = torch.where(live[:, None], x.double(), 0.0)
    want = dz.t().contiguous() @ x64
    tol = err.t().contiguous() @ x64.abs() + (T + 40) * U * (dz.t().contiguous().abs() @ x64.abs()) + H * want.abs()
    for only in (False, True):
        dx = None if only else torch.empty_like(x)
        dw, buf = strided(tuple(w.shape), (w.shape[1] + pads[1], 1), BF16)
        be.dispatch_linear_xent_grad(x, w, t, lse, up, dx, dw, _params(T, D, V, BF16, wide, x, w, lddw=dw.stride(0)))
        recent = [be.recent_kernel(i) for i in range(3)]
        assert any(k.startswith(("bwpp_xent_rowsums_r", "bwpp_xent_rows_r")) for k in recent), recent
        assert bool(((_vd(dw, wide).double() - want).abs() <= tol).all()), only
        assert untouched(dw, buf)


@pytest.mark.parametrize("wide,T,D,V", [("vd", 3000, 256, 1500), ("dv", 300, 130, 516)])
def test_recorded(be, wide, T, D, V):
    """Its planes lie in the handle's workspace, so a recorded graph takes the same
    kernels and gives the same bits; a smaller call runs between the replays."""
    import bwpp
    x, w, t = _case(T, D, V, BF16, wide, 23)
    x2, w2, t2 = _case(40, 64, 300, BF16, "vd", 24)
    b, side = bwpp.HipBackend(0), torch.cuda.Stream()
    torch.cuda.synchronize()
    b.set_stream(side)
    lse, lse2 = torch.empty(T, device="cuda"), torch.empty(40, device="cuda")
    out, small = (torch.empty_like(x), torch.empty_like(w)), (torch.empty_like(x2), torch.empty_like(w2))
    torch.cuda.synchronize()

    def call(a, c, d, l, o, p):
        b.dispatch_linear_xent(a, c, d, None, l, None, p)
        b.dispatch_linear_xent_grad(a, c, d, l, None, *o, p)

    p, p2 = _params(T, D, V, BF16, wide, x, w), _params(40, 64, 300, BF16, "vd", x2, w2)
    call(x, w, t, lse, out, p)
    assert any(b.recent_kernel(i).startswith(("bwpp_xent_rowsums_r", "bwpp_xent_rows_r")) for i in range(3))
    side.synchronize()
    want = [v.clone() for v in out]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(x, w, t, lse, out, p)
    for i in range(4):
        for v in (*out, lse):
            v.fill_(3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        call(x2, w2, t2, lse2, small, p2)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i
    b.close()

"""Cross entropy against a vocabulary, and its gradients, against 64 bits.

Bounds, with u = 2^-24.  A logit is a sum of D products in fp32: off by at most
(D + 2) u S, S the row's largest sum of |x w| (times the scale).  exp and the
sums add a relative 16 u to each term (and (V / 64 + 32) u, summed in runs of 16
a thread and then 64 to a tile, tile after tile), so lse is off by at most
(D + 2) u S + (V / 64 + 48) u + u |lse|, and the loss by that and the target's
(D + 2) u S.  dz is then off by a relative 2 (D + 2) u S + (V / 64 + 64) u, in
bf16 by half a step more, and dx and dW by that of the sum of magnitudes of
their terms, (terms) u for their sums, and their own rounding.  The second check
is on the norm of the error, which random signs keep far below that: the
roundings r of dz, |r| <= half a step of |dz|, reach dx as r W, and |r W| <= |r|
s(W) in norm, s its largest singular value (dW: x's); the result's rounding adds
half a step of its norm, and what fp32 adds is bounded as above.  (That is not
relative to the result: dz of a target is p - 1, which keeps p's absolute error;
with p = 1 - 2^-10 a relative 2^-23 of p is 2^-13 of p - 1.)"""
import pytest
import torch

import bwpp
from lm64 import HALF_STEP, strided, untouched, xent64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(1234)


F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def _case(T, D, V, dtype, wide, seed, pads=(0, 0), lean=4.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, D, device="cuda", generator=g) * 1.5 / D ** 0.5
    t = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
    x = torch.randn(T, D, device="cuda", generator=g) + lean * torch.rand(T, 1, device="cuda", generator=g) * w[t.long()]
    w = w.to(dtype) if wide == "vd" else w.t().contiguous().to(dtype)
    xs = strided((T, D), (D + pads[0], 1), dtype, x)[0]
    ws = strided(tuple(w.shape), (w.shape[1] + pads[1], 1), dtype, w)[0]
    return xs, ws, t


def _params(T, D, V, dtype, wide, x, w, scale=1.0, **kw):
    return bwpp.LinearXentParams(rows=T, vocab=V, dim=D, ldx=x.stride(0) if T > 1 else D, ldw=w.stride(0),
                                 trans_w=int(wide == "vd"), dtype=int(dtype == BF16), scale=scale, **kw)


def _vd(w, wide):
    return w if wide == "vd" else w.t()


def _logit_error(x, w_vd, scale):
    size = (x.double().abs() @ w_vd.double().abs().t().contiguous()).amax(dim=1) * abs(scale)
    return (x.shape[1] + 2) * U * size


def _forward(be, x, w, t, dtype, wide, scale=1.0):
    T, D = x.shape
    V = w.shape[0] if wide == "vd" else w.shape[1]
    want, want_lse = xent64(x, _vd(w, wide), t, scale)
    loss, lse, sums = (torch.full((n,), 7.0, device="cuda") for n in (T, T, 2))
    be.dispatch_linear_xent(x, w, t, loss, lse, sums, _params(T, D, V, dtype, wide, x, w, scale))
    e = _logit_error(x, _vd(w, wide), scale)
    tol = e + (V / 64 + 48) * U + U * want_lse.abs()
    assert bool(((lse.double() - want_lse).abs() <= tol).all())
    live = (t >= 0) & (t < V)
    assert bool(((loss.double() - want).abs() <= tol + e).all())
    assert bool((loss[~live] == 0).all())
    assert float(sums[1]) == float(live.sum())
    total = loss.double().sum()
    assert abs(float(sums[0]) - float(total)) <= 2 * U * float(loss.double().abs().sum())
    return loss, lse, want_lse


def _largest_stretch(a):
    a = a.double()
    g = a.t().contiguous() @ a if a.shape[0] > a.shape[1] else a @ a.t().contiguous()
    return float(torch.linalg.eigvalsh(g.cpu()).amax().clamp(min=0.0).sqrt()) * (1 + 1e-9)


def _gradient(be, x, w, t, lse, dloss, dtype, wide, scale=1.0, pads=(0, 0), scalar=False, only=None):
    T, D = x.shape
    V = w.shape[0] if wide == "vd" else w.shape[1]
    rows = dloss.expand(T) if dloss is not None else torch.ones(T, device="cuda")
    wv = _vd(w, wide)
    live = (t >= 0) & (t < V)
    xz = torch.where(live[:, None], x.double(), 0.0)
    _, _, dx64, dw64 = xent64(x, wv, t, scale, rows)
    # magnitudes of the terms
    z = scale * (x.double() @ wv.double().t().contiguous())
    p = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
    p[torch.arange(T, device="cuda")[live], t[live].long()] += 1.0
    p = torch.where(live[:, None], p * rows.double().abs()[:, None], 0.0) * abs(scale)
    rel = (2 * _logit_error(x, wv, scale) + (V / 64 + 64) * U)[:, None]
    half = HALF_STEP[dtype] if dtype == BF16 else 0.0
    pe = p * (rel + half)
    dx, dxb = strided((T, D), (D + pads[0], 1), dtype)
    dw, dwb = strided(tuple(w.shape), (w.shape[1] + pads[1], 1), dtype)
    prm = _params(T, D, V, dtype, wide, x, w, scale, lddx=D + pads[0], lddw=w.shape[1] + pads[1], dloss_scalar=int(scalar))
    be.dispatch_linear_xent_grad(x, w, t, lse, dloss, dx if only != "dw" else None, dw if only != "dx" else None, prm)
    dw_vd = _vd(dw, wide)
    for name, got, want, err, size, terms in (
            ("dx", dx, dx64, pe @ wv.double().abs(), p @ wv.double().abs(), V),
            ("dw", dw_vd, dw64, pe.t().contiguous() @ xz.abs(), p.t().contiguous() @ xz.abs(), T)):
        if only and only != name:
            continue
        tol = err + (terms + 8) * U * size + HALF_STEP[dtype] * want.abs()
        assert bool(((got.double() - want).abs() <= tol).all()), name
        fp32 = (p * rel) @ wv.double().abs() if name == "dx" else (p * rel).t().contiguous() @ xz.abs()
        bound = HALF_STEP[dtype] * want.norm() + half * p.norm() * _largest_stretch(wv if name == "dx" else xz) + (
            fp32 + (terms + 8) * U * size).norm()
        assert float((got.double() - want).norm()) <= float(bound), name
    assert untouched(dx, dxb) and untouched(dw, dwb)
    assert only == "dw" or bool((dx[~live] == 0).all())
    return dx, dw


SIZES = [(1, 8, 8), (1, 64, 1000), (3, 100, 333), (32, 128, 2048), (33, 96, 77), (64, 64, 50), (65, 200, 515),
         (129, 256, 1001), (130, 64, 256), (257, 520, 3000), (300, 72, 4099), (600, 1024, 1536)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wide", ["vd", "dv"])
@pytest.mark.parametrize("T,D,V", SIZES)
def test_sizes(be, dtype, wide, T, D, V):
    x, w, t = _case(T, D, V, dtype, wide, T + V)
    if T > 2:
        t[1], t[2] = -1, V  # left out
    if T > 40:
        t[10:20] = -100
    _, lse, _ = _forward(be, x, w, t, dtype, wide)
    g = torch.randn(T, device="cuda")
    _gradient(be, x, w, t, lse, g, dtype, wide)


@pytest.mark.parametrize("wide,D,V", [("vd", 3, 5), ("dv", 1, 3), ("vd", 1, 1), ("dv", 5, 40)])
def test_tiny_fp32(be, wide, D, V):
    x, w, t = _case(6, D, V, F32, wide, 5)
    _, lse, _ = _forward(be, x, w, t, F32, wide)
    _gradient(be, x, w, t, lse, None, F32, wide)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wide,D,V", [("vd", 8, 1), ("vd", 8, 3), ("dv", 8, 8), ("vd", 9, 9), ("dv", 11, 17)])
def test_small_vocabularies(be, dtype, wide, D, V):
    for T in (1, 5, 200):
        x, w, t = _case(T, D, V, dtype, wide, 6)
        _, lse, _ = _forward(be, x, w, t, dtype, wide)
        g = torch.rand(T, device="cuda") + 0.5
        T_, one = x.shape[0], V == 1
        if one:  # the only logit: dz = 0 up to exp's rounding, relative to nothing
            dx, dw = torch.empty_like(x.contiguous()), torch.empty_like(w.contiguous())
            be.dispatch_linear_xent_grad(x, w, t, lse, g, dx, dw, _params(T_, D, V, dtype, wide, x, w))
            bound = (2 * float(_logit_error(x, _vd(w, wide), 1.0).max()) + 130 * U) * 1.5 * 1.01
            assert float(dx.abs().max()) <= bound * float(w.abs().max())
            assert float(dw.abs().max()) <= bound * T * float(x.abs().max())
        else:
            _gradient(be, x, w, t, lse, g, dtype, wide)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wide", ["vd", "dv"])
@pytest.mark.parametrize("pads,scale", [((1, 3), 0.5), ((8, 16), -1.25), ((4, 0), 2.0)])
def test_strides_scales_and_scalars(be, dtype, wide, pads, scale):
    T, D, V = 150, 96, 1300
    x, w, t = _case(T, D, V, dtype, wide, 3, pads)
    t[5] = 1 << 30
    _, lse, _ = _forward(be, x, w, t, dtype, wide, scale)
    _gradient(be, x, w, t, lse, torch.full((1,), 1.0 / 149, device="cuda"), dtype, wide, scale, pads, scalar=True)
    full = _gradient(be, x, w, t, lse, None, dtype, wide, scale, pads)
    for only in ("dx", "dw"):
        part = _gradient(be, x, w, t, lse, None, dtype, wide, scale, pads, only=only)
        i = only == "dw"
        assert torch.equal(part[i], full[i])


@pytest.mark.parametrize("dtype,wide,T,D,V", [(BF16, "vd", 20000, 64, 15400), (BF16, "dv", 20000, 64, 15400),
                                              (BF16, "vd", 70003, 40, 4100), (BF16, "dv", 70003, 40, 4099),
                                              (F32, "vd", 20000, 64, 7000), (F32, "dv", 20000, 64, 7001)])
def test_pieces(be, dtype, wide, T, D, V):
    """Several pieces of the vocabulary, a last one of odd size, dx in planes."""
    x, w, t = _case(T, D, V, dtype, wide, 4)
    t[::7] = -1
    _, lse, _ = _forward(be, x, w, t, dtype, wide)
    _gradient(be, x, w, t, lse, None, dtype, wide)


@pytest.mark.parametrize("wide", ["vd", "dv"])
@pytest.mark.parametrize("T,D,V", [(300, 64, 33000), (600, 1536, 33000)])
def test_last_round_and_planes(be, wide, T, D, V):
    """258 tiles: the last round's columns on smaller ones (a target at each side
    of the border); 387: one kernel; and dx's few tiles split over planes of K."""
    x, w, t = _case(T, D, V, BF16, wide, 12)
    t[:6] = torch.tensor([0, 32767, 32768, 32999, -1, 32760], dtype=torch.int32)
    _, lse, _ = _forward(be, x, w, t, BF16, wide)
    last = "bwpp_xent_stats_r128" if T == 300 else "bwpp_xent_stats_p"
    assert be.recent_kernel(2).startswith(last)  # then the join and the sums
    _gradient(be, x, w, t, lse, None, BF16, wide)


@pytest.mark.parametrize("wide", ["vd", "dv"])
@pytest.mark.parametrize("T,D,V", [(2048, 1024, 8205), (2050, 1040, 8200), (1500, 2056, 4100)])
def test_ragged_wide_products(be, wide, T, D, V):
    """Products on the wide tiles with ragged sizes on every side: tokens and
    vocabulary that are no multiple of 32 (dx in two products, dW's K filled up
    with zero rows), rows of dW that start anywhere."""
    x, w, t = _case(T, D, V, BF16, wide, 14, (0, 8 - (V % 8) if wide == "dv" else 0))
    t[::11] = -1
    _, lse, _ = _forward(be, x, w, t, BF16, wide)
    _gradient(be, x, w, t, lse, None, BF16, wide)
    _gradient(be, x, w, t, lse, None, BF16, wide, pads=(3, 1))
    assert be.recent_kernel(1) == "bwpp_xent_rows_p_t10" or be.recent_kernel(0) == "bwpp_xent_round_bf16"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wide", ["vd", "dv"])
def test_left_out_rows_hold_anything(be, dtype, wide):
    T, D, V = 140, 64, 700
    x, w, t = _case(T, D, V, dtype, wide, 9)
    dead = torch.arange(0, T, 9, device="cuda")
    t[dead] = -1
    clean = x.clone()
    clean[dead] = 0.0
    x[dead[0]], x[dead[1]], x[dead[2], 3] = float("nan"), float("inf"), -float("inf")
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    sums = torch.empty(2, device="cuda")
    p = _params(T, D, V, dtype, wide, x, w)
    be.dispatch_linear_xent(x, w, t, loss, lse, sums, p)
    want = torch.empty_like(loss), torch.empty_like(lse), torch.empty_like(sums)
    be.dispatch_linear_xent(clean, w, t, *want, p)
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[dead] = False
    assert torch.equal(loss, want[0]) and torch.equal(lse[keep], want[1][keep]) and torch.equal(sums, want[2])
    a, b = ((torch.empty_like(clean), torch.empty_like(w)) for _ in range(2))
    be.dispatch_linear_xent_grad(x, w, t, lse, None, *a, p)
    be.dispatch_linear_xent_grad(clean, w, t, want[1], None, *b, p)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # nothing counts at all
    t[:] = -1
    be.dispatch_linear_xent(x, w, t, loss, lse, sums, p)
    be.dispatch_linear_xent_grad(x, w, t, lse, None, *a, p)
    assert all(bool((v == 0).all()) for v in (loss, sums, *a))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_extreme_logits(be, dtype):
    """Logits to 3e4 (all but the largest vanish), one vocabulary row of -inf
    logits, and an infinite logit: lse is infinite, as the formula's."""
    T, D, V = 40, 32, 400
    x, w, t = _case(T, D, V, dtype, "vd", 2, lean=0.0)
    big = (x.float() * 1000).to(dtype)
    _forward(be, big, w, t, dtype, "vd")
    x[:, 0] = 1.0
    w[7, 0] = -float("inf")
    t[t == 7] = 8
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    p = _params(T, D, V, dtype, "vd", x, w)
    be.dispatch_linear_xent(x, w, t, loss, lse, None, p)
    rest = [i for i in range(V) if i != 7]
    want = torch.logsumexp(x.double() @ w[rest].double().t().contiguous(), dim=1)
    assert bool(((lse.double() - want).abs() <= 1e-4).all())
    w[7, 0] = float("inf")
    be.dispatch_linear_xent(x, w, t, loss, lse, None, p)
    assert bool(torch.isposinf(lse).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 17, 64, 65, 300])
def test_outputs_left_out(be, dtype, T):
    x, w, t = _case(T, 64, 200, dtype, "vd", 2)
    t[T // 2] = -1
    p = _params(T, 64, 200, dtype, "vd", x, w)
    full = torch.empty(T, device="cuda"), torch.empty(T, device="cuda"), torch.empty(2, device="cuda")
    be.dispatch_linear_xent(x, w, t, *full, p)
    for keep in (0, 1, 2):
        got = [torch.empty_like(v) if i == keep else None for i, v in enumerate(full)]
        be.dispatch_linear_xent(x, w, t, *got, p)
        assert torch.equal(got[keep], full[keep])


def test_no_rows(be):
    w = torch.ones(20, 16, device="cuda")
    t = torch.zeros(1, device="cuda", dtype=torch.int32)
    sums, dw = torch.full((2,), 7.0, device="cuda"), torch.full((20, 18), 7.0, device="cuda")
    p = bwpp.LinearXentParams(rows=0, vocab=20, dim=16, trans_w=1, lddw=18)
    be.dispatch_linear_xent(w, w, t, None, None, sums, p)
    be.dispatch_linear_xent_grad(w, w, t, sums, None, None, dw, p)
    assert bool((sums == 0).all()) and bool((dw[:, :16] == 0).all()) and bool((dw[:, 16:] == 7.0).all())


def test_gradient_against_differences(be):
    T, D, V = 5, 24, 60
    x, w, t = _case(T, D, V, F32, "vd", 7)
    t[3] = -1
    g = torch.rand(T, device="cuda") + 0.5
    _, lse, _ = _forward(be, x, w, t, F32, "vd")
    dx, dw = _gradient(be, x, w, t, lse, g, F32, "vd")
    sx, sw = torch.randn(T, D, device="cuda", dtype=torch.float64), torch.randn(V, D, device="cuda", dtype=torch.float64)
    f = lambda h: float((xent64(x.double() + h * sx, w.double() + h * sw, t)[0] * g.double()).sum())
    h = 1e-5
    want = (f(h) - f(-h)) / (2 * h)
    have = float((dx.double() * sx).sum() + (dw.double() * sw).sum())
    size = float((dx.double() * sx).abs().sum() + (dw.double() * sw).abs().sum())
    assert abs(want - have) <= size * 1e-5


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recorded_graph_between_other_work(be, dtype):
    """Recorded after an eager call, replayed with eager calls of other sizes on
    the same handle between (which use the same workspace, in order)."""
    T, D, V = 200, 128, 3001
    x, w, t = _case(T, D, V, dtype, "vd", 8)
    x2, w2, t2 = _case(30, 64, 999, dtype, "dv", 9)
    p, p2 = _params(T, D, V, dtype, "vd", x, w), _params(30, 64, 999, dtype, "dv", x2, w2)
    out = [torch.empty(T, device="cuda"), torch.empty(T, device="cuda"), torch.empty(2, device="cuda"),
           torch.empty_like(x), torch.empty_like(w)]
    small = [torch.empty(30, device="cuda"), torch.empty(30, device="cuda"), torch.empty(2, device="cuda"),
             torch.empty_like(x2), torch.empty_like(w2)]

    def call(o, a, b, c, prm):
        be.dispatch_linear_xent(a, b, c, *o[:3], prm)
        be.dispatch_linear_xent_grad(a, b, c, o[1], None, o[3], o[4], prm)

    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(main)
    try:
        be.set_stream(side)
        call(out, x, w, t, p)
        side.synchronize()
        want = [v.clone() for v in out]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(out, x, w, t, p)
        for i in range(4):
            for v in out:
                v.fill_(3.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                graph.replay()
            call(small, x2, w2, t2, p2)
            torch.cuda.synchronize()
            for a, b in zip(out[:3], want[:3]):
                assert torch.equal(a, b), i
            # the products of a caller's recording do without the split scratch: sums in another order
            for a, b in zip(out[3:], want[3:]):
                assert float((a.double() - b.double()).norm() / b.double().norm()) <= (2.0 ** -8 if dtype == BF16 else 1e-6)
    finally:
        be.set_stream(main)


def test_recording_never_grows_the_workspace():
    """A first call inside a recording is refused; the recording goes on."""
    b = bwpp.HipBackend(0)
    T, D, V = 64, 64, 500
    x, w, t = _case(T, D, V, BF16, "vd", 8)
    loss = torch.empty(T, device="cuda")
    side = torch.cuda.Stream()
    b.set_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(bwpp.BwppError) as e:
            b.dispatch_linear_xent(x, w, t, loss, None, None, _params(T, D, V, BF16, "vd", x, w))
        loss.zero_()
    assert e.value.status == bwpp.Status.OUT_OF_MEMORY
    graph.replay()
    torch.cuda.synchronize()
    assert bool((loss == 0).all())
    b.close()


# ------------------------------------------- fp32 in bf16 terms (the matrix cores)
TERMS = [("vd", 300, 520, 3000, None), ("dv", 300, 520, 3001, None), ("vd", 777, 1021, 8003, True),
         ("dv", 777, 1021, 8003, True), ("dv", 1025, 33, 20000, None), ("vd", 2048, 1024, 4100, True),
         ("dv", 260, 2048, 33001, None), ("vd", 260, 2048, 33001, None), ("vd", 20011, 72, 7001, None),
         ("vd", 4100, 1024, 9001, True), ("dv", 4100, 1024, 9001, True), ("vd", 1025, 4100, 9001, True),
         ("dv", 1025, 4100, 9001, True)]


@pytest.mark.parametrize("wide,T,D,V,terms", TERMS)
def test_fp32_in_terms(be, wide, T, D, V, terms):
    """The same bounds hold: three bf16 terms are an fp32 number, the products of
    terms that are left out are 2^-26 of theirs.  Ragged on every side, in pieces
    (9001 columns, of the gradient for 4100 rows, of the loss too for 4100 dim),
    dx and dW in planes; and sizes near the choice's border."""
    x, w, t = _case(T, D, V, F32, wide, 15, (1, 3))
    t[::13] = -1
    t[3], t[4] = V - 1, 0
    _, lse, _ = _forward(be, x, w, t, F32, wide, 1.25)
    full = _gradient(be, x, w, t, lse, torch.randn(T, device="cuda"), F32, wide, 1.25, (3, 1))
    assert terms is None or any(be.recent_kernel(i).startswith("bwpp_xent_sums_s") for i in range(1, 5))
    assert full[0].isfinite().all()


@pytest.mark.parametrize("wide", ["vd", "dv"])
def test_fp32_terms_scale_exactly(be, wide):
    """Scaling x by 2^60 and W by 2^-60 changes no bit of the loss: the terms of a
    number are as large as it allows, none is lost."""
    T, D, V = 1200, 512, 8000
    x, w, t = _case(T, D, V, F32, wide, 16)
    x1, w1 = x * 2.0 ** 60, w * 2.0 ** -60
    out = []
    for a, b in ((x, w), (x1, w1)):
        p = _params(T, D, V, F32, wide, a, b)
        loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        be.dispatch_linear_xent(a, b, t, loss, lse, None, p)
        dx, dw = torch.empty_like(a), torch.empty_like(b)
        be.dispatch_linear_xent_grad(a, b, t, lse, None, dx, dw, p)
        out.append((loss, lse, dx, dw))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    assert torch.equal(out[0][2] * 2.0 ** -60, out[1][2]) and torch.equal(out[0][3] * 2.0 ** 60, out[1][3])


@pytest.mark.parametrize("wide", ["vd", "dv"])
def test_fp32_terms_infinities(be, wide):
    """As the formula's: a vocabulary row of -inf logits vanishes, an infinite or
    NaN token spoils its own row alone, a left-out one nothing."""
    T, D, V = 1200, 256, 8000
    x, w, t = _case(T, D, V, F32, wide, 17)
    wv = _vd(w, wide)
    x[:, 0] = 1.0
    wv[7, 0] = -float("inf")
    t[t == 7] = 8
    x[11, 5], x[12, 5], x[13, 5] = float("inf"), float("nan"), float("inf")
    t[13] = -1
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    p = _params(T, D, V, F32, wide, x, w)
    be.dispatch_linear_xent(x, w, t, loss, lse, None, p)
    assert any(be.recent_kernel(i).startswith("bwpp_xent_stats_s") for i in range(1, 3))
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[11:14] = False
    rest = torch.arange(V, device="cuda") != 7
    want, want_lse = xent64(x[keep].contiguous(), wv[rest].contiguous(), torch.where(t[keep] > 7, t[keep] - 1, t[keep]))[:2]
    e = _logit_error(x[keep], wv[rest], 1.0)
    tol = e + (V / 64 + 48) * U + U * want_lse.abs()
    assert bool(((lse[keep].double() - want_lse).abs() <= tol).all())
    assert bool(((loss[keep].double() - want).abs() <= tol + e).all())
    assert float(loss[13]) == 0.0 and not bool(loss[11:13].isfinite().any())
    wv[7, 0] = 1.0
    t[11] = t[12] = -1
    be.dispatch_linear_xent(x, w, t, loss, lse, None, p)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    be.dispatch_linear_xent_grad(x, w, t, lse, None, dx, dw, p)
    assert bool((dx[11:14] == 0).all()) and bool(dx.isfinite().all()) and bool(dw.isfinite().all())


@pytest.mark.parametrize("wide,T,D,V,dw_too", [
    ("vd", 2048, 1024, 8205, True), ("dv", 2048, 1024, 8200, True), ("vd", 9000, 512, 16400, False),
    ("dv", 9000, 520, 16400, False), ("vd", 9000, 1032, 16400, True), ("dv", 9000, 1032, 16400, True),
    ("vd", 300, 72, 2001, False), ("dv", 300, 72, 2000, False), ("vd", 210, 201, 9001, True), ("dv", 230, 600, 33000, True)])
def test_targets_keep_their_bits(be, wide, T, D, V, dw_too):
    """In dx and in dW of the wide products the targets' dz, the largest of their rows,
    counts with its rounding's remainder (rounded to bf16 for dW): two half steps of it are off,
    one after the other.  A log-sum-exp 7 above the logits' leaves little else in a
    row, so that one half step of dz would show in the elements' bound.  One target
    of many tokens (more than a step of the matrix instructions takes), the last of
    the vocabulary, and some left out; two pieces for 9000 tokens.  dW with few tiles
    for many tokens is another kernel's, and has dz's half step."""
    x, w, t = _case(T, D, V, BF16, wide, 18, lean=0.0)
    t[100:180], t[200:203], t[4000:] = 5, V - 1, torch.where(t[4000:] < 600, 600, t[4000:])
    t[::11] = -1
    wv, live = _vd(w, wide), t >= 0
    z = x.double() @ wv.double().t().contiguous()
    lse = (torch.logsumexp(z, dim=1) + 7.0).float()
    g = torch.rand(T, device="cuda") + 0.5
    p = torch.exp(z - lse.double()[:, None]) * torch.where(live, g.double(), 0.0)[:, None]
    rel = (_logit_error(x, wv, 1.0) + 20 * U)[:, None]
    err = p * (rel + HALF_STEP[BF16])
    rows = torch.arange(T, device="cuda")[live]
    cols = t[live].long()
    dz = p.clone()
    dz[rows, cols] -= g.double()[live]
    err[rows, cols] = p[rows, cols] * rel[live, 0] + dz[rows, cols].abs() * (HALF_STEP[BF16] ** 2 + 4 * U)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    be.dispatch_linear_xent_grad(x, w, t, lse, g, dx, dw, _params(T, D, V, BF16, wide, x, w))
    assert be.recent_kernel(0).startswith("bwpp_xent_round_bf16")
    assert (be.recent_kernel(1) == "bwpp_xent_rows_p_t10") == dw_too
    dw_err = err.clone()
    if not dw_too:
        dw_err[rows, cols] += dz[rows, cols].abs() * HALF_STEP[BF16]
    x64 = torch.where(live[:, None], x.double(), 0.0)
    for got, want, e, size, terms in (
            (dx, dz @ wv.double(), err @ wv.double().abs(), dz.abs() @ wv.double().abs(), V),
            (_vd(dw, wide), dz.t().contiguous() @ x64, dw_err.t().contiguous() @ x64.abs(), dz.t().contiguous().abs() @ x64.abs(), T)):
        assert bool(((got.double() - want).abs() <= e + (terms + 8) * U * size + HALF_STEP[BF16] * want.abs()).all())


def test_piece_with_a_short_rest(be):
    """A vocabulary one past a multiple of every narrower piece: pieces grow until
    the last has a chunk of 8 columns (stepping down would end at none)."""
    T, D, V = 131072, 8, 6145
    x, w, t = _case(T, D, V, BF16, "vd", 20)
    t[::5] = -1
    lse = torch.empty(T, device="cuda")
    p = _params(T, D, V, BF16, "vd", x, w)
    be.dispatch_linear_xent(x, w, t, None, lse, None, p)
    _gradient(be, x, w, t, lse, None, BF16, "vd")

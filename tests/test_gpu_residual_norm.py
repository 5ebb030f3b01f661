"""The residual join with its norms, and its gradient, against 64-bit forms.

Bounds.  A sum of n squares or products in fp32, taken 8 or 16 a thread and then
in a tree, is off by at most (16 + 10 + 2) x 2^-24 of its terms' magnitudes;
halved by the root and with a division, a root and the addition of eps, rstd is
off by at most 18 x 2^-24 relative.  r adds at most 6 roundings of its terms, y
rstd's error twice over (its own and that of r's terms) and 4 roundings; t, do
and the column terms at most 2 rstd's, one mean (30 x 2^-24) and 10 roundings:
80 x 2^-24 of the magnitudes of their terms, which the 64-bit form adds up, and
column sums of n rows n + 64 more in the worst order.  Rows over 16384 columns
are summed 32 and more a thread: (cols / 512) x 2^-24 more."""
import pytest
import torch

import bwpp
from lm64 import HALF_STEP, resnorm64, resnorm_grad64, strided, untouched

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(1234)


F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
EPS = 1e-6

COLS = [1, 3, 7, 8, 63, 64, 511, 512, 513, 1000, 1024, 1026, 2047, 2048, 4096, 4098, 8191, 8192, 8200, 16384, 16391]


def _in(rows, cols, ld, dtype, g, std=1.0):
    return strided((rows, cols), (ld, 1), dtype, torch.randn(rows, cols, device="cuda", generator=g).mul_(std))[0]


def _case(rows, cols, dtype, pads, post, gate_rows, pre, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ldx, ldo, ldy, ldg = (cols + p for p in pads)
    n = (rows + gate_rows - 1) // gate_rows if gate_rows else 1
    w = lambda: (torch.rand(cols, device="cuda", generator=g) + 0.5).to(dtype)
    c = dict(x=_in(rows, cols, ldx, dtype, g, 3.0), o=_in(rows, cols, ldo, dtype, g, 0.5),
             gate=None if gate_rows is None else _in(n, cols, ldg, dtype, g), post=w() if post == 2 else None,
             pre=w() if pre else None, dr=_in(rows, cols, ldx, dtype, g), dy=_in(rows, cols, ldy, dtype, g))
    p = bwpp.ResidualNormParams(rows=rows, cols=cols, ldx=ldx, ldo=ldo, ldy=ldy, ldg=ldg, post_norm=int(post > 0),
                                gate_rows=gate_rows or 0, eps=EPS, stream_scale=1.5, branch_scale=-0.25,
                                dtype=int(dtype == BF16))
    return c, p


def _forward(be, c, p, rows, cols, dtype, in_place=False):
    gr, post_norm = p.gate_rows, bool(p.post_norm)
    want_r, want_y, size = resnorm64(c["x"], c["o"], c["post"], c["gate"], c["pre"], gr, EPS, 1.5, -0.25, post_norm)
    hs, extra = HALF_STEP[dtype], cols / 512
    r, rbuf = strided((rows, cols), (p.ldx, 1), dtype, c["x"] if in_place else None)
    y, ybuf = strided((rows, cols), (p.ldy, 1), dtype)
    be.dispatch_residual_norm(r if in_place else c["x"], c["o"], c["post"], c["gate"], c["pre"], r, y, p)
    tol_r = hs * want_r.abs() + (24 + extra) * U * size
    assert bool(((r.double() - want_r).abs() <= tol_r).all())
    ir = want_y.abs() / want_r.abs().clamp(min=1e-30)
    tol_y = hs * want_y.abs() + (46 + 2 * extra) * U * (want_y.abs() + ir * size)
    assert bool(((y.double() - want_y).abs() <= tol_y).all())
    assert untouched(r, rbuf) and untouched(y, ybuf)
    return r, y


def _gradient(be, c, p, rows, cols, dtype, outs=("dx", "do", "dpost", "dgate", "dpre"), dr_in_place=False):
    gr, post_norm = p.gate_rows, bool(p.post_norm)
    want = resnorm_grad64(c["o"], c["x"], c["post"], c["gate"], c["pre"], c["dr"], c["dy"], gr, EPS, 1.5, -0.25, post_norm)
    n = (rows + gr - 1) // gr if gr else 1
    shapes = dict(dx=((rows, cols), (p.ldx, 1)), do=((rows, cols), (p.ldo, 1)), dgate=((n, cols), (p.ldg, 1)),
                  dpost=((cols,), (1,)), dpre=((cols,), (1,)))
    got = {k: strided(*shapes[k], dtype) for k in outs if not (k == "dpost" and not post_norm)}
    dr = c["dr"]
    if dr_in_place:
        got["dx"][0].copy_(dr)
        dr = got["dx"][0]
    ptr = lambda k: got[k][0] if k in got else None
    be.dispatch_residual_norm_grad(c["o"], c["x"], c["post"], c["gate"], c["pre"], dr, c["dy"], ptr("dx"), ptr("do"),
                                   ptr("dpost"), ptr("dgate"), ptr("dpre"), p)
    hs, extra = HALF_STEP[dtype], 2 * cols / 512
    for k, (t, buf) in got.items():
        w, size = want[k]
        n_sum = 0 if k in ("dx", "do") else rows + 64
        tol = hs * w.abs() + (80 + extra + n_sum) * U * size
        assert bool(((t.double() - w).abs() <= tol).all()), (k, float(((t.double() - w).abs() - tol).max()))
        assert untouched(t, buf), k
    return {k: t for k, (t, _) in got.items()}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", COLS)
def test_row_lengths(be, dtype, cols):
    for rows, pads, post, gate_rows, pre in ((5, (0, 0, 0, 0), 2, 0, True), (9, (1, 2, 3, 5), 1, 4, False)):
        c, p = _case(rows, cols, dtype, pads, post, gate_rows, pre, cols)
        _forward(be, c, p, rows, cols, dtype)
        _gradient(be, c, p, rows, cols, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 4096), (3, 100), (700, 520), (4100, 64), (1030, 4096), (2100, 2050)])
@pytest.mark.parametrize("gate_rows", [None, 0, 1, 7, 512, 100000])
def test_gates_and_many_rows(be, dtype, rows, cols, gate_rows):
    """Workers that share a gate row, that take one each, and several."""
    c, p = _case(rows, cols, dtype, (8, 0, 8, 0), rows % 3, gate_rows, True, rows)
    _forward(be, c, p, rows, cols, dtype)
    _gradient(be, c, p, rows, cols, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [40, 4096, 20000])
def test_in_place_and_left_out(be, dtype, cols):
    c, p = _case(37, cols, dtype, (0, 0, 0, 0), 2, 5, True, 1)
    a = _forward(be, c, p, 37, cols, dtype)
    b = _forward(be, c, p, 37, cols, dtype, in_place=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    r = torch.full_like(a[0], 7.0)
    be.dispatch_residual_norm(c["x"], c["o"], c["post"], c["gate"], None, r, None, p)  # no norm after
    assert torch.equal(r, a[0])
    full = _gradient(be, c, p, 37, cols, dtype)
    again = _gradient(be, c, p, 37, cols, dtype, dr_in_place=True)
    for k in full:
        assert torch.equal(full[k], again[k]), k
    for outs in (("dx",), ("do",), ("dpre",), ("dgate",), ("dpost", "dx")):
        part = _gradient(be, c, p, 37, cols, dtype, outs=outs)
        for k in part:
            # without dgate the rows are cut otherwise: sums in another order
            assert k in ("dpre", "dpost") or torch.equal(part[k], full[k]), k
    for gone in ("dr", "dy"):
        d = dict(c)
        d[gone] = None
        _gradient(be, d, p, 37, cols, dtype)


def test_gradient_against_differences(be):
    """Central differences of a weighted sum of r and y, computed in 64 bits, in
    directions of all inputs at once."""
    rows, cols = 6, 40
    c, p = _case(rows, cols, F32, (0, 0, 0, 0), 2, 3, True, 5)
    c64 = {k: v.double() for k, v in c.items()}
    r64 = resnorm64(c64["x"], c64["o"], c64["post"], c64["gate"], c64["pre"], 3, EPS, 1.5, -0.25, True)[0]
    c["stream"], c["x"] = c["x"], r64.float()  # the gradient takes r
    got = _gradient(be, c, p, rows, cols, F32)
    gen = torch.Generator(device="cuda").manual_seed(9)
    names = dict(x="dx", o="do", post="dpost", gate="dgate", pre="dpre")
    step = {k: torch.randn(c64[k].shape, device="cuda", generator=gen, dtype=torch.float64) for k in names}

    def f(h):
        v = {k: c64[k] + h * step[k] for k in names}
        r, y, _ = resnorm64(v["x"], v["o"], v["post"], v["gate"], v["pre"], 3, EPS, 1.5, -0.25, True)
        return float((r * c64["dr"]).sum() + (y * c64["dy"]).sum())

    h = 1e-5
    want = (f(h) - f(-h)) / (2 * h)
    have = sum(float((got[d].double() * step[k]).sum()) for k, d in names.items())
    size = sum(float((got[d].double() * step[k]).abs().sum()) for k, d in names.items())
    # differences: h^2 and 2^-52 / h; the gradients and r's rounding: 200 x 2^-24
    assert abs(want - have) <= size * (200 * U + 1e-8)


def test_zero_rows_zero_branch_and_non_finite(be):
    """A row of zeros has rstd 1/sqrt(eps); an infinity or NaN stays in its row."""
    rows, cols = 8, 96
    c, p = _case(rows, cols, F32, (0, 0, 0, 0), 2, 0, True, 3)
    r0, y0 = _forward(be, c, p, rows, cols, F32)
    g0 = _gradient(be, c, p, rows, cols, F32)
    bad = {k: (v.clone() if v is not None else None) for k, v in c.items()}
    bad["o"][2, 5], bad["x"][4, 7] = float("nan"), float("inf")
    r, y = torch.empty_like(r0), torch.empty_like(y0)
    be.dispatch_residual_norm(bad["x"], bad["o"], bad["post"], bad["gate"], bad["pre"], r, y, p)
    keep = [0, 1, 3, 5, 6, 7]
    assert torch.equal(r[keep], r0[keep]) and torch.equal(y[keep], y0[keep])
    dx, do = torch.empty_like(r0), torch.empty_like(r0)
    be.dispatch_residual_norm_grad(bad["o"], bad["x"], bad["post"], bad["gate"], bad["pre"], bad["dr"], bad["dy"], dx,
                                   do, None, None, None, p)
    assert torch.equal(dx[keep], g0["dx"][keep]) and torch.equal(do[keep], g0["do"][keep])
    c["x"][1] = 0.0
    c["o"][1] = 0.0
    _forward(be, c, p, rows, cols, F32)
    _gradient(be, c, p, rows, cols, F32)


@pytest.mark.parametrize("gate_rows", [0, 4])
def test_no_rows(be, gate_rows):
    """Sums over no rows are zero (a gate row per rows: there is none)."""
    x = torch.zeros(1, 64, device="cuda")
    o, y = torch.zeros(1, 64, device="cuda"), torch.full((1, 64), 7.0, device="cuda")
    p = bwpp.ResidualNormParams(rows=0, cols=64, eps=EPS, post_norm=1, gate_rows=gate_rows)
    be.dispatch_residual_norm(x, o, None, None, None, y, None, p)
    d = [torch.full((64,), 7.0, device="cuda") for _ in range(3)]
    be.dispatch_residual_norm_grad(o, x, None, None, None, x, None, None, None, d[0], d[1], d[2], p)
    assert bool((y == 7.0).all()) and bool((d[0] == 0).all()) and bool((d[2] == 0).all())
    assert bool((d[1] == (7.0 if gate_rows else 0.0)).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recorded_graph_and_another_stream(be, dtype):
    """Recorded after one eager call (the workspace has its size), replayed
    between eager calls, on a stream of its own."""
    rows, cols = 300, 1000
    c, p = _case(rows, cols, dtype, (0, 0, 0, 0), 2, 50, True, 8)
    want = _gradient(be, c, p, rows, cols, dtype)
    out = {k: torch.empty_like(v) for k, v in want.items()}
    side = torch.cuda.Stream()
    main = torch.cuda.current_stream()

    def call():
        be.dispatch_residual_norm_grad(c["o"], c["x"], c["post"], c["gate"], c["pre"], c["dr"], c["dy"], out["dx"],
                                       out["do"], out["dpost"], out["dgate"], out["dpre"], p)

    side.wait_stream(main)
    try:
        be.set_stream(side)
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    finally:
        be.set_stream(main)
    for i in range(4):
        for v in out.values():
            v.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(out[k], want[k]), (k, i)
        be.dispatch_residual_norm(c["x"], c["o"], None, None, None, out["dx"], out["do"], p)

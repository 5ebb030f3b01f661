"""Rules on logits against a 64-bit form.  Bounds, u = 2^-24: the penalty is one
rounding of z / r or z r (u), frequency times count plus presence two (2 u of the
sum of their magnitudes), and every subtraction and addition one of its result;
so 4 u of |z| max(r, 1 / r, 1) + |frequency| count + |presence| + |bias| covers
them, and the output's rounding comes on top."""
import math

import pytest
import torch

import bwpp
from cache64 import BF16, F32, bits, i32
from lm64 import HALF_STEP, strided, untouched

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def rules64(x, history, starts, prompt, rep, pres, freq, bias, mask):
    z = x.double()
    size = z.abs()
    R, V = z.shape
    for r in range(R):
        past = [t for t in history[max(0, starts[r]):max(0, starts[r + 1])]]
        given = max(0, prompt[r]) if prompt is not None else 0
        for t in set(past):
            if not 0 <= t < V:
                continue
            n = sum(1 for u in past[given:] if u == t)
            if rep is not None:
                rho = float(rep[r])
                z[r, t] = z[r, t] / rho if z[r, t] > 0 else z[r, t] * rho
                size[r, t] = size[r, t] * max(rho, 1 / rho, 1.0)
            if n:
                f, p = (float(a[r]) if a is not None else 0.0 for a in (freq, pres))
                z[r, t] -= f * n + p
                size[r, t] += abs(f) * n + abs(p)
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    if mask is not None:
        z = z.masked_fill(~mask, -math.inf)
    return z, size


def _check(be, R, V, tx, ty, lengths, prompt=True, rep=True, pres=True, freq=True, bias="shared", mask="rows", pad=0,
           in_place=False, seed=0, x=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    xv = (rnd(R, V) * 4).to(tx) if x is None else x
    x, xbuf = strided((R, V), (V + pad, 1), tx, xv)
    y, ybuf = (x, xbuf) if in_place else strided((R, V), (V + 2 * pad, 1), ty)
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    history = torch.randint(-2, min(V, 50) + 2, (starts[-1],), generator=g, device="cuda", dtype=torch.int32)
    given = [n // 3 for n in lengths]
    rho = torch.rand(R, generator=g, device="cuda") + 0.6 if rep else None
    p, f = (rnd(R) if pres else None), (rnd(R) if freq else None)
    b = None if bias is None else rnd(1 if bias == "shared" else R, V + pad)
    m = None if mask is None else torch.rand(1 if mask == "shared" else R, V, generator=g, device="cuda") < 0.7
    want, size = rules64(xv, history.tolist(), starts, given if prompt else None, rho, p, f,
                         None if b is None else b[:, :V], m)
    par = bwpp.LogitRulesParams(rows=R, vocab=V, ldx=x.stride(0), ldy=y.stride(0), dtype_x=int(tx == BF16),
                                dtype_y=int(ty == BF16), history=starts[-1],
                                ld_bias=V + pad if bias == "rows" else 0, ld_mask=-(-V // 32) if mask == "rows" else 0)
    be.dispatch_logit_rules(x, history, i32(starts), i32(given) if prompt else None, rho, p, f, b,
                            None if m is None else bits(m), y, par)
    torch.cuda.synchronize()
    hidden = torch.zeros_like(want, dtype=torch.bool) if m is None else ~m.expand(R, V)
    assert bool((y[hidden] == -math.inf).all())
    tol = HALF_STEP[ty] * want.abs() + 4 * U * (1 + HALF_STEP[ty]) * size
    got = y.double()
    fine = ((got - want).abs() <= tol) | (got == want) | (torch.isnan(want) & torch.isnan(got))
    assert bool(fine[~hidden].all())
    assert untouched(y, ybuf) and untouched(x, xbuf)


@pytest.mark.parametrize("tx,ty", [(F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("R,V,pad", [(1, 1, 0), (3, 31, 1), (2, 33, 0), (5, 1000, 0), (1, 20000, 3), (4, 4097, 1), (300, 130, 0)])
def test_rules(be, tx, ty, R, V, pad):
    lengths = [(7 * r + 90) % 133 for r in range(R)]
    _check(be, R, V, tx, ty, lengths, pad=pad)
    _check(be, R, V, tx, ty, lengths, pad=pad, bias="rows", mask="shared", prompt=False, seed=1)


@pytest.mark.parametrize("rep,pres,freq", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 0, 0), (1, 1, 0)])
def test_single_rules(be, rep, pres, freq):
    _check(be, 3, 500, F32, F32, [40, 0, 77], rep=rep, pres=pres, freq=freq, bias=None, mask=None)
    _check(be, 3, 500, BF16, F32, [0, 0, 0], rep=rep, pres=pres, freq=freq, bias=None)
    _check(be, 3, 500, F32, F32, [40, 5, 77], rep=rep, pres=pres, freq=freq, mask=None)


@pytest.mark.parametrize("t", [F32, BF16])
def test_in_place_and_wide(be, t):
    _check(be, 2, 777, t, t, [50, 60], in_place=True, pad=1)
    _check(be, 40, 70001, t, t, [100] * 40, seed=3)      # the widest chunks
    _check(be, 2, 3000, t, F32, [200000, 3], seed=4)      # a long history


def test_infinities_and_nan(be):
    x = torch.randn(2, 200, device="cuda")
    x[0, 3], x[0, 7], x[1, 9], x[0, 64] = math.inf, -math.inf, math.nan, -0.0
    _check(be, 2, 200, F32, F32, [150, 150], bias=None, mask=None, x=x)
    x[:, :] = math.nan
    m = torch.zeros(2, 200, dtype=torch.bool, device="cuda")
    y = torch.empty_like(x)
    be.dispatch_logit_rules(x, None, None, None, None, None, None, None, bits(m), y,
                            bwpp.LogitRulesParams(rows=2, vocab=200, ld_mask=7))
    assert bool((y == -math.inf).all())  # nothing allowed


def test_history_is_cut(be):
    """Starts outside the history, ends before beginnings, counts of the given
    part below zero and past the end."""
    x = torch.ones(4, 64, device="cuda")
    y = torch.empty_like(x)
    history = i32([1, 2, 3, 4])
    be.dispatch_logit_rules(x, history, i32([-5, 2, 1, 3, 2 ** 31 - 1]), i32([-1, 0, 99, 0]), None, None,
                            torch.full((4,), 0.5, device="cuda"), None, None, y,
                            bwpp.LogitRulesParams(rows=4, vocab=64, history=4))
    want = x.clone()
    want[0, 1] = want[0, 2] = want[3, 4] = 0.5  # row 2's are all given
    assert bool((y == want).all())

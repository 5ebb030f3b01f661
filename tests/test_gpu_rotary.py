"""Rotary positions against a 64-bit form.  Error of an element y = m (p cos a
-+ q sin a) in fp32: cosine and sine are off by at most 2 steps of 2^-24 (the
remainder's rounding, the series, its last addition) and, times m, half a step
more; a product and the sum half a step each, so 4 x 2^-24 of m (|p| + |q|)
covers it (the angle's 2^-52 p f is 2^-30 at most here), and the output's
rounding comes on top."""
import pytest
import torch

import bwpp
from lm64 import HALF_STEP, rotary64, strided, untouched

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(1234)


F32, BF16 = torch.float32, torch.bfloat16
PARTS = dict(scaling=2, factor=16.0, context=8192, low_turns=1.0, high_turns=32.0, magnitude=1.25)


def _strides(order, B, T, H, d, pad):
    """[B, T, H, d] strides for the row orders in use."""
    if order == "bshd":
        ts = H * d + pad
        return (T * ts, ts, d, 1)
    hs = T * (d + pad)
    return (H * hs, d + pad, hs, 1)


def _check(be, dtype, B, T, Hq, Hk, d, rot, inter, scal, positions, order_in, order_out, pad=0, grad=False, offset=0,
           in_place=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda H: torch.randn(B, T, H, d, device="cuda", generator=g).to(dtype)
    pos = None
    if positions:
        pos = torch.randint(-1000, 1 << 20, (B, T + 3), device="cuda", dtype=torch.int32, generator=g)
    p64 = pos[:, :T] if positions else (torch.arange(T, device="cuda") + offset)[None, :].expand(B, T)
    kw = dict(scal)
    sides = {}
    for name, H in (("q", Hq), ("k", Hk)):
        si = _strides(order_in, B, T, max(H, 1), d, pad)
        so = si if in_place else _strides(order_out, B, T, max(H, 1), d, pad)
        v = mk(max(H, 1))
        src, sbuf = strided(v.shape, si, dtype, v)
        dst, dbuf = (src, sbuf) if in_place else strided(v.shape, so, dtype)
        sides[name] = (v, src, dst, dbuf, H)
        a, b = (name + "o", name) if grad else (name, name + "o")
        for key, s in ((a, si), (b, so)):
            kw["ld" + key], kw[key + "_head_stride"], kw[key + "_batch_stride"] = s[1], s[2], s[0]
    p = bwpp.RotaryParams(tokens=T, q_heads=Hq, k_heads=Hk, dim=d, batch=B, rot_dim=rot, layout=int(inter),
                          dtype=int(dtype == BF16), pos_batch_stride=T + 3 if positions else 0, pos_offset=offset, **kw)
    fn = be.dispatch_rotary_grad if grad else be.dispatch_rotary
    fn(sides["q"][1] if Hq else None, sides["k"][1] if Hk else None, pos, sides["q"][2] if Hq else None,
       sides["k"][2] if Hk else None, p)
    for v, src, dst, dbuf, H in sides.values():
        if H == 0:
            continue
        want, size = rotary64(v, p64, rot or d, inter, scaling=scal.get("scaling", 0), factor=scal.get("factor", 1.0),
                              context=scal.get("context", 0), low=scal.get("low_turns", 0.0),
                              high=scal.get("high_turns", 0.0), magnitude=scal.get("magnitude", 1.0), grad=grad)
        err = (dst.double() - want).abs()
        n = rot or d
        tol = HALF_STEP[dtype] * want.abs() + 4 * 2.0 ** -24 * (1 + HALF_STEP[dtype]) * size
        tol[..., n:] = 0.0  # copied
        assert bool((err <= tol).all()), float((err - tol).max())
        assert untouched(dst, dbuf)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hk,d,rot", [(1, 1, 1, 1, 2, 0), (2, 3, 4, 2, 64, 0), (1, 65, 3, 1, 128, 0),
                                             (3, 37, 5, 5, 80, 40), (2, 9, 2, 1, 96, 24), (1, 130, 7, 2, 50, 34),
                                             (2, 5, 40, 8, 256, 128), (1, 17, 1, 1, 33, 6), (1, 4, 1, 1, 600, 600)])
def test_sizes(be, dtype, inter, B, T, Hq, Hk, d, rot):
    _check(be, dtype, B, T, Hq, Hk, d, rot, inter, {}, True, "bshd", "bhsd")
    _check(be, dtype, B, T, Hq, Hk, d, rot, inter, PARTS, True, "bhsd", "bshd", pad=3, grad=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scal", [{}, dict(scaling=1, factor=4.0), PARTS, dict(magnitude=-0.5)])
@pytest.mark.parametrize("grad", [False, True])
def test_scalings(be, dtype, scal, grad):
    _check(be, dtype, 2, 33, 4, 2, 128, 64, False, scal, False, "bshd", "bshd", grad=grad, offset=100000)
    _check(be, dtype, 2, 33, 4, 2, 128, 64, True, scal, True, "bshd", "bhsd", pad=1, grad=grad)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rot", [0, 32, 36, 6])
def test_in_place_and_one_side(be, dtype, inter, rot):
    _check(be, dtype, 2, 19, 4, 2, 64, rot, inter, {}, True, "bshd", "bshd", pad=5, in_place=True)
    _check(be, dtype, 2, 19, 4, 0, 64, rot, inter, {}, False, "bshd", "bhsd")
    _check(be, dtype, 2, 19, 0, 3, 64, rot, inter, {}, False, "bhsd", "bshd", offset=-7)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_tokens_and_heads(be, dtype):
    """Tiles of several tokens with a last one that is not full, and more heads
    than a block takes."""
    _check(be, dtype, 3, 2801, 4, 1, 32, 0, False, {}, True, "bshd", "bshd")
    _check(be, dtype, 1, 3, 300, 213, 32, 16, True, {}, True, "bshd", "bshd")


def test_gradient_is_the_transpose(be):
    """<R x, g> = <x, R^T g> to the rounding of the sums, and R^T R = m^2."""
    B, T, H, d = 2, 40, 3, 64
    x, g = (torch.randn(B, H, T, d, device="cuda", dtype=F32) for _ in range(2))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    p = bwpp.RotaryParams(tokens=T, q_heads=H, dim=d, batch=B, rot_dim=48, pos_offset=5000, **PARTS)
    be.dispatch_rotary(x, None, None, y, None, p)
    be.dispatch_rotary_grad(g, None, None, dx, None, p)
    a, b = (y.double() * g.double()).sum(), (x.double() * dx.double()).sum()
    bound = 8 * 2.0 ** -24 * 1.25 * 2 * (x.abs().double().sum() * g.abs().double().max())
    assert abs(float(a - b)) <= float(bound)
    be.dispatch_rotary_grad(y, None, None, dx, None, p)
    m2 = torch.ones(d, device="cuda", dtype=torch.float64)
    m2[:48] = 1.25 ** 2
    assert bool(((dx.double() - m2 * x.double()).abs() <= 20 * 2.0 ** -24 * 1.5625 * x.abs().double().amax()).all())


def test_shared_positions_and_empty(be):
    """pos_batch_stride 0: one row of positions for every batch; no tokens:
    nothing is written."""
    B, T, H, d = 3, 8, 2, 16
    pos = torch.randint(0, 1000, (T,), device="cuda", dtype=torch.int32)
    x = torch.randn(B, H, T, d, device="cuda")
    y = torch.full_like(x, 7.0)
    be.dispatch_rotary(x, None, pos, y, None, bwpp.RotaryParams(tokens=0, q_heads=H, dim=d, batch=B))
    assert bool((y == 7.0).all())
    be.dispatch_rotary(x, None, pos, y, None, bwpp.RotaryParams(tokens=T, q_heads=H, dim=d, batch=B))
    want, size = rotary64(x.transpose(1, 2), pos[None].expand(B, T), d, False)
    assert bool(((y.transpose(1, 2).double() - want).abs() <= 6 * 2.0 ** -24 * size).all())


def test_far_strides(be):
    """A batch stride past 2^31 elements (bf16, a 4.3 GB buffer)."""
    d, far = 32, (1 << 31) + 64
    buf = torch.zeros(far + 4 * d, device="cuda", dtype=BF16)
    x = torch.as_strided(buf, (2, 4, 1, d), (far, d, d, 1))
    v = torch.randn(2, 4, 1, d, device="cuda").to(BF16)
    x.copy_(v)
    p = bwpp.RotaryParams(tokens=4, q_heads=1, dim=d, batch=2, dtype=1, q_batch_stride=far, qo_batch_stride=far)
    be.dispatch_rotary(x, None, None, x, None, p)
    want, size = rotary64(v, torch.arange(4, device="cuda")[None].expand(2, 4), d, False)
    assert bool(((x.double() - want).abs() <= 2.0 ** -8 * want.abs() + 5 * 2.0 ** -24 * size).all())

"""Rows longer than the kernels' 32-bit columns can step past are refused before
any launch (found by reading: a column near 2^32 wraps round, and a loop over it
does not end or a chunk passes the row's end)."""
import pytest

import bwpp
from bwpp import _lib

S = bwpp.Status
A, B, C, D, E, F = (0x10000000000 * (i + 1) for i in range(6))


def _call(name, *args):
    lib = _lib.load()
    st = getattr(lib, "bwpp_hip_dispatch_" + name)(None, *args)
    return S(st), lib.bwpp_hip_last_error(None).decode()


@pytest.mark.parametrize("dim,refused", [(2 ** 32 - 1, True), (2 ** 31 + 1, True), (2 ** 31, False), (4096, False)])
@pytest.mark.parametrize("name", ["rotary", "rotary_grad"])
def test_rotary(name, dim, refused):
    st, msg = _call(name, A, None, None, B, None, bwpp.RotaryParams(tokens=1, q_heads=1, dim=dim, rot_dim=64))
    assert (st == S.UNSUPPORTED) == refused and ("rotary" in msg) == refused, (st, msg)
    # nothing to do is no error
    st, msg = _call(name, A, None, None, B, None, bwpp.RotaryParams(tokens=0, q_heads=1, dim=dim, rot_dim=64))
    assert st == S.INVALID_ARG and "rotary" not in msg


@pytest.mark.parametrize("cols,refused", [(2 ** 32 - 1, True), (2 ** 32 - 512, True), (2 ** 31, True), (2 ** 31 - 1, False)])
def test_residual_norm(cols, refused):
    p = bwpp.ResidualNormParams(rows=1, cols=cols, eps=1e-6)
    for name, args in (("residual_norm", (A, B, None, None, None, C, D)),
                       ("residual_norm_grad", (A, B, None, None, None, C, D, E, F, None, None, None))):
        st, msg = _call(name, *args, p)
        assert (st == S.UNSUPPORTED) == refused and (name in msg) == refused, (st, msg)


@pytest.mark.parametrize("cols,refused", [(2 ** 28 - 63, True), (2 ** 28 - 64, False)])
@pytest.mark.parametrize("which", range(3))
def test_residual_norm_sums(cols, refused, which):
    """Their second launch has 16 threads a column: refused before the first."""
    p = bwpp.ResidualNormParams(rows=1, cols=cols, eps=1e-6, post_norm=1)
    grads = [None] * 3
    grads[which] = 7 * 0x10000000000
    st, msg = _call("residual_norm_grad", A, B, None, None, None, C, D, E, F, *grads, p)
    assert (st == S.UNSUPPORTED) == refused and ("residual_norm_grad" in msg) == refused, (st, msg)

"""Calls with no rows take NULL operands (an empty tensor's address): without a
handle, they get as far as that."""
import pytest

import bwpp
from bwpp import _lib

S = bwpp.Status
A = 0x100000000


def _call(name, *args):
    lib = _lib.load()
    st = getattr(lib, "bwpp_hip_dispatch_" + name)(None, *args)
    return S(st), lib.bwpp_hip_last_error(None).decode()


NONE = [None] * 13
ROTARY = lambda n: bwpp.RotaryParams(tokens=n, q_heads=2, k_heads=1, dim=8)
NORM = lambda n: bwpp.ResidualNormParams(rows=n, cols=64, eps=1e-6)
XENT = lambda n: bwpp.LinearXentParams(rows=n, vocab=100, dim=64, trans_w=1)


@pytest.mark.parametrize("name,args,params", [
    ("rotary", NONE[:5], ROTARY), ("rotary_grad", NONE[:5], ROTARY), ("residual_norm", NONE[:7], NORM),
    ("residual_norm_grad", NONE[:12], NORM), ("residual_norm_grad", NONE[:9] + [None, A, A * 2], NORM),
    ("linear_xent", [None, A, None, None, None, A * 2], XENT), ("linear_xent", [None, A, None, None, None, None], XENT),
    ("linear_xent_grad", [None, A, None, None, None, None, A * 2], XENT), ("linear_xent_grad", NONE[:7], XENT)])
def test_no_rows(name, args, params):
    st, msg = _call(name, *args, params(0))
    assert st == S.INVALID_ARG and name not in msg, (st, msg)
    st, msg = _call(name, *args, params(3))
    assert st == S.INVALID_ARG and name in msg, (st, msg)

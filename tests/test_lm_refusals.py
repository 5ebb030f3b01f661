"""Refusals of the operators around the block, without a GPU: arguments are
checked before the handle is touched, so a call without one reports the same
status and text (addresses are never read)."""
import ctypes

import pytest

import bwpp
from bwpp import _lib

S = bwpp.Status
A, B, C, D, E, F = (0x100000000 * (i + 1) for i in range(6))  # far apart
BF16 = int(bwpp.DType.BF16)


def _lib_call(name, *args):
    lib = _lib.load()
    st = getattr(lib, "bwpp_hip_dispatch_" + name)(None, *args)
    return st, lib.bwpp_hip_last_error(None).decode()


def _rot(**kw):
    d = dict(tokens=8, q_heads=4, k_heads=2, dim=64, batch=2)
    d.update(kw)
    return bwpp.RotaryParams(**d)


def test_struct_sizes():
    assert ctypes.sizeof(bwpp.RotaryParams) == 4 * 12 + 8 * 9 + 4 * 8
    assert bwpp.RotaryParams.pos_batch_stride.offset == 112
    assert ctypes.sizeof(bwpp.ResidualNormParams) == 48


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "dtype"), (dict(layout=2), "layout"), (dict(scaling=3), "scaling"),
    (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=66), "rot_dim"), (dict(dim=33), "rot_dim"),
    (dict(base=-1.0), "base"), (dict(base=float("inf")), "base"), (dict(factor=-2.0), "factor"),
    (dict(magnitude=float("nan")), "magnitude"),
    (dict(scaling=2, context=0, low_turns=1, high_turns=4), "by parts"),
    (dict(scaling=2, context=4096, low_turns=4, high_turns=4), "by parts"),
    (dict(ldq=32), "stride"), (dict(ldko=63), "stride"),
    (dict(qo_head_stride=32, ldqo=256, qo_batch_stride=2048), "overlap"),
])
@pytest.mark.parametrize("name", ["rotary", "rotary_grad"])
def test_rotary_bad_arguments(name, kw, text):
    if text == "overlap" and name == "rotary_grad":
        kw = {k.replace("qo", "q"): v for k, v in kw.items()}
    st, msg = _lib_call(name, A, B, None, C, D, _rot(**kw))
    assert st == S.INVALID_ARG and text in msg, (st, msg)


def test_rotary_missing_operands():
    for args in ((None, B, None, C, D), (A, None, None, C, D), (A, B, None, None, D), (A, B, None, C, None)):
        assert _lib_call("rotary", *args, _rot())[0] == S.INVALID_ARG
    assert _lib_call("rotary", A, B, None, C, D, _rot(dim=8192, rot_dim=8192))[0] == S.UNSUPPORTED
    # nothing to refuse: only the handle is missing (no text of an operator)
    st, msg = _lib_call("rotary", A, None, None, C, None, _rot(k_heads=0))
    assert st == S.INVALID_ARG and "rotary" not in msg


def test_rotary_aliases():
    es = 4
    n = 2 * 4 * 8 * 64 * es
    alias = [
        (A, B, A + 64 * es, D, {}),        # shifted by a row
        (A, B, C, A, {}),                  # ko on q
        (A, B, B, D, {}),                  # qo on k
        (A, B, C, C + n - 4, {}),          # ko on qo's last element
        (A, B, A, D, dict(ldqo=64, qo_head_stride=512, qo_batch_stride=4096)),  # same place, other batch stride
    ]
    for q, k, qo, ko, kw in alias:
        st, msg = _lib_call("rotary", q, k, None, qo, ko, _rot(**kw))
        assert st == S.ALIAS, (st, msg, kw)
    assert _lib_call("rotary", A, B, C + n - 4, C, D, _rot())[0] == S.ALIAS  # positions on qo's last element
    # in place, and q, k side by side in one fused row: taken (the handle is missing)
    fused = dict(ldq=512, ldk=512, ldqo=512, ldko=512, q_head_stride=64, k_head_stride=64, qo_head_stride=64,
                 ko_head_stride=64, q_batch_stride=4096, k_batch_stride=4096, qo_batch_stride=4096,
                 ko_batch_stride=4096)
    st, msg = _lib_call("rotary", A, A + 256 * es, None, A, A + 256 * es, _rot(**fused))
    assert st == S.INVALID_ARG and "rotary" not in msg
    st, msg = _lib_call("rotary", A, A + 255 * es, None, A, A + 255 * es, _rot(**fused))
    assert st == S.ALIAS


def _res(**kw):
    d = dict(rows=16, cols=64, eps=1e-6)
    d.update(kw)
    return bwpp.ResidualNormParams(**d)


def test_residual_norm_refusals():
    ok = (A, B, None, None, None, C, D)
    for i in (0, 1, 5):
        args = list(ok)
        args[i] = None
        assert _lib_call("residual_norm", *args, _res())[0] == S.INVALID_ARG
    for kw in (dict(dtype=7), dict(ldx=63), dict(ldo=1), dict(ldy=63), dict(ldg=3), dict(eps=-1.0),
               dict(eps=float("nan"))):
        st, msg = _lib_call("residual_norm", *ok, _res(**kw))
        assert st == S.INVALID_ARG and "residual_norm" in msg, kw
    for args in ((A, B, None, None, None, B, D), (A, B, None, None, None, C, C), (A, B, None, None, None, C, A),
                 (A, B, None, None, None, A + 4, D), (A, B, None, C, None, C, D), (A, B, None, None, D, C, D)):
        assert _lib_call("residual_norm", *args, _res())[0] == S.ALIAS, args
    # without a post-norm its weights are not read
    st, msg = _lib_call("residual_norm", A, B, C, None, None, C, D, _res())
    assert st == S.INVALID_ARG and "residual_norm" not in msg
    # in place
    st, msg = _lib_call("residual_norm", A, B, None, None, None, A, D, _res())
    assert st == S.INVALID_ARG and "residual_norm" not in msg


def test_residual_norm_grad_refusals():
    def call(o=A, r=B, post=None, gate=None, pre=None, dr=C, dy=D, dx=E, dout=F, dpost=None, dgate=None, dpre=None, **kw):
        return _lib_call("residual_norm_grad", o, r, post, gate, pre, dr, dy, dx, dout, dpost, dgate, dpre, _res(**kw))

    G = 7 * 0x100000000
    for kw in (dict(o=None), dict(r=None), dict(dr=None, dy=None), dict(dx=None, dout=None), dict(dpost=G),
               dict(dtype=2), dict(ldo=5)):
        st, msg = call(**kw)
        assert st == S.INVALID_ARG and "residual_norm_grad" in msg, kw
    for kw in (dict(dx=D), dict(dx=C + 4), dict(dout=A), dict(dout=E), dict(dpre=E), dict(dgate=B),
               dict(dgate=E - 4, gate_rows=4), dict(dpost=A, post_norm=1)):
        assert call(**kw)[0] == S.ALIAS, kw
    for kw in (dict(dx=C), dict(dx=None, dout=None, dpre=G), dict(dr=None), dict(dy=None)):
        st, msg = call(**kw)
        assert st == S.INVALID_ARG and "residual_norm_grad" not in msg, kw


def _xent(**kw):
    d = dict(rows=8, vocab=100, dim=64, trans_w=1)
    d.update(kw)
    return bwpp.LinearXentParams(**d)


def test_linear_xent_refusals():
    assert ctypes.sizeof(bwpp.LinearXentParams) == 44
    ok = (A, B, C, D, E, F)
    for i in (0, 1, 2):
        args = list(ok)
        args[i] = None
        assert _lib_call("linear_xent", *args, _xent())[0] == S.INVALID_ARG
    assert _lib_call("linear_xent", A, B, C, None, None, None, _xent())[0] == S.INVALID_ARG
    for kw in (dict(dtype=2), dict(vocab=0), dict(dim=0), dict(ldx=63), dict(ldw=63), dict(trans_w=0, ldw=99),
               dict(scale=float("nan")), dict(scale=float("inf"))):
        for name, args in (("linear_xent", ok), ("linear_xent_grad", (A, B, C, D, None, E, F))):
            st, msg = _lib_call(name, *args, _xent(**kw))
            assert st == S.INVALID_ARG and name in msg, kw
    for kw in (dict(dtype=1, dim=7), dict(dtype=1, trans_w=0, vocab=7), dict(rows=1 << 27), dict(vocab=1 << 31)):
        assert _lib_call("linear_xent", *ok, _xent(**kw))[0] == S.UNSUPPORTED, kw
    for args in ((A, B, C, A, E, F), (A, B, C, D, D, F), (A, B, C, D, E, E + 28), (A, B, C, C + 4, E, F)):
        assert _lib_call("linear_xent", *args, _xent())[0] == S.ALIAS, args
    st, msg = _lib_call("linear_xent", *ok, _xent())
    assert st == S.INVALID_ARG and "linear_xent" not in msg  # only the handle is missing


def test_linear_xent_grad_refusals():
    for args in ((None, B, C, D, None, E, F), (A, None, C, D, None, E, F), (A, B, None, D, None, E, F),
                 (A, B, C, None, None, E, F), (A, B, C, D, None, None, None)):
        assert _lib_call("linear_xent_grad", *args, _xent())[0] == S.INVALID_ARG
    G = 7 * 0x100000000
    for args in ((A, B, C, D, None, A, F), (A, B, C, D, None, E, B + 4), (A, B, C, D, G, G, F), (A, B, C, D, None, E, E),
                 (A, B, C, D, None, E, D)):
        assert _lib_call("linear_xent_grad", *args, _xent())[0] == S.ALIAS, args
    st, msg = _lib_call("linear_xent_grad", A, B, C, D, G, E, F, _xent(lddx=70, lddw=65))
    assert st == S.INVALID_ARG and "linear_xent" not in msg

"""Where rotary's q, k and outputs may lie, without a GPU (a call that passes the
checks is refused for its missing handle): in place in a fused buffer, tokens or
heads first; and against a list of the elements, for random strides, a call that
the checks take never has an output on another operand."""
import itertools
import random

import pytest

import bwpp
from bwpp import _lib

S = bwpp.Status
A = 0x100000000
BF16 = int(bwpp.DType.BF16)


def _call(q, k, qo, ko, p):
    lib = _lib.load()
    st = lib.bwpp_hip_dispatch_rotary(None, q, k, None, qo, ko, p)
    msg = lib.bwpp_hip_last_error(None).decode()
    return "taken" if st == S.INVALID_ARG and "rotary" not in msg else S(st)


def _params(B, T, Hq, Hk, d, **kw):
    return bwpp.RotaryParams(tokens=T, q_heads=Hq, k_heads=Hk, dim=d, batch=B, dtype=BF16, **kw)


def _both(hs, bs, ld):
    """The same strides for q, k and, in place, their outputs."""
    r = {}
    for n in ("q", "k", "qo", "ko"):
        r.update({f"ld{n}": ld, f"{n}_head_stride": hs, f"{n}_batch_stride": bs})
    return r


@pytest.mark.parametrize("B,T,Hq,Hk,d", [(1, 9, 4, 2, 64), (3, 9, 4, 2, 64), (2, 1, 4, 4, 64), (8, 1, 32, 8, 128), (2, 5, 1, 1, 8)])
def test_in_place_in_a_fused_buffer(B, T, Hq, Hk, d):
    H = Hq + 2 * Hk
    heads_first = _both(T * d, H * T * d, d)
    assert _call(A, A + 2 * Hq * T * d, A, A + 2 * Hq * T * d, _params(B, T, Hq, Hk, d, **heads_first)) == "taken"
    tokens_first = _both(d, T * H * d, H * d)
    assert _call(A, A + 2 * Hq * d, A, A + 2 * Hq * d, _params(B, T, Hq, Hk, d, **tokens_first)) == "taken"
    if T == 1:  # the token stride means nothing
        assert _call(A, A + 2 * Hq * d, A, A + 2 * Hq * d, _params(B, T, Hq, Hk, d, **_both(d, H * d, 0))) == "taken"
    # one element too near
    for p, at in ((heads_first, Hq * T * d - 1), (tokens_first, Hq * d - 1)):
        assert _call(A, A + 2 * at, A, A + 2 * at, _params(B, T, Hq, Hk, d, **p)) == S.ALIAS


def test_heads_in_turn():
    """q's and k's heads alternate."""
    B, T, H, d = 2, 5, 3, 16
    p = _both(2 * d, T * 2 * H * d, 2 * H * d)
    assert _call(A, A + 2 * d, A, A + 2 * d, _params(B, T, H, H, d, **p)) == "taken"
    assert _call(A, A + 2 * (d - 1), A, A + 2 * (d - 1), _params(B, T, H, H, d, **p)) == S.ALIAS


def test_taken_calls_share_no_element():
    rng = random.Random(3)
    taken = 0
    for _ in range(4000):
        B, T, Hq, Hk, d = rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 3), rng.choice([2, 4])
        units = [d, 2 * d, 3 * d, 4 * d, 6 * d, 8 * d, 9 * d, 12 * d, 18 * d, 24 * d, 36 * d, d + 1, 5 * d]
        st = [[rng.choice(units) for _ in range(3)] for _ in range(4)]  # ld, head, batch of q, k, qo, ko
        if rng.random() < 0.7:
            st[1] = list(st[0])
        same = rng.random() < 0.6
        if same:
            st[2], st[3] = list(st[0]), list(st[1])
        at = [0, rng.randint(0, 40 * d), 0, 0]
        at[2], at[3] = (at[0], at[1]) if same else (rng.randint(0, 60 * d), rng.randint(0, 60 * d))
        kw = {}
        for n, (ld, hs, bs) in zip(("q", "k", "qo", "ko"), st):
            kw.update({f"ld{n}": ld, f"{n}_head_stride": hs, f"{n}_batch_stride": bs})
        r = _call(*(A + 2 * a for a in at), _params(B, T, Hq, Hk, d, **kw))
        if r != "taken":
            continue
        taken += 1

        def elements(i):
            ld, hs, bs = st[i]
            return [at[i] + b * bs + t * ld + h * hs + e for b, t, h, e in
                    itertools.product(range(B), range(T), range((Hq, Hk)[i % 2]), range(d))]

        q, k, qo, ko = (elements(i) for i in range(4))
        assert len(set(qo)) == len(qo) and len(set(ko)) == len(ko)
        assert not set(qo) & set(ko) and not set(qo) & set(k) and not set(ko) & set(q)
        assert q == qo or not set(q) & set(qo)
        assert k == ko or not set(k) & set(ko)
    assert taken > 200, taken

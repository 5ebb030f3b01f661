"""Refusals of the paged cache's operators and of the rules on logits, without a
GPU: arguments are checked before the handle is touched, so a call without one
reports the same status and text (addresses are never read)."""
import ctypes

import pytest

import bwpp
from bwpp import _lib

S = bwpp.Status
A, B, C, D, E, F, G, H, I, J, K = (0x10000000000 * (i + 1) for i in range(11))  # far apart


def _call(name, *args):
    lib = _lib.load()
    st = getattr(lib, "bwpp_hip_dispatch_" + name)(None, *args)
    return st, lib.bwpp_hip_last_error(None).decode()


def _cache(**kw):
    d = dict(pages=10, page_tokens=16, heads=2, dim=64, batch=3, max_pages=4, tokens=8, q_heads=4)
    d.update(kw)
    return bwpp.CacheParams(**d)


NAMES = ("cache_append", "cache_attention", "cache_keep")


def _op(name, cache={}, args={}, **kw):
    """One call with far operands; `args` replaces some by position."""
    if name == "cache_append":  # q k v positions table starts held qo k_cache v_cache
        a, p = [A, B, C, None, D, E, F, G, H, I], bwpp.CacheAppendParams(cache=_cache(**cache), **kw)
    elif name == "cache_attention":  # q k_cache v_cache table starts held mask o lse
        a, p = [A, B, C, D, E, F, None, G, H], bwpp.CacheAttentionParams(cache=_cache(**cache), **kw)
    else:  # k_cache v_cache table held kept counts
        kw.setdefault("max_kept", 4)
        a, p = [A, B, C, D, E, F], bwpp.CacheKeepParams(cache=_cache(**cache), **kw)
    for i, v in args.items():
        a[i] = v
    return _call(name, *a, p)


def _taken(name, *args, **kw):
    st, msg = _op(name, *args, **kw)
    return st == S.INVALID_ARG and name not in msg  # only the handle is missing


def test_struct_sizes():
    assert ctypes.sizeof(bwpp.CacheParams) == 64
    assert ctypes.sizeof(bwpp.CacheAppendParams) == 64 + 16 + 32 + 40
    assert ctypes.sizeof(bwpp.CacheAttentionParams) == 64 + 8 + 16 + 8
    assert ctypes.sizeof(bwpp.CacheKeepParams) == 72
    assert ctypes.sizeof(bwpp.LogitRulesParams) == 36


@pytest.mark.parametrize("name", NAMES)
def test_cache_shape(name):
    assert _taken(name)
    for kw, text in ((dict(dtype=2), "dtype"), (dict(page_tokens=0), "power"), (dict(page_tokens=24), "power"),
                     (dict(heads=0), "heads"), (dict(dim=0), "dim"), (dict(ld_table=3), "ld_table")):
        st, msg = _op(name, kw)
        assert st == S.INVALID_ARG and name in msg and text in msg, (kw, msg)
    for kw in (dict(batch=(1 << 24) + 1), dict(heads=(1 << 16) + 4, q_heads=(1 << 17) + 8), dict(dim=4097),
               dict(page_stride=1 << 58)):
        assert _op(name, kw)[0] == S.UNSUPPORTED, kw
    if name != "cache_keep":
        assert _op(name, dict(q_heads=3))[0] == S.INVALID_ARG
        assert _op(name, dict(tokens=1 << 29))[0] == S.UNSUPPORTED
    # nothing to do: operands may be missing
    assert _taken(name, dict(batch=0), {i: None for i in range(6)})
    if name != "cache_keep":
        assert _taken(name, dict(tokens=0), {i: None for i in range(6)})


@pytest.mark.parametrize("name,optional", [("cache_append", (3,)), ("cache_attention", (6, 8)), ("cache_keep", ())])
def test_missing_operands(name, optional):
    for i in range({"cache_append": 10, "cache_attention": 9, "cache_keep": 6}[name]):
        if i in optional:
            assert _taken(name, args={i: None})
        else:
            st, msg = _op(name, args={i: None})
            assert st == S.INVALID_ARG and name in msg, i


def test_append_refusals():
    name = "cache_append"
    for kw, text in ((dict(rot_dim=63), "rot_dim"), (dict(rot_dim=66), "rot_dim"), (dict(layout=2), "layout"),
                     (dict(scaling=3), "scaling"), (dict(base=-1.0), "base"), (dict(ldq=63), "stride"),
                     (dict(ldk=32), "stride"), (dict(ldqo=100), "overlap"), (dict(qo_head_stride=32), "overlap")):
        st, msg = _op(name, {}, **kw)
        assert st == S.INVALID_ARG and text in msg, (kw, msg)
    assert _op(name, dict(dim=33, token_stride=40))[0] == S.INVALID_ARG  # an odd row cannot be turned whole
    assert _taken(name, dict(dim=33), no_rotation=1)
    assert _taken(name, dict(q_heads=0), {0: None, 7: None})
    for kw in (dict(token_stride=63), dict(head_stride=64), dict(page_stride=64)):
        st, msg = _op(name, kw)
        assert st == S.INVALID_ARG and "pool" in msg, kw
    n = 8 * 4 * 64 * 4  # bytes of q
    pool = 10 * 2 * 16 * 64 * 4
    for args in ({7: A + 4}, {7: B}, {7: C}, {7: H}, {8: I}, {9: H + pool - 4}, {8: A}, {9: B}, {8: C + 4}, {7: E - n + 4},
                 {8: D - 4}, {9: F - pool + 4}, {3: G + 4}, {4: H + 8}):
        assert _op(name, args=args)[0] == S.ALIAS, args
    assert _taken(name, args={7: A})  # in place
    # keys and values side by side in one buffer: in a page's rows, or page by page
    assert _taken(name, dict(token_stride=128, head_stride=16 * 128), {8: H, 9: H + 64 * 4})
    assert _taken(name, dict(page_stride=2 * 2 * 16 * 64), {8: H, 9: H + 2 * 16 * 64 * 4})
    # no pool: nothing is appended, q is turned
    assert _taken(name, dict(pages=0), {8: None, 9: None, 4: None})


def test_attention_refusals():
    name = "cache_attention"
    for kw in (dict(scale=float("nan")), dict(scale=float("inf")), dict(ldq=63), dict(ldo=100), dict(o_head_stride=8)):
        assert _op(name, {}, **kw)[0] == S.INVALID_ARG, kw
    assert _op(name, dict(q_heads=0))[0] == S.INVALID_ARG
    st, msg = _op(name, args={6: I})
    assert st == S.INVALID_ARG and "mask" in msg
    assert _taken(name, args={6: I}, mask_words=1)
    assert _op(name, dict(dim=257))[0] == S.UNSUPPORTED
    assert _op(name, dict(tokens=1 << 28, max_pages=1 << 26))[0] == S.UNSUPPORTED
    # sequences of which each could, by its starts, count all rows
    assert _op(name, dict(tokens=1 << 24, max_pages=1 << 12, batch=1 << 24))[0] == S.UNSUPPORTED
    assert _taken(name, dict(tokens=1 << 24, max_pages=1 << 12, batch=1 << 10))
    for args in ({7: A}, {7: B + 4}, {7: C}, {8: A}, {8: B}, {8: G}, {7: D}, {8: E}, {7: F - 4}):
        assert _op(name, args=args)[0] == S.ALIAS, args
    assert _op(name, args={6: G + 4}, mask_words=2)[0] == S.ALIAS


def test_keep_refusals():
    name = "cache_keep"
    assert _op(name, ld_kept=3)[0] == S.INVALID_ARG
    assert _taken(name, max_kept=0, args={i: None for i in range(6)})
    assert _op(name, dict(page_stride=64))[0] == S.INVALID_ARG
    for args in ({1: A}, {1: A + 4}, {2: A + 64}, {3: B}, {4: B + 8}, {5: A}):
        assert _op(name, args=args)[0] == S.ALIAS, args


def _rules(args={}, **kw):
    d = dict(rows=4, vocab=1000, history=50)
    d.update(kw)
    a = [A, B, C, D, E, F, G, H, I, J]  # x history starts prompt repetition presence frequency bias mask y
    for i, v in args.items():
        a[i] = v
    return _call("logit_rules", *a, bwpp.LogitRulesParams(**d))


def test_logit_rules_refusals():
    ok = lambda *a, **kw: _rules(*a, **kw)[0] == S.INVALID_ARG and "logit_rules" not in _rules(*a, **kw)[1]
    assert ok()
    for kw in (dict(dtype_x=2), dict(dtype_y=5), dict(ldx=999), dict(ldy=1), dict(ld_bias=999), dict(ld_mask=31)):
        st, msg = _rules(**kw)
        assert st == S.INVALID_ARG and "logit_rules" in msg, kw
    for kw in (dict(vocab=1 << 31), dict(history=1 << 31)):
        assert _rules(**kw)[0] == S.UNSUPPORTED, kw
    for i in (0, 1, 2, 9):
        st, msg = _rules({i: None})
        assert st == S.INVALID_ARG and "NULL" in msg, i
    none = {i: None for i in (1, 2, 3, 4, 5, 6, 7, 8)}
    assert ok(none) and ok({3: None, 4: None, 5: None, 7: None, 8: None}) and ok({1: None, 2: None}, history=0)
    assert ok({9: A}) and ok({9: A}, dtype_x=1, dtype_y=1) and ok(rows=0) and ok(vocab=0)
    assert ok({9: A + 4000}, ldx=2000, ldy=2000)  # other columns of one buffer
    for args, kw in (({9: A}, dict(dtype_y=1)), ({9: A}, dict(ldy=1001)), ({9: A + 4}, {}), ({9: B}, {}), ({9: C}, {}),
                     ({9: D}, {}), ({9: E}, {}), ({9: F}, {}), ({9: G}, {}), ({9: H + 8}, {}), ({9: I}, {}),
                     ({9: H + 4 * 3500}, dict(ld_bias=1000))):
        assert _rules(args, **kw)[0] == S.ALIAS, (args, kw)


def test_python_refuses_other_integers():
    import torch

    be = object.__new__(bwpp.HipBackend)
    be._h, be.lib = None, _lib.load()
    p = bwpp.CacheKeepParams(cache=_cache(), max_kept=4)
    for name, bad in (("table", torch.zeros(3, 4)), ("held", torch.zeros(3, dtype=torch.int64)),
                      ("kept", torch.zeros(3, 8, dtype=torch.int32)[:, ::2]), ("counts", torch.zeros(6, dtype=torch.int32)[::2])):
        args = dict(table=C, held=D, kept=E, counts=F)
        args[name] = bad
        with pytest.raises(ValueError, match=name):
            be.dispatch_cache_keep(A, B, args["table"], args["held"], args["kept"], args["counts"], p)

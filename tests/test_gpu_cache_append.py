"""Appending to a paged cache, against a 64-bit form (bounds: cache64.append64;
keys outside the rotated part, values and everything that is not appended keep
their bits)."""
import pytest
import torch

import bwpp
from cache64 import BF16, F32, Cache, append64, i32
from lm64 import strided, untouched

pytestmark = pytest.mark.gpu
PARTS = dict(scaling=2, factor=16.0, context=8192, low_turns=1.0, high_turns=32.0, magnitude=1.25)
LINEAR = dict(scaling=1, factor=4.0, base=500.0)


def _check(be, c, Hq, rot=0, inter=False, scal={}, positions=False, fused=False, in_place=False, rotate=True, pad=0):
    T, d, Hk = c.tokens, c.d, c.Hk
    n = rot or d
    if fused:  # q, k, v side by side in a token's row
        row = (Hq + 2 * Hk) * d + pad
        qkv, _ = strided((T, Hq + 2 * Hk, d), (row, d, 1), c.dtype, c.normal(T, Hq + 2 * Hk, d))
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
    else:
        q, k, v = (strided((T, h, d), (h * d + pad, d, 1), c.dtype, c.normal(T, h, d))[0] for h in (Hq, Hk, Hk))
    pos = torch.randint(-1000, 1 << 20, (T,), device="cuda", dtype=torch.int32, generator=c.g) if positions else None
    p64 = pos
    if pos is None:
        p64 = torch.zeros(T, dtype=torch.int64, device="cuda")
        for s, (h, m) in enumerate(zip(c.held, c.new)):
            p64[c.first[s]:c.first[s] + m] = torch.arange(h, h + m, device="cuda")
    qo64, tq, kc, tkc, vc, live = append64(c, q, k, v, p64, n, inter, scal, rotate)
    q0 = q.clone()
    qo, qbuf = (q, None) if in_place else strided((T, Hq, d), (Hq * d + 3 * pad, d, 1), c.dtype)
    p = bwpp.CacheAppendParams(cache=c.params(Hq), ldq=q.stride(0), ldk=k.stride(0), ldv=v.stride(0),
                               ldqo=qo.stride(0), no_rotation=int(not rotate), rot_dim=rot, layout=int(inter), **scal)
    be.dispatch_cache_append(q if Hq else None, k, v, pos, c.table, c.starts, c.held_t, qo if Hq else None, c.k, c.v, p)
    torch.cuda.synchronize()
    assert be.last_kernel.startswith("bwpp_cache_append_" + ("bf16" if c.dtype == BF16 else "f32"))
    if Hq:
        assert bool(((qo.double() - qo64).abs() <= tq)[live].all())
        assert bool((qo[~live] == (q0[~live] if in_place else 5.0)).all())  # rows of no sequence
        if qbuf is not None:
            assert untouched(qo, qbuf)
    assert bool(((c.k.double() - kc).abs() <= tkc).all())
    assert bool((c.v.double() == vc).all())
    assert untouched(c.k, c.kbuf) and untouched(c.v, c.vbuf)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("held,new,Hq,Hk,d,rot,page,pad", [
    ([0], [1], 1, 1, 2, 0, 1, 0), ([5, 0, 40], [1, 1, 1], 8, 2, 128, 0, 16, 0), ([15, 16, 17], [3, 0, 33], 6, 3, 80, 40, 16, 1),
    ([0, 100], [130, 7], 4, 4, 64, 0, 32, 8), ([3, 2, 1, 0], [1, 2, 3, 4], 2, 1, 24, 12, 2, 3), ([1000], [300], 2, 2, 256, 128, 128, 0),
    ([7] * 300, [1] * 300, 4, 1, 32, 0, 8, 0), ([0, 0], [70, 70], 1, 1, 4096, 0, 64, 0)])
def test_append(be, dtype, by_token, held, new, Hq, Hk, d, rot, page, pad):
    for inter in (False, True):
        c = Cache(held, new, Hk, d, page, dtype, by_token, pad=pad, before=2, after=3, ld_table=0, seed=d + page)
        _check(be, c, Hq, rot, inter, PARTS if inter else {}, positions=inter, pad=pad)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_operands(be, dtype):
    mk = lambda **kw: Cache([9, 0, 30], [4, 1, 50], 2, 96, 16, dtype, **kw)
    _check(be, mk(), 4, fused=True, scal=LINEAR)
    _check(be, mk(pad=1, by_token=True), 4, fused=True, pad=1, scal=LINEAR)  # rows at any address
    _check(be, mk(), 4, fused=True, in_place=True)
    _check(be, mk(), 4, 32, in_place=True, inter=True)
    _check(be, mk(), 0)                      # no queries
    _check(be, mk(), 4, rotate=False)        # k as it is, q copied
    _check(be, mk(), 4, rotate=False, in_place=True)
    _check(be, mk(ld_table=11), 4)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_slots_that_do_not_exist(be, dtype):
    """A table too short for the sequence, pages outside the pool, lengths below
    zero and starts past the operands: nothing leaves the pools."""
    c = Cache([30, 14], [10, 10], 2, 64, 16, dtype, max_pages=2)
    _check(be, c, 2)
    _check(be, Cache([40, 14], [10, 10], 2, 64, 16, dtype, max_pages=2), 2)  # longer than the table: q goes on
    c = Cache([30, 14, 0], [10, 10, 5], 2, 64, 16, dtype)
    c.table[0, 2], c.table[1, 1], c.table[2, 0] = -1, c.pages, 2 ** 31 - 1
    _check(be, c, 2)
    c = Cache([0, 0], [6, 6], 1, 64, 16, dtype)
    c.held_t = i32([-5, -(2 ** 31)])
    _check(be, c, 2)
    c = Cache([4, 4], [6, 6], 1, 64, 16, dtype)
    c.starts = i32([0, 6, 2 ** 31 - 1])
    _check(be, c, 2)
    c = Cache([4, 4], [6, 0], 1, 64, 16, dtype, after=4)
    c.starts = i32([-7, 6, 3])  # the second ends before it begins
    _check(be, c, 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_short_sequences(be, dtype):
    """More sequences than starts fit in LDS, empty ones among them."""
    new = [(i * 7) % 3 for i in range(1500)]
    c = Cache([i % 11 for i in range(1500)], new, 1, 16, 4, dtype, before=1, after=2)
    _check(be, c, 2)


def test_values_keep_their_bits(be):
    c = Cache([3], [5], 1, 64, 16, BF16)
    raw = torch.randint(0, 1 << 16, (5, 1, 64), device="cuda", generator=c.g).to(torch.int32).to(torch.int16)
    v, k = raw.view(BF16), c.normal(5, 1, 64)
    p = bwpp.CacheAppendParams(cache=c.params(0))
    be.dispatch_cache_append(None, k, v, None, c.table, c.starts, c.held_t, None, c.k, c.v, p)
    for i in range(5):
        at = c.slot(0, 3 + i)
        assert bool((c.v[at].view(torch.int16) == raw[i]).all())


def test_page_past_32_bits(be):
    """A pool of more than 2^32 elements: 17 GB of keys in bf16, the page at its end."""
    pages, page, d = (1 << 32) // (256 * 128) + 3, 256, 128
    k_cache = torch.empty(pages, 1, page, d, dtype=BF16, device="cuda")
    v_cache = torch.empty(8, 1, page, d, dtype=BF16, device="cuda")
    k, v = torch.randn(2, 4, 1, d, device="cuda").to(BF16)
    last = pages - 1
    k_cache[last].fill_(5.0)
    k_cache[last - (1 << 32) // (256 * 128)].fill_(5.0)
    v_cache = torch.empty_like(k_cache)
    p = bwpp.CacheAppendParams(cache=bwpp.CacheParams(pages=pages, page_tokens=page, heads=1, dim=d, batch=1, max_pages=1,
                                                      tokens=4, dtype=1), no_rotation=1)
    be.dispatch_cache_append(None, k, v, None, i32([[last]]), i32([0, 4]), i32([252]), None, k_cache, v_cache, p)
    assert bool((k_cache[last, 0, 252:] == k[:, 0]).all()) and bool((k_cache[last, 0, :252] == 5.0).all())
    assert bool((v_cache[last, 0, 252:] == v[:, 0]).all())
    assert bool((k_cache[last - (1 << 32) // (256 * 128)] == 5.0).all())


def test_no_pool(be):
    """No pages: nothing is appended, q is turned as with them."""
    c = Cache([3], [4], 2, 64, 16, F32)
    q, k, v = c.normal(4, 4, 64), c.normal(4, 2, 64), c.normal(4, 2, 64)
    a, b = torch.empty_like(q), torch.empty_like(q)
    be.dispatch_cache_append(q, k, v, None, c.table, c.starts, c.held_t, a, c.k, c.v, bwpp.CacheAppendParams(cache=c.params(4)))
    be.dispatch_cache_append(q, k, v, None, None, c.starts, c.held_t, b, None, None,
                             bwpp.CacheAppendParams(cache=c.params(4, pages=0)))
    assert bool((a == b).all())


def test_pools_side_by_side(be):
    """Keys and values in one buffer: of a page one behind the other, and of a token."""
    for shape, at in (((5, 2, 2, 16, 64), lambda t, i: t[:, i]), ((5, 2, 16, 2, 64), lambda t, i: t[:, :, :, i])):
        buf = torch.full(shape, 5.0, device="cuda")
        kc, vc = at(buf, 0), at(buf, 1)  # [page, head, token, d]
        k, v = torch.randn(2, 20, 2, 64, device="cuda")
        cp = bwpp.CacheParams(pages=5, page_tokens=16, heads=2, dim=64, batch=1, max_pages=2, tokens=20,
                              page_stride=kc.stride(0), head_stride=kc.stride(1), token_stride=kc.stride(2))
        be.dispatch_cache_append(None, k, v, None, i32([[4, 1]]), i32([0, 20]), i32([6]), None, kc, vc,
                                 bwpp.CacheAppendParams(cache=cp, no_rotation=1))
        for c, x in ((kc, k), (vc, v)):
            assert bool((c[4, :, 6:].transpose(0, 1) == x[:10]).all()) and bool((c[1, :, :10].transpose(0, 1) == x[10:]).all())
            assert bool((c[4, :, :6] == 5.0).all()) and bool((c[[0, 2, 3]] == 5.0).all()) and bool((c[1, :, 10:] == 5.0).all())

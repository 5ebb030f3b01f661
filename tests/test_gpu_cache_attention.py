"""Attention over a paged cache against a 64-bit form (bounds: the docstring of
cache64.attention64): steps, trees and pieces of prompts, ragged and padded
batches, pages that end inside a tile, tokens that see nothing, slots that do
not exist, infinities and NaN where nobody looks."""
import math

import pytest
import torch

import bwpp
from cache64 import BF16, F32, Cache, attention64, bits, i32, tree
from lm64 import strided, untouched

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", [F32, BF16])


def _run(be, c, q, sees=None, scale=None, lse=True, mask=None, pad=0):
    """(o, lse) of one call; guards around them are checked."""
    T, Hq, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    o, obuf = strided((T, Hq, d), (Hq * d + pad, d, 1), c.dtype)
    l, lbuf = strided((T, Hq), (Hq, 1), F32)
    if sees is not None and mask is None:
        n = max(c.new + [1])
        rows = torch.ones(T, n, dtype=torch.bool)  # rows of no sequence: anything
        for s, m in enumerate(c.new):
            rows[c.first[s]:c.first[s] + m] = False
            rows[c.first[s]:c.first[s] + m, :m] = sees[s].cpu()
        mask = bits(rows)
    p = bwpp.CacheAttentionParams(cache=c.params(Hq), ldq=q.stride(0), ldo=o.stride(0), scale=scale,
                                  mask_words=0 if mask is None else mask.shape[1])
    be.dispatch_cache_attention(q, c.k, c.v, c.table, c.starts, c.held_t, mask, o, l if lse else None, p)
    torch.cuda.synchronize()
    assert untouched(o, obuf) and untouched(l, lbuf)
    return o, l


def _check(be, c, Hq, sees=None, scale=None, std=2.5, q=None, pad=0, lse=True):
    T, d = c.tokens, c.d
    if q is None:
        q, _ = strided((T, Hq, d), (Hq * d + pad, d, 1), c.dtype, c.normal(T, Hq, d, std=std))
    o, l = _run(be, c, q, sees, scale, lse, pad=pad)
    want, wl, to, tl = attention64(c, q, d ** -0.5 if scale is None else scale, sees)
    live = torch.zeros(T, dtype=torch.bool, device="cuda")
    live[c.first[0]:c.first[-1]] = True
    err = (o.double() - want).abs()
    fine = (err <= to) | (o.double() == want) | (torch.isnan(want) & torch.isnan(o))
    assert bool(fine[live].all()), (float((err / to)[live].nan_to_num(0).max()), c.held, c.new)
    assert bool((o[~live] == 5.0).all())
    if lse:
        inf = torch.isinf(wl) & (l.double() == wl)
        fine = ((l.double() - wl).abs() <= tl) | inf | (torch.isnan(wl) & torch.isnan(l))
        assert bool(fine[live].all()), float(((l.double() - wl).abs() / tl)[live].nan_to_num(0, 0, 0).max())
        assert bool((l[~live] == 5.0).all())
    else:
        assert bool((l == 5.0).all())
    return o


@DTYPES
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("held,Hq,Hk,page", [
    ([0], 1, 1, 1), ([1, 0, 15, 16, 17], 4, 1, 16), ([31, 32, 33, 63, 64, 65], 8, 2, 32), ([127, 500, 3], 6, 6, 64),
    ([1023, 0, 2049], 8, 1, 256), ([70, 300], 40, 1, 8), ([9000], 2, 1, 128), ([200] * 70, 2, 2, 2)])
def test_one_token(be, dtype, d, held, Hq, Hk, page):
    _check(be, Cache(held, [1] * len(held), Hk, d, page, dtype, by_token=page == 16, seed=page), Hq)


@DTYPES
@pytest.mark.parametrize("d", [1, 3, 16, 48, 80, 96, 100, 112, 160, 192, 255, 256])
def test_head_dims(be, dtype, d):
    _check(be, Cache([40, 0, 333], [1, 1, 1], 2, d, 16, dtype), 8)
    _check(be, Cache([40, 0, 333], [5, 40, 9], 2, d, 16, dtype, before=1, after=1), 8)


@DTYPES
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("held,new,Hq,Hk,page", [
    ([0], [2], 1, 1, 16), ([0, 100, 5], [13, 7, 64], 4, 4, 16), ([30, 1], [33, 31], 8, 2, 32), ([500], [64], 8, 1, 64),
    ([3000, 10], [17, 1], 6, 2, 16), ([0, 0], [100, 129], 4, 2, 1)])
def test_trees(be, dtype, d, held, new, Hq, Hk, page):
    c = Cache(held, new, Hk, d, page, dtype, before=1, after=2, seed=len(new))
    _check(be, c, Hq, [tree(n, c.g) for n in new])


@DTYPES
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("held,new,Hq,Hk,page", [
    ([0], [200], 2, 1, 64), ([0, 50, 0], [65, 0, 130], 4, 2, 16), ([129, 1], [300, 1], 4, 1, 128), ([7], [511], 2, 2, 8)])
def test_prompts(be, dtype, d, held, new, Hq, Hk, page):
    _check(be, Cache(held, new, Hk, d, page, dtype, by_token=True, pad=8, before=3), Hq)


@DTYPES
@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("new", [[1, 1], [9, 40]])
def test_strides(be, dtype, pad, new):
    """Rows at any address: pools, queries and results."""
    for by_token in (False, True):
        _check(be, Cache([77, 130], new, 2, 64, 32, dtype, by_token, pad=pad, ld_table=30), 4, pad=pad)


@DTYPES
@pytest.mark.parametrize("scale", [1.0, 0.5, -0.25, 1e-30])
@pytest.mark.parametrize("new", [1, 30])
def test_scales(be, dtype, scale, new):
    _check(be, Cache([100, 0], [new, new], 2, 64, 16, dtype), 4, scale=scale, std=0.5)
    _check(be, Cache([100, 0], [new, new], 2, 100, 16, dtype), 4, scale=scale, std=0.5, lse=False)


@DTYPES
@pytest.mark.parametrize("d", [64, 80])
@pytest.mark.parametrize("n", [3, 40])
def test_tokens_that_see_nothing(be, dtype, d, n):
    c = Cache([0, 20, 0], [n, n, n], 2, d, 16, dtype)
    sees = [torch.zeros(n, n, dtype=torch.bool) for _ in range(3)]
    sees[2][n // 2:] = tree(n, c.g)[n // 2:]
    o = _check(be, c, 4, sees)
    assert bool((o[:n] == 0).all()) and bool((o[2 * n:2 * n + n // 2] == 0).all())


@DTYPES
@pytest.mark.parametrize("d", [64, 80])
def test_masks_narrower_and_wider_than_the_tree(be, dtype, d):
    c = Cache([10], [40], 1, d, 16, dtype)
    q = c.normal(40, 2, d)
    full = torch.ones(40, 40, dtype=torch.bool)
    narrow = full.clone()
    narrow[:, 32:] = False  # bits past the row: not seen
    one = torch.full((40, 1), -1, dtype=torch.int32, device="cuda")
    wide = torch.full((40, 5), -1, dtype=torch.int32, device="cuda")
    for mask, sees in ((one, narrow), (wide, full)):
        o, _ = _run(be, c, q, mask=mask)
        want, _, to, _ = attention64(c, q, d ** -0.5, [sees])
        assert bool(((o.double() - want).abs() <= to).all())


@DTYPES
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("new", [[1, 1, 1], [6, 9, 40]])
def test_slots_that_do_not_exist(be, dtype, d, new):
    """Pages outside the pool (first, middle, last), and a table too short."""
    c = Cache([100, 300, 64], new, 2, d, 16, dtype)
    c.table[0, 0] = -1
    c.table[1, 5:9] = torch.tensor([c.pages, 2 ** 31 - 1, -2 ** 31, -1], dtype=torch.int32)
    c.table[2, :4] = -1  # only the new tokens are left
    _check(be, c, 4)
    c = Cache([100, 300, 64], new, 2, d, 16, dtype, max_pages=6)
    c.held = [96, 96, 64]  # what the table holds, for the plain form
    c.new = new
    got = _run(be, c, q := c.normal(c.tokens, 4, d))[0]
    for s, n in enumerate(new):  # nothing past the table is seen, the held tokens all are
        k, v, _ = c.gather(s, c.held[s] + (min(n, 32) if s == 2 else 0))
        for i in (0, n - 1):
            L = min(64 + i + 1, 96) if s == 2 else 96
            t = c.first[s] + i
            z = q[t, 3].double() @ k[:L, 1].double().T * d ** -0.5
            want = torch.softmax(z, dim=0) @ v[:L, 1].double()
            assert float((got[t, 3].double() - want).abs().max()) <= 0.02


@DTYPES
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("n", [5, 40])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_nobody_sees_stays_out(be, dtype, d, n, bad):
    """Infinities and NaN in keys and values: past the last slot, in pages of
    other sequences, and in drafts that some tokens do not see."""
    c = Cache([37, 20], [n, n], 2, d, 16, dtype)
    seen = torch.zeros(c.pages, c.page, dtype=torch.bool, device="cuda")
    for s in range(2):
        for p in range(c.held[s] + n):
            seen[c.slot(s, p)] = True
    c.k[~seen], c.v[~seen] = bad, bad
    sees = [tree(n, c.g) for _ in range(2)]
    at = c.slot(0, 37 + 2)  # a draft that its descendants alone see
    c.v[at][0, 1] = bad
    o = _check(be, c, 4, sees)
    hit = sees[0][:, 2].cuda()
    assert bool(torch.isfinite(o[:n][~hit]).all())
    assert not bool(torch.isfinite(o[:n][hit][:, 0, 1]).any())
    q = c.normal(c.tokens, 4, d)
    c.k[at] = bad  # a key: whoever sees it may get anything, nobody else
    c.v[at] = 1.0
    o, l = _run(be, c, q, sees)
    c.k[at] = 0.0
    want, wl, to, tl = attention64(c, q, d ** -0.5, sees)
    assert bool(((o.double() - want).abs() <= to)[:n][~hit].all()) and bool(((l.double() - wl).abs() <= tl)[:n][~hit].all())


@DTYPES
@pytest.mark.parametrize("d", [64, 80])
def test_large_and_equal_scores(be, dtype, d):
    c = Cache([500, 2], [1, 30], 1, d, 16, dtype)
    c.k.mul_(40.0)
    _check(be, c, 8, std=30.0)
    c.k.fill_(1.0)
    _check(be, c, 8)
    c.k.fill_(-3e4)  # scores far below zero
    _check(be, c, 8, std=1.0, scale=1.0)


@DTYPES
def test_ragged_and_padded(be, dtype):
    """Idle sequences, rows before the first and behind the last, one long
    sequence among short ones, and more sequences than threads."""
    _check(be, Cache([0, 5000, 3, 0, 64], [0, 1, 1, 0, 1], 2, 128, 64, dtype, before=3, after=5), 8)
    held = [(i * 37) % 90 for i in range(700)]
    _check(be, Cache(held, [i % 3 for i in range(700)], 1, 64, 16, dtype, after=1), 2)
    _check(be, Cache([40], [0], 1, 64, 16, dtype, after=4), 2)


@DTYPES
@pytest.mark.parametrize("d", [64, 80])
def test_starts_and_lengths_are_cut(be, dtype, d):
    c = Cache([30, 7], [4, 4], 1, d, 16, dtype)
    q = c.normal(8, 2, d)
    a, _ = _run(be, c, q)
    c.starts = i32([-3, 4, 2 ** 31 - 1])
    assert bool((_run(be, c, q)[0] == a).all())
    c.held_t = i32([30, -2 ** 31])  # below zero: none
    b, _ = _run(be, c, q)
    assert bool((b[:4] == a[:4]).all())
    c.held_t = i32([2 ** 31 - 1, 7])  # past the table: as many as it has
    b, _ = _run(be, c, q)
    assert bool((b[4:] == a[4:]).all()) and bool(torch.isfinite(b.float()).all())


@DTYPES
@pytest.mark.parametrize("d", [64, 80, 100])
def test_no_pool(be, dtype, d):
    """No pages, or a table without columns: nothing is seen."""
    c = Cache([0, 0], [1, 40], 2, d, 16, dtype)
    q = c.normal(41, 4, d)
    for kw in (dict(pages=0), dict(max_pages=0)):
        o, l = torch.full_like(q, 5.0), torch.full((41, 4), 5.0, device="cuda")
        be.dispatch_cache_attention(q, None, None, None, c.starts, c.held_t, None, o, l,
                                    bwpp.CacheAttentionParams(cache=c.params(4, **kw)))
        assert bool((o == 0).all()) and bool((l == -math.inf).all())


@DTYPES
@pytest.mark.parametrize("d", [64, 72, 128])
@pytest.mark.parametrize("Hq,n", [(96, 1), (33, 1), (64, 7), (100, 3), (300, 1)])
def test_many_query_heads_a_key_head(be, dtype, d, Hq, n):
    """More rows of one token than a tile has, and tokens that end inside one."""
    _check(be, Cache([70, 1300, 0], [n, n, n], 1, d, 16, dtype), Hq)
    c = Cache([70, 600], [n, n], 1, d, 16, dtype)
    _check(be, c, Hq, [tree(n, c.g) for _ in range(2)])


@DTYPES
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("page", [1, 2, 16])
def test_more_pages_than_are_kept_in_lds(be, dtype, d, page):
    _check(be, Cache([1100 * page, 2500, 70], [1, 1, 1], 1, d, page, dtype, seed=page), 2)
    _check(be, Cache([1100 * page, 2500], [70, 3], 1, d, page, dtype, seed=page), 2)


@DTYPES
@pytest.mark.parametrize("d", [64, 80])
def test_same_bits_every_time(be, dtype, d):
    c = Cache([4000, 100, 9], [1, 1, 1], 2, d, 16, dtype)
    q = c.normal(3, 8, d)
    a, la = _run(be, c, q)
    for _ in range(3):
        b, lb = _run(be, c, q)
        assert bool((a == b).all()) and bool((la == lb).all())


def test_page_past_32_bits(be):
    """Keys and values past 2^32 elements of their pool."""
    pages, page, d = (1 << 32) // (256 * 128) + 3, 256, 128
    k_cache = torch.empty(pages, 1, page, d, dtype=BF16, device="cuda")
    v_cache = torch.empty_like(k_cache)
    use = [pages - 1, 1, pages - 2]
    for i in use:
        k_cache[i].copy_(torch.randn(1, page, d, device="cuda"))
        v_cache[i].copy_(torch.randn(1, page, d, device="cuda"))
        j = i - (1 << 32) // (256 * 128)
        if j >= 0 and j not in use:
            k_cache[j].fill_(math.nan), v_cache[j].fill_(math.nan)
    for n in (1, 40):
        q = torch.randn(n, 4, d, device="cuda").to(BF16)
        o = torch.empty_like(q)
        p = bwpp.CacheAttentionParams(cache=bwpp.CacheParams(pages=pages, page_tokens=page, heads=1, dim=d, batch=1,
                                                             max_pages=3, tokens=n, q_heads=4, dtype=1), scale=d ** -0.5)
        be.dispatch_cache_attention(q, k_cache, v_cache, i32([use]), i32([0, n]), i32([700]), None, o, None, p)
        k, v = (torch.cat([x[i, 0] for i in use])[:700 + n].double() for x in (k_cache, v_cache))
        z = torch.einsum("thd,ld->thl", q.double(), k) * d ** -0.5
        z = z.masked_fill(torch.arange(700 + n, device="cuda")[None, None] > 700 + torch.arange(n, device="cuda")[:, None, None], -math.inf)
        want = torch.softmax(z, dim=2) @ v
        assert float((o.double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 1e-4


@pytest.mark.parametrize("d,page", [(64, 64), (128, 16), (128, 64), (256, 64)])
@pytest.mark.parametrize("n", [1, 16, 48])
def test_more_keys_than_the_caches_hold(be, d, page, n):
    """Sequences that share their pages: 2500 tokens, 8 key heads, often enough
    that keys and values count for more than 400 MB; each has the same result."""
    Hk, Hq, N = 8, 32, 400_000_000 // (2500 * 8 * d * 4) + 1
    c = Cache([2500], [n], Hk, d, page, BF16)
    q = c.normal(n, Hq, d, std=2.5)
    want, wl, to, tl = attention64(c, q, d ** -0.5)
    o, l = torch.empty(N, n, Hq, d, dtype=BF16, device="cuda"), torch.empty(N, n, Hq, device="cuda")
    p = bwpp.CacheAttentionParams(cache=c.params(Hq, batch=N, tokens=N * n), scale=d ** -0.5)
    be.dispatch_cache_attention(q.expand(N, n, Hq, d).contiguous(), c.k, c.v, c.table.expand(N, -1).contiguous(),
                                i32([s * n for s in range(N + 1)]), i32([2500] * N), None, o, l, p)
    torch.cuda.synchronize()
    assert bool(((o.double() - want).abs() <= to).all()) and bool(((l.double() - wl).abs() <= tl).all())


@DTYPES
@pytest.mark.parametrize("d,n", [(64, 2), (80, 30), (128, 60)])
def test_starts_that_descend(be, dtype, d, n):
    """Sequences whose rows overlap: rows of one sequence alone have its results,
    shared ones are written by either, the others stay as they were."""
    c = Cache([900, 70, 1300], [n, n, n], 2, d, 16, dtype)
    q = c.normal(3 * n, 8, d)
    c.starts = i32([0, n, n // 2, n // 2 + n])  # the second has none, the third overlaps the first
    o, l = _run(be, c, q)
    half = n // 2
    one = Cache([900, 70, 1300], [n, n, n], 2, d, 16, dtype)
    want, wl, to, tl = attention64(one, q, d ** -0.5)
    assert bool(((o[:half].double() - want[:half]).abs() <= to[:half]).all())
    assert bool(((l[:half].double() - wl[:half]).abs() <= tl[:half]).all())
    assert bool(torch.isfinite(o[:n + half].double()).all())
    assert bool((o[n + half:] == 5.0).all()) and bool((l[n + half:] == 5.0).all())

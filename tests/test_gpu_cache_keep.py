"""Moving the accepted drafts of a paged cache together: exact copies, read
before they are overwritten."""
import pytest
import torch

import bwpp
from cache64 import BF16, F32, Cache, i32
from lm64 import untouched

pytestmark = pytest.mark.gpu


def _check(be, c, kept, counts, ld=0):
    want_k, want_v = c.k.clone(), c.v.clone()
    for s, row in enumerate(kept):
        for i, j in enumerate(row[:max(0, counts[s])]):
            a, b = c.slot(s, c.held[s] + j) if j >= 0 else None, c.slot(s, c.held[s] + i)
            if a is not None and b is not None:
                want_k[b], want_v[b] = c.k[a], c.v[a]
    width = max(len(r) for r in kept)
    t = torch.full((len(kept), ld or width), -9, dtype=torch.int32, device="cuda")
    for s, row in enumerate(kept):
        t[s, :len(row)] = i32(row)
    p = bwpp.CacheKeepParams(cache=c.params(0), max_kept=width, ld_kept=ld)
    be.dispatch_cache_keep(c.k, c.v, c.table, c.held_t, t, i32(counts), p)
    torch.cuda.synchronize()
    same = lambda a, b: bool((a.contiguous().view(torch.uint8) == b.contiguous().view(torch.uint8)).all())
    assert same(c.k, want_k) and same(c.v, want_v)
    assert untouched(c.k, c.kbuf) and untouched(c.v, c.vbuf)
    return be.last_kernel


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("Hk,d,page,pad", [(2, 64, 16, 0), (1, 80, 4, 8), (3, 7, 2, 1), (8, 128, 64, 0), (12, 256, 32, 0),
                                           (1, 2, 1, 0)])
def test_keep(be, dtype, by_token, Hk, d, page, pad):
    c = Cache([14, 0, 100], [40, 40, 3], Hk, d, page, dtype, by_token, pad=pad)
    _check(be, c, [[0, 1, 4, 9, 39], [0, 3, 3, 20, 21], [0, 2, 2, 2, 2]], [5, 4, 2])
    c = Cache([14, 5], [80, 80], Hk, d, page, dtype, by_token, pad=pad)
    _check(be, c, [list(range(0, 80, 2)), list(range(40, 80))], [40, 40], ld=45)  # several rounds


def test_widths(be):
    assert _check(be, Cache([3], [9], 2, 64, 8, BF16), [[0, 5]], [2]) == "bwpp_cache_keep_16"
    assert _check(be, Cache([3], [9], 2, 63, 8, F32), [[0, 5]], [2]) == "bwpp_cache_keep_4"
    assert _check(be, Cache([3], [9], 2, 64, 8, BF16, pad=1), [[0, 5]], [2]) == "bwpp_cache_keep_2"


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_moves_nothing(be, dtype):
    c = Cache([14, 0, 3, 3], [20, 20, 20, 20], 2, 64, 16, dtype)
    c.table[1, 1] = -1
    c.table[2, 0] = c.pages
    _check(be, c, [[0, 7], [0, 17], [4, 15], [-1, 2 ** 31 - 1]], [-3, 2, 2, 2])
    c.held_t = i32([2 ** 31 - 1, -7, 0, 0])
    c.held = [2 ** 31 - 1, 0, 0, 0]
    _check(be, c, [[1, 7], [1, 3], [1, 18], [0, 0]], [2, 2, 2, 0])


def test_any_order_within_a_round(be):
    """As if all were read before any is written."""
    c = Cache([10], [16], 2, 64, 16, F32)
    _check(be, c, [[15, 14, 13, 3, 2, 1, 0, 0]], [8])

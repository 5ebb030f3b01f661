"""Attention over a paged cache in bf16: what the probabilities' own precision gives.
The matrix-core kernels of head dims 64, 80, 96, 160, 192 and 256 take them as two bf16
terms, as attention over whole rows does for every dim but 128; the kernels of other
dims and of rows at any address keep them in fp32.

Bounds: those of cache64.attention64 for fp32 operands (scores, exponentials, sums), for
two terms 2^-16 and 2^-23 of the weighted sum's terms (a probability's upper 16 bits and
its rest below 2^-7 of it, raised by 2^-23 and rounded to 8 bits), and the result's own
rounding, half a step of what was computed."""
import copy

import pytest

from cache64 import BF16, F32, Cache, attention64, tree
from lm64 import HALF_STEP, strided
from test_gpu_cache_attention import _run

pytestmark = pytest.mark.gpu


def _check(be, c, Hq, terms, sees=None, pad=0, std=2.5):
    T, d = c.tokens, c.d
    q, _ = strided((T, Hq, d), (Hq * d + pad, d, 1), c.dtype, c.normal(T, Hq, d, std=std))
    o, l = _run(be, c, q, sees, pad=pad)
    kernel = be.last_kernel if "join" not in be.last_kernel else be.recent_kernel(1)
    want, wl, to, tl = attention64(c, q.float(), d ** -0.5, sees)
    whole = copy.copy(c)
    whole.v = c.v.abs()
    size = attention64(whole, q.float(), d ** -0.5, sees)[0]
    to = (to + (2.0 ** -16 + 2.0 ** -23 if terms == 2 else 0.0) * size) * (1 + HALF_STEP[c.dtype])
    if c.dtype == BF16:
        to = to + HALF_STEP[BF16] * want.abs()
    live = slice(c.first[0], c.first[-1])
    err = (o.double() - want).abs()
    assert bool((err <= to)[live].all()), (kernel, float((err / to)[live].max()))
    assert bool(((l.double() - wl).abs() <= tl)[live].all())
    return kernel


@pytest.mark.parametrize("d", [64, 80, 96, 160, 192, 256])
@pytest.mark.parametrize("held,new", [([0, 3], [7, 5]), ([40, 300], [30, 40]), ([0, 5], [100, 90]), ([2500], [70])])
def test_probabilities_in_two_terms(be, d, held, new):
    for sees in (False, True):
        c = Cache(held, new, 2, d, 16, BF16, seed=d)
        kernel = _check(be, c, 4, 2, [tree(n, c.g) for n in new] if sees else None)
        rows = -(-sum(new) // len(new)) * 2
        assert ("few" in kernel) == (rows <= 32)


@pytest.mark.parametrize("d,pad", [(48, 0), (112, 0), (255, 0), (64, 1), (96, 3)])
@pytest.mark.parametrize("held,new", [([40, 300], [3, 9]), ([0, 5], [40, 90]), ([700], [70])])
def test_probabilities_in_fp32(be, d, pad, held, new):
    c = Cache(held, new, 2, d, 16, BF16, pad=pad, seed=d)
    kernel = _check(be, c, 4, 0, [tree(n, c.g) for n in new], pad=pad)
    assert "attend_bf16" in kernel


@pytest.mark.parametrize("dtype,d,terms", [(F32, 64, 0), (F32, 128, 0), (BF16, 48, 0), (BF16, 80, 2), (BF16, 160, 2)])
@pytest.mark.parametrize("new", [[1, 1, 1], [6, 9, 40]])
def test_a_table_too_short(be, dtype, d, terms, new):
    """Held tokens and new ones past the last column."""
    for held in ([100, 300, 64], [96, 0, 95]):
        _check(be, Cache(held, new, 2, d, 16, dtype, max_pages=6), 4, terms)

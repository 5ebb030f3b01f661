"""Every kernel of the paged cache and of the rules on logits is what some call
takes, and which one: the variant of a call follows from its sizes, types and
alignment."""
import pytest
import torch

import bwpp
from cache64 import BF16, F32, Cache, i32
from test_cache_codeobj import kernel_names

pytestmark = pytest.mark.gpu


def _append(be, dtype, rot, inter):
    c = Cache([0], [2], 1, 64, 16, dtype)
    k, v = c.normal(2, 1, 64), c.normal(2, 1, 64)
    p = bwpp.CacheAppendParams(cache=c.params(0), rot_dim=rot, layout=int(inter))
    be.dispatch_cache_append(None, k, v, None, c.table, c.starts, c.held_t, None, c.k, c.v, p)
    return [be.last_kernel]


def _attend(be, dtype, d, n, held=0, pad=0):
    c = Cache([held], [n], 1, d, 16, dtype, pad=pad)
    q = c.normal(n, 1, d)
    o = torch.empty_like(q)
    p = bwpp.CacheAttentionParams(cache=c.params(1))
    be.dispatch_cache_attention(q, c.k, c.v, c.table, c.starts, c.held_t, None, o, None, p)
    return [be.last_kernel] if held == 0 else [be.recent_kernel(1), be.last_kernel]


def test_every_kernel_is_reached(be):
    seen = set()
    for dtype, chunks in ((BF16, (64, 8, 2)), (F32, (64, 2))):
        for rot in chunks:
            for inter in (False, True):
                seen.update(_append(be, dtype, rot, inter))
    for d in (64, 80, 96, 128, 160, 192, 256):
        for n, kernel in ((32, "few"), (128, "r128"), (129, "r256" if d <= 128 else "r128")):
            k = _attend(be, BF16, d, n)
            assert k == [f"bwpp_cache_attend_{kernel}_d{d}"]
            seen.update(k)
    for dtype, name, pad in ((F32, "f32", 0), (BF16, "bf16", 1)):
        for d in range(32, 257, 32):
            for n, kernel in ((64, f"d{-(-d // 64) * 64}"), (65, f"rows_d{d}")):
                k = _attend(be, dtype, d, n, pad=pad)
                assert k == [f"bwpp_cache_attend_{name}_{kernel}"]
                seen.update(k)
    for dtype, d, n, join in ((F32, 64, 1, "f32_16"), (F32, 64, 65, "f32_128"), (BF16, 63, 1, "bf16_16"),
                              (BF16, 64, 1, "bf16_32"), (BF16, 64, 128, "bf16_128"), (BF16, 64, 129, "bf16_256")):
        k = _attend(be, dtype, d, n, held=2000)
        assert k[1] == f"bwpp_cache_join_{join}"
        seen.update(k)
    for dtype, pad, name in ((F32, 0, "16"), (F32, 1, "4"), (BF16, 1, "2")):
        c = Cache([0], [4], 1, 64, 16, dtype, pad=pad)
        p = bwpp.CacheKeepParams(cache=c.params(0), max_kept=2)
        be.dispatch_cache_keep(c.k, c.v, c.table, c.held_t, i32([[0, 2]]), i32([2]), p)
        assert be.last_kernel == f"bwpp_cache_keep_{name}"
        seen.add(be.last_kernel)
    for tx in (F32, BF16):
        for ty in (F32, BF16):
            x, y = torch.ones(1, 8, device="cuda", dtype=tx), torch.empty(1, 8, device="cuda", dtype=ty)
            be.dispatch_logit_rules(x, None, None, None, None, None, None, None, None, y,
                                    bwpp.LogitRulesParams(rows=1, vocab=8, dtype_x=int(tx == BF16), dtype_y=int(ty == BF16)))
            seen.add(be.last_kernel)
    assert seen == set(kernel_names()), set(kernel_names()) ^ seen


def test_one_launch_for_tables_of_few_columns(be):
    """A table that bounds all lengths by few keys: no item is shared, no join."""
    for dtype, keys in ((BF16, 512), (F32, 256)):
        for columns, launches in ((keys // 16, 1), (keys // 16 + 1, 2)):
            c = Cache([40], [1], 1, 64, 16, dtype, max_pages=columns)
            q = c.normal(1, 1, 64)
            p = bwpp.CacheAttentionParams(cache=c.params(1))
            be.dispatch_logit_rules(torch.ones(1, 8, device="cuda"), None, None, None, None, None, None, None, None,
                                    torch.empty(1, 8, device="cuda"), bwpp.LogitRulesParams(rows=1, vocab=8))
            be.dispatch_cache_attention(q, c.k, c.v, c.table, c.starts, c.held_t, None, torch.empty_like(q), None, p)
            assert be.recent_kernel(launches) == "bwpp_logit_rules_f32"

"""Attention over tables that are full: as many slots as sequences may have without a
workspace, sequences that fill the table or end past it, lengths that name any slot.
Against the 64-bit form, whose slots past the table do not exist either."""
import pytest
import torch

from cache64 import BF16, F32, Cache, i32
from test_gpu_cache_attention import _check

pytestmark = pytest.mark.gpu

# dtype, dim, query heads, key heads, new tokens of a call (its rows decide the tile), slots that need no workspace
KERNELS = pytest.mark.parametrize("dtype,d,Hq,Hk,n,slots", [
    (F32, 64, 4, 2, 1, 256), (F32, 128, 8, 2, 16, 256), (F32, 64, 4, 2, 48, 256), (F32, 160, 2, 1, 300, 256),
    (BF16, 48, 4, 2, 1, 256), (BF16, 112, 4, 1, 40, 256),
    (BF16, 64, 4, 2, 1, 512), (BF16, 128, 32, 8, 1, 512), (BF16, 128, 8, 2, 8, 512), (BF16, 256, 4, 2, 2, 512),
    (BF16, 128, 4, 1, 24, 1024), (BF16, 64, 4, 1, 48, 1024), (BF16, 128, 8, 2, 300, 1024), (BF16, 192, 2, 1, 300, 1024)])


def _no_join(be):
    assert "join" not in be.last_kernel


@KERNELS
def test_sequences_at_the_end_of_their_table(be, dtype, d, Hq, Hk, n, slots):
    for held in ([max(0, slots - n)], [slots], [slots - n // 2 - 1], [slots + 7, slots, 3]):
        c = Cache(held, [n] * len(held), Hk, d, 64, dtype, max_pages=slots // 64, before=1, after=1)
        _check(be, c, Hq)
        _no_join(be)


@KERNELS
def test_more_new_tokens_than_the_table_has_slots(be, dtype, d, Hq, Hk, n, slots):
    if n == 1:
        n = 2  # as many as make whole tiles of the kernel for few rows
    table = 64 if n < 40 else 128
    count = table + 40 if n >= 40 else n
    c = Cache([table - 1, 0], [count, count], Hk, d, 64, dtype, max_pages=table // 64)
    _check(be, c, Hq)
    _no_join(be)


@KERNELS
def test_lengths_that_name_any_slot(be, dtype, d, Hq, Hk, n, slots):
    c = Cache([slots, 5, slots], [n] * 3, Hk, d, 64, dtype, max_pages=slots // 64)
    c.held_t = i32([2 ** 31 - 1, 5, slots + 12345])
    _check(be, c, Hq)
    _no_join(be)


@KERNELS
def test_the_slots_behind_one_more_column(be, dtype, d, Hq, Hk, n, slots):
    """One column more: there is a workspace, and parts may be joined."""
    for held in ([slots + 64], [max(0, slots + 64 - n)], [slots + 20, 3]):
        c = Cache(held, [n] * len(held), Hk, d, 64, dtype, max_pages=slots // 64 + 1)
        _check(be, c, Hq)


@pytest.mark.parametrize("dtype,d,slots", [(F32, 128, 256), (BF16, 128, 512)])
def test_a_recorded_step_that_reaches_the_end(be, dtype, d, slots):
    """Replays whose sequence grows up to the table's last slot and past it."""
    import bwpp
    c = Cache([slots - 3], [1], 8, d, 64, dtype, max_pages=slots // 64)
    q = c.normal(1, 32, d)
    o = torch.empty_like(q)
    p = bwpp.CacheAttentionParams(cache=c.params(32), scale=d ** -0.5)
    call = lambda: be.dispatch_cache_attention(q, c.k, c.v, c.table, c.starts, c.held_t, None, o, None, p)
    call()
    torch.cuda.synchronize()
    graph, old = torch.cuda.CUDAGraph(), torch.cuda.current_stream()
    side = torch.cuda.Stream()
    side.wait_stream(old)
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            be.set_stream(side)
            call()
    be.set_stream(old)
    torch.cuda.synchronize()
    for held in range(slots - 3, slots + 3):
        c.held_t.fill_(held)
        o.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone()
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, o)
        c.held = [held]
        _check(be, c, 32, q=q)

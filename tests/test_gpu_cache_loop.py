"""The paged cache's operators together, as a serving loop runs them: prompts,
single tokens, trees of drafts that are verified and kept, rules and the greedy
choice; eager, in a graph whose replays follow the lengths, on several streams."""
import pytest
import torch

import bwpp
from cache64 import BF16, F32, Cache, bits, i32, tree
from lm64 import HALF_STEP, rotary64

pytestmark = pytest.mark.gpu
D, HK, HQ, PAGE = 64, 2, 8, 16


class Loop:
    """A batch of sequences over one pool, and what each holds in 64 bits."""

    def __init__(self, be, seqs, dtype, room=160, seed=0):
        self.be, self.dtype, self.n = be, dtype, seqs
        self.c = Cache([room] * seqs, [0] * seqs, HK, D, PAGE, dtype, seed=seed)
        self.held = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.keys = [torch.zeros(0, HK, D, dtype=torch.float64, device="cuda") for _ in range(seqs)]
        self.values = [torch.zeros(0, HK, D, dtype=torch.float64, device="cuda") for _ in range(seqs)]

    def params(self, tokens):
        return self.c.params(HQ, tokens=tokens)

    def step(self, new, sees=None, depth=None):
        """Appends `new` tokens a sequence and attends with them; checks the
        result; the 64-bit side holds them behind the sequence's own."""
        c, T = self.c, sum(new)
        qkv = c.normal(T, HQ + 2 * HK, D)
        q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
        starts = i32([sum(new[:i]) for i in range(self.n + 1)])
        held = self.held.tolist()
        pos = torch.cat([h + (depth[s].cuda() if depth else torch.arange(m, device="cuda")) for s, (h, m) in enumerate(zip(held, new))])
        qo = torch.empty(T, HQ, D, dtype=self.dtype, device="cuda")
        pa = bwpp.CacheAppendParams(cache=self.params(T), ldq=qkv.stride(0), ldk=qkv.stride(0), ldv=qkv.stride(0))
        self.be.dispatch_cache_append(q, k, v, pos.int() if depth else None, c.table, starts, self.held, qo, c.k, c.v, pa)
        mask = None
        if sees is not None:
            n = max(new)
            mask = bits(torch.cat([torch.nn.functional.pad(s, (0, n - s.shape[1])) for s in sees]))
        o = torch.empty_like(qo)
        pt = bwpp.CacheAttentionParams(cache=self.params(T), scale=D ** -0.5, mask_words=0 if mask is None else mask.shape[1])
        self.be.dispatch_cache_attention(qo, c.k, c.v, c.table, starts, self.held, mask, o, None, pt)
        first = 0
        for s, m in enumerate(new):
            r = slice(first, first + m)
            first += m
            if m == 0:
                continue
            kr = rotary64(k[r][None], pos[r][None], D, False)[0][0]
            qr = rotary64(q[r][None], pos[r][None], D, False)[0][0]
            self.keys[s], self.values[s] = torch.cat([self.keys[s], kr]), torch.cat([self.values[s], v[r].double()])
            ok = torch.ones(m, held[s] + m, dtype=torch.bool, device="cuda")
            ok[:, held[s]:] = (torch.ones(m, m, dtype=torch.bool).tril() if sees is None else sees[s]).cuda()
            z = torch.stack([qr[:, h] @ self.keys[s][:, h // (HQ // HK)].T for h in range(HQ)], dim=1) * D ** -0.5
            p = torch.softmax(z.masked_fill(~ok[:, None, :], -torch.inf), dim=2)
            want = torch.stack([p[:, h] @ self.values[s][:, h // (HQ // HK)] for h in range(HQ)], dim=1)
            # q and k are rounded after their turn: scores are off by 2 half steps of S = scale sum |q k|
            # and a little, weights relatively by that, the result twice that (weights and their sum); P may
            # be rounded, the result is (half a step each)
            S = torch.stack([qr[:, h].abs() @ self.keys[s][:, h // (HQ // HK)].abs().T for h in range(HQ)]).max() * D ** -0.5
            half = HALF_STEP[self.dtype]
            err = float((o[r].double() - want).abs().max() / self.values[s].abs().max())
            assert err <= 4.1 * half * float(S) + 2 * half + 1e-5, (err, s, new)
        self.held += i32(new)

    def keep(self, new, kept):
        """After `step(new)`: of each sequence's last `new` tokens only `kept` stay."""
        self.held -= i32(new)
        width = max(len(r) for r in kept)
        t = i32([r + [0] * (width - len(r)) for r in kept])
        p = bwpp.CacheKeepParams(cache=self.params(0), max_kept=width)
        self.be.dispatch_cache_keep(self.c.k, self.c.v, self.c.table, self.held, t, i32([len(r) for r in kept]), p)
        for s, r in enumerate(kept):
            h = int(self.held[s])
            at = torch.tensor(list(range(h)) + [h + j for j in r], device="cuda")
            self.keys[s], self.values[s] = self.keys[s][at], self.values[s][at]
        self.held += i32([len(r) for r in kept])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_serving_loop(be, dtype):
    lp = Loop(be, 3, dtype)
    lp.step([70, 3, 40])          # prompts
    for _ in range(3):
        lp.step([1, 1, 1])
    for i in range(3):            # trees of drafts, then their accepted paths
        new = [13, 13, 13]
        sees = [tree(13, lp.c.g) for _ in range(3)]
        depth = [s.sum(dim=1) - 1 for s in sees]
        lp.step(new, sees, depth)
        paths = [torch.nonzero(s[12 - i]).flatten().tolist() for s in sees]
        lp.keep(new, paths)
        lp.step([1, 1, 1])
    lp.step([1, 0, 20])           # an idle sequence, another piece of a prompt


def test_rules_and_greedy_choice(be):
    """Logits through the rules to reduce_max: the forbidden and the repeated
    token are not chosen again."""
    V = 5000
    x = torch.zeros(2, V, device="cuda", dtype=BF16)
    x[:, 17], x[:, 40], x[0, 99], x[1, 7] = 9.0, 8.0, 7.0, 6.0
    allowed = torch.ones(2, V, dtype=torch.bool)
    allowed[:, 40] = False
    y, top, at = torch.empty(2, V, device="cuda"), torch.empty(2, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    be.dispatch_logit_rules(x, i32([17, 17, 17, 17]), i32([0, 2, 4]), None, None, torch.full((2,), 5.0, device="cuda"), None,
                            None, bits(allowed), y, bwpp.LogitRulesParams(rows=2, vocab=V, dtype_x=1, history=4, ld_mask=-(-V // 32)))
    be.dispatch_reduce_max(y, top, at, bwpp.ReduceParams(2, V, V, 1))
    assert at.tolist() == [99, 7] and top.tolist() == [7.0, 6.0]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("room", [200, 2000])
def test_recorded_step_follows_the_lengths(dtype, room):
    """A recorded step (append, attention, rules) replayed while the lengths grow
    in device memory: the same bits as eager calls, replay after replay, with
    other work of the handle between."""
    be = bwpp.HipBackend(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        be.set_stream(side)
        seqs = 5
        c = Cache([room] * seqs, [40] * seqs, HK, D, PAGE, dtype)
        held = i32([3, 0, room, 77, room // 2])
        starts = i32(range(seqs + 1))
        qkv = c.normal(seqs, HQ + 2 * HK, D)
        qo, o = (torch.empty(seqs, HQ, D, dtype=dtype, device="cuda") for _ in range(2))
        lse = torch.empty(seqs, HQ, device="cuda")
        x, y = c.normal(seqs, 999), torch.empty(seqs, 999, device="cuda")
        rep, history, hs = torch.full((seqs,), 1.3, device="cuda"), i32(range(50)), i32([0, 10, 10, 30, 45, 50])
        cp = c.params(HQ, tokens=seqs)
        pa = bwpp.CacheAppendParams(cache=cp, ldq=qkv.stride(0), ldk=qkv.stride(0), ldv=qkv.stride(0))
        pt = bwpp.CacheAttentionParams(cache=cp, scale=D ** -0.5)
        pr = bwpp.LogitRulesParams(rows=seqs, vocab=999, dtype_x=int(dtype == BF16), history=50)

        def step():
            be.dispatch_cache_append(qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:], None, c.table, starts, held, qo, c.k, c.v, pa)
            be.dispatch_cache_attention(qo, c.k, c.v, c.table, starts, held, None, o, lse, pt)
            be.dispatch_logit_rules(x, history, hs, None, rep, None, None, None, None, y, pr)

        step()  # once before: the workspace
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for i in range(6):
            qkv.copy_(c.normal(seqs, HQ + 2 * HK, D))
            x.copy_(c.normal(seqs, 999))
            graph.replay()
            got = [t.clone() for t in (qo, o, lse, y, c.k, c.v)]
            for t in (qo, o, lse, y):
                t.fill_(7.0)
            step()
            for a, b in zip(got, (qo, o, lse, y, c.k, c.v)):
                assert bool((a == b).all()), i
            held += 1 + i % 3
            side.synchronize()
    be.close()


def test_recording_without_workspace_is_refused():
    be = bwpp.HipBackend(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        be.set_stream(side)
        c = Cache([2000], [1], HK, D, PAGE, BF16)
        q = c.normal(1, HQ, D)
        o = torch.empty_like(q)
        pt = bwpp.CacheAttentionParams(cache=c.params(HQ))
        call = lambda: be.dispatch_cache_attention(q, c.k, c.v, c.table, c.starts, c.held_t, None, o, None, pt)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(bwpp.BwppError, match="run the call once before") as e:
                call()
        assert e.value.status == bwpp.Status.OUT_OF_MEMORY
        call()
        side.synchronize()
        assert bool(torch.isfinite(o.float()).all())
    be.close()


def test_two_handles_on_two_streams():
    """Calls at once on handles of their own, over one pool."""
    c = Cache([3000, 500], [1, 1], HK, D, PAGE, BF16)
    qs = [c.normal(2, HQ, D) for _ in range(8)]
    pt = bwpp.CacheAttentionParams(cache=c.params(HQ), scale=D ** -0.5)
    backends = [bwpp.HipBackend(0) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = []
    backends[0].set_stream(torch.cuda.current_stream())
    for q in qs:
        o = torch.empty_like(q)
        backends[0].dispatch_cache_attention(q, c.k, c.v, c.table, c.starts, c.held_t, None, o, None, pt)
        want.append(o)
    torch.cuda.synchronize()
    got = [torch.empty_like(q) for q in qs]
    for b, s in zip(backends, streams):
        b.set_stream(s)
    for i, q in enumerate(qs):
        backends[i % 2].dispatch_cache_attention(q, c.k, c.v, c.table, c.starts, c.held_t, None, got[i], None, pt)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert bool((a == b).all())
    for b in backends:
        b.close()

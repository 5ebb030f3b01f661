"""A decoding step as a launch plan: against 64 bits, and recorded, its replays
following the lengths in device memory.  fp32 bar: 1e-4 relative max-norm, the
other plans'."""
import pytest
import torch

import bwpp
from bwpp import plan
from cache64 import bits, i32
from cacheplan import DECODE
from conftest import rel_max_err
from lm64 import rotary64

pytestmark = pytest.mark.gpu
S, D, HQ, HK, E, V = 3, 64, 4, 2, 16, 100


def _inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    allowed = torch.rand(S, V, generator=g, device="cuda") < 0.8
    return dict(x=n(S, D), wqkv=n(D, 128) / 8, wv=n(HQ * E, V) / 8, kc=n(12, HK, 8, E), vc=n(12, HK, 8, E),
                table=i32([[3, 7, 0, 1], [2, 9, 5, 11], [4, 6, 8, 10]]), starts=i32([0, 1, 2, 3]), held=i32([5, 0, 23]),
                history=i32([i * 7 % V for i in range(20)]), hstarts=i32([0, 4, 4, 20]), rep=n(S).abs() + 1.0,
                mask=bits(allowed)), allowed


def _step64(t, allowed):
    """y, ctx of a step; the caches as they are before it."""
    d = {k: v.double() if v.is_floating_point() else v for k, v in t.items()}
    qkv = d["x"] @ d["wqkv"]
    ctx = torch.zeros(S, HQ * E, dtype=torch.float64, device="cuda")
    for s in range(S):
        held = int(t["held"][s])
        turn = lambda v: rotary64(v.reshape(1, 1, -1, E), t["held"][s:s + 1, None], 8, False, scaling=1, factor=2.0)[0][0, 0]
        q, k, v = turn(qkv[s, :64]), turn(qkv[s, 64:96]), qkv[s, 96:].reshape(HK, E)
        at = [(int(t["table"][s, p // 8]), p % 8) for p in range(held)]
        for h in range(HQ):
            ks = torch.stack([d["kc"][a, h // 2, b] for a, b in at] + [k[h // 2]])
            vs = torch.stack([d["vc"][a, h // 2, b] for a, b in at] + [v[h // 2]])
            ctx[s, h * E:(h + 1) * E] = torch.softmax(ks @ q[h] * E ** -0.5, dim=0) @ vs
    y = ctx @ d["wv"]
    hs = t["hstarts"].tolist()
    for s in range(S):
        for v in set(t["history"][hs[s]:hs[s + 1]].tolist()):
            y[s, v] = y[s, v] / d["rep"][s] if y[s, v] > 0 else y[s, v] * d["rep"][s]
    return ctx, y.masked_fill(~allowed, -torch.inf)


def _plan(be, t):
    p = plan.Plan(be, DECODE)
    p.allocate()
    for k, v in t.items():
        p.bind(k, v)
    return p


def test_step(be):
    t, allowed = _inputs(1)
    p = _plan(be, t)
    for _ in range(4):  # the cache grows by what each step appended
        ctx, y = _step64(t, allowed)
        p.run()
        assert rel_max_err(p.host("ctx", (S, HQ * E)), ctx.cpu().numpy()) <= 1e-4
        got = p.host("y", (S, V))
        assert ((got == -float("inf")) == (~allowed).cpu().numpy()).all()
        assert rel_max_err(got, y.cpu().numpy()) <= 1e-4
        t["held"] += 1
        torch.cuda.synchronize()
    p.close()


def test_step_recorded():
    b = bwpp.HipBackend(0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    b.set_stream(side)
    t, _ = _inputs(2)
    torch.cuda.synchronize()
    p = _plan(b, t)
    shapes = dict(ctx=(S, HQ * E), lse=(S, HQ), y=(S, V))
    p.capture()
    for i in range(5):
        t["x"].copy_(_inputs(30 + i)[0]["x"])
        torch.cuda.synchronize()
        p.run()
        eager = {n: p.host(n, s) for n, s in shapes.items()}
        p.replay()
        for n, s in shapes.items():
            assert (p.host(n, s) == eager[n]).all(), (i, n)
        t["held"] += 1
        torch.cuda.synchronize()
    p.close()
    b.close()

"""The operators around the block run together: a training step of one block
with its loss as a launch plan, eager and recorded, and a scoring pass in bf16
through the entry points.  fp32 bar: 1e-4 relative max-norm, the other plans'."""
import pytest
import torch

import bwpp
from bwpp import plan
from conftest import rel_max_err
from lm64 import resnorm64, rotary64, xent64
from lmplan import GRADS, TRAIN, inputs, step64

pytestmark = pytest.mark.gpu
TOL = 1e-4


def _plan(be, t, **dims):
    text = TRAIN
    for k, v in dims.items():
        text = text.replace(f"dim {k} {dict(B=2, T=24, D=64, HEADS=4, F=96, V=500)[k]}\n", f"dim {k} {v}\n")
    p = plan.Plan(be, text)
    p.allocate()
    for k, v in t.items():
        p.bind(k, v)
    return p


@pytest.mark.parametrize("B,T,D,HEADS,F,V", [(2, 24, 64, 4, 96, 500), (1, 1, 32, 2, 32, 40), (3, 130, 192, 3, 256, 2001)])
def test_training_step(be, B, T, D, HEADS, F, V):
    t = inputs(B, T, D, F, V, 5)
    t["targets"][0] = 3
    want_loss, want_y2, want = step64(t, B, T, HEADS)
    p = _plan(be, t, B=B, T=T, D=D, HEADS=HEADS, F=F, V=V)
    p.run()
    assert rel_max_err(p.host("loss", (B * T,)), want_loss.cpu().numpy()) <= TOL
    assert rel_max_err(p.host("y2", (B * T, D)), want_y2.cpu().numpy()) <= TOL
    for name, src in GRADS.items():
        assert rel_max_err(p.host(name, tuple(t[src].shape)), want[name].cpu().numpy()) <= TOL, name
    p.close()


def test_training_step_recorded():
    """Replays between eager runs, with new inputs: the same bits each time."""
    b = bwpp.HipBackend(0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    b.set_stream(side)
    t = inputs(2, 24, 64, 96, 500, 7)
    torch.cuda.synchronize()
    p = _plan(b, t)
    names = ["loss", "y2"] + list(GRADS)
    shape = lambda n: (48,) if n == "loss" else (48, 64) if n == "y2" else tuple(t[GRADS[n]].shape)
    p.capture()
    for i in range(4):
        t["x"].copy_(inputs(2, 24, 64, 96, 500, 20 + i)["x"])
        torch.cuda.synchronize()
        p.run()
        eager = {n: p.host(n, shape(n)) for n in names}
        p.replay()
        for n in names:
            assert (p.host(n, shape(n)) == eager[n]).all(), (i, n)
    p.close()
    b.close()


def test_scoring_in_bf16(be):
    """Norm, projection, rotary positions in the projection's place, attention,
    join and loss on bf16 rows.  Each step against 64 bits of its own bf16
    inputs; those before them have tests of their own."""
    B, T, D, H, Hk, V = 2, 70, 256, 4, 4, 3000
    d = D // H
    W = (H + 2 * Hk) * d
    g = torch.Generator(device="cuda").manual_seed(3)
    bf = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).bfloat16()
    x, o, gpre, gpost = bf(B * T, D), bf(B * T, D), bf(D).abs() + 0.5, bf(D).abs() + 0.5
    wqkv, wv = bf(D, W, std=D ** -0.5), bf(V, D, std=D ** -0.5)
    r, y, qkv = torch.empty_like(x), torch.empty_like(x), torch.empty(B * T, W, device="cuda", dtype=torch.bfloat16)
    rp = bwpp.ResidualNormParams(rows=B * T, cols=D, eps=1e-5, post_norm=1, dtype=1)
    be.dispatch_residual_norm(x, o, gpost, None, gpre, r, y, rp)
    _, y64, _ = resnorm64(x, o, gpost, None, gpre, 0, 1e-5, 1.0, 1.0, True)
    assert rel_max_err(y.double().cpu(), y64.cpu()) <= 2.0 ** -8
    be.dispatch_matmul(y, wqkv, qkv, None, bwpp.MatmulParams(B * T, W, D, D, W, W, 1, 0, 0, 0))
    before = qkv.clone()
    q, k = qkv[:, :H * d], qkv[:, H * d:(H + Hk) * d]
    st = {f"{n}{o_}_{s}": v for n in "qk" for o_ in ("", "o") for s, v in (("head_stride", d), ("batch_stride", T * W))}
    be.dispatch_rotary(q, k, None, q, k, bwpp.RotaryParams(tokens=T, q_heads=H, k_heads=Hk, dim=d, batch=B, dtype=1, ldq=W,
                                                           ldk=W, ldqo=W, ldko=W, pos_offset=1000, **st))
    pos = (torch.arange(T, device="cuda") + 1000)[None].expand(B, T)
    want, _ = rotary64(before[:, :(H + Hk) * d].reshape(B, T, H + Hk, d), pos, d, False)
    got = qkv[:, :(H + Hk) * d].reshape(B, T, H + Hk, d).double()
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all())
    assert torch.equal(qkv[:, (H + Hk) * d:], before[:, (H + Hk) * d:])
    ctx = torch.empty(B * T, D, device="cuda", dtype=torch.bfloat16)
    ap = bwpp.AttentionParams(M=T, N=T, K=d, D=d, ldq=W, ldk=W, ldv=W, ldo=D, batch=B, heads=H, q_batch_stride=T * W,
                              q_head_stride=d, k_batch_stride=T * W, k_head_stride=d, v_batch_stride=T * W,
                              v_head_stride=d, o_batch_stride=T * D, o_head_stride=d, scale=d ** -0.5, causal=1, dtype=1)
    be.dispatch_attention(q, k, qkv[:, 2 * D:], ctx, ap)
    heads = lambda t: t.reshape(B, T, H, d).permute(0, 2, 1, 3).double().contiguous()
    s = heads(q) @ heads(k).transpose(-1, -2).contiguous() * d ** -0.5
    s = s.masked_fill(~torch.ones(T, T, dtype=torch.bool, device="cuda").tril(), -float("inf"))
    want = (torch.softmax(s, dim=-1) @ heads(qkv[:, 2 * D:])).permute(0, 2, 1, 3).reshape(B * T, D)
    assert rel_max_err(ctx.double().cpu(), want.cpu()) <= 2e-2  # the attention tests' bar
    be.dispatch_residual_norm(r, ctx, gpost, None, gpre, r, y, rp)
    t = torch.randint(0, V, (B * T,), device="cuda", generator=g, dtype=torch.int32)
    loss = torch.empty(B * T, device="cuda")
    be.dispatch_linear_xent(y, wv, t, loss, None, None, bwpp.LinearXentParams(rows=B * T, vocab=V, dim=D, trans_w=1, dtype=1))
    want = xent64(y, wv, t)[0]
    assert float((loss.double() - want).abs().max()) <= (D + 2) * 2.0 ** -24 * float((y.abs().double() @ wv.abs().double().t()).max()) * 2 + 1e-5

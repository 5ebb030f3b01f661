"""Negative numbers in a plan's ops are the entry points' (the same kernels on
the same values: the same bits)."""
import pytest
import torch

import bwpp
from bwpp import plan

pytestmark = pytest.mark.gpu

PLAN = """bwpp.plan 1
dim T 37
dim D 64
value x f32 [T,D] input
value o f32 [T,D] input
value wv f32 [200,D] param
value t i32 [T] input
value rot f32 [T,D] output
value r f32 [T,D] output
value y f32 [T,D] output
value l f32 [T] output
value a f32 [T,D] output
op rotary out=rot in=x heads=2 offset=-7 magnitude=-2
op residual_norm out=r,y in=x,o stream_scale=-1 branch_scale=-3 eps=1e-6
op linear_xent out=l in=x,wv,t gives=loss trans_w=1 scale=-1
op attention out=a in=x,o,x heads=2 scale=-1 causal=1
"""


def test_negative_numbers(be):
    T, D, V = 37, 64, 200
    g = torch.Generator(device="cuda").manual_seed(2)
    x, o, wv = (torch.randn(n, D, device="cuda", generator=g) * 0.3 for n in (T, T, V))
    t = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
    p = plan.Plan(be, PLAN)
    p.allocate()
    for name, v in dict(x=x, o=o, wv=wv, t=t).items():
        p.bind(name, v)
    p.run()
    rot, r, y, a = (torch.empty_like(x) for _ in range(4))
    loss = torch.empty(T, device="cuda")
    st = {f"{n}_head_stride": 32 for n in ("q", "qo")}
    be.dispatch_rotary(x, None, None, rot, None, bwpp.RotaryParams(tokens=T, q_heads=2, dim=32, ldq=D, ldqo=D, pos_offset=-7,
                                                                   magnitude=-2.0, **st))
    be.dispatch_residual_norm(x, o, None, None, None, r, y, bwpp.ResidualNormParams(rows=T, cols=D, eps=1e-6, stream_scale=-1.0,
                                                                                    branch_scale=-3.0))
    be.dispatch_linear_xent(x, wv, t, loss, None, None, bwpp.LinearXentParams(rows=T, vocab=V, dim=D, trans_w=1, scale=-1.0))
    ap = bwpp.AttentionParams(M=T, N=T, K=32, D=32, ldq=D, ldk=D, ldv=D, ldo=D, batch=1, heads=2, scale=-1.0, causal=1,
                              **{f"{n}_head_stride": 32 for n in "qkvo"}, **{f"{n}_batch_stride": T * D for n in "qkvo"})
    be.dispatch_attention(x, o, x, a, ap)
    for name, want in dict(rot=rot, r=r, y=y, l=loss, a=a).items():
        got = torch.from_numpy(p.host(name, tuple(want.shape)))
        assert torch.equal(got, want.cpu()), name
        assert bool(got.isfinite().all())
    p.close()

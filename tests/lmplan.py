"""A language model's training step around one block as a launch plan, and the
same step in 64 bits: joins with their norms, rotary positions, causal
attention, an MLP, the cross entropy against a vocabulary, and back."""
import torch

TRAIN = """bwpp.plan 1
dim B 2
dim T 24
dim D 64
dim HEADS 4
dim F 96
dim V 500

value x f32 [B*T,D] input
value o0 f32 [B*T,D] input
value targets i32 [B*T] input
value pos i32 [T] input
value gpre0 f32 [D] param
value wqkv f32 [D,3*D] param
value wo f32 [D,D] param
value gpost1 f32 [D] param
value gate1 f32 [1,D] param
value gpre1 f32 [D] param
value w1 f32 [D,F] param
value w2 f32 [F,D] param
value gpost2 f32 [D] param
value gate2 f32 [B,D] param
value gpre2 f32 [D] param
value wv f32 [V,D] param
value one f32 [1,1] const=1

value r0 f32 [B*T,D] temp
value y0 f32 [B*T,D] temp
value qkv f32 [B*T,3*D] temp
view q of=qkv offset=0 ld=3*D shape=[B*T,D]
view k of=qkv offset=D ld=3*D shape=[B*T,D]
view v of=qkv offset=2*D ld=3*D shape=[B*T,D]
value ctx f32 [B*T,D] temp
value alse f32 [B,HEADS,T] temp
value ao f32 [B*T,D] temp
value r1 f32 [B*T,D] temp
value y1 f32 [B*T,D] temp
value hpre f32 [B*T,F] temp
value h f32 [B*T,F] temp
value m f32 [B*T,D] temp
value r2 f32 [B*T,D] temp
value y2 f32 [B*T,D] output
value loss f32 [B*T] output
value xlse f32 [B*T] temp
value sums f32 [2] output
view count of=sums offset=1 ld=1 shape=[1,1]
value dl f32 [1,1] temp
value dy2 f32 [B*T,D] temp
value dwv f32 [V,D] output
value dr1 f32 [B*T,D] temp
value dm f32 [B*T,D] temp
value dgpost2 f32 [D] output
value dgate2 f32 [B,D] output
value dgpre2 f32 [D] output
value dw2 f32 [F,D] output
value dh f32 [B*T,F] temp
value dhpre f32 [B*T,F] temp
value dw1 f32 [D,F] output
value dy1 f32 [B*T,D] temp
value dr0 f32 [B*T,D] temp
value dao f32 [B*T,D] temp
value dgpost1 f32 [D] output
value dgate1 f32 [1,D] output
value dgpre1 f32 [D] output
value dwo f32 [D,D] output
value dctx f32 [B*T,D] temp
value dqkv f32 [B*T,3*D] temp
view dq of=dqkv offset=0 ld=3*D shape=[B*T,D]
view dk of=dqkv offset=D ld=3*D shape=[B*T,D]
view dv of=dqkv offset=2*D ld=3*D shape=[B*T,D]
value dwqkv f32 [D,3*D] output
value dy0 f32 [B*T,D] temp
value dx f32 [B*T,D] output
value do0 f32 [B*T,D] output
value dgpre0 f32 [D] output

op residual_norm out=r0,y0 in=x,o0,gpre0 with=pre
op matmul out=qkv in=y0,wqkv
op rotary out=q,k in=q,k,pos batch=B heads=HEADS rot=8 scaling=parts factor=4 context=64 low=0.5 high=4 magnitude=1.125
op attention out=ctx,alse in=q,k,v batch=B heads=HEADS causal=1 scale=auto
op matmul out=ao in=ctx,wo
op residual_norm out=r1,y1 in=r0,ao,gpost1,gate1,gpre1 with=post,gate,pre branch_scale=0.5
op matmul out=hpre in=y1,w1
op silu out=h in=hpre
op matmul out=m in=h,w2
op residual_norm out=r2,y2 in=r1,m,gpost2,gate2,gpre2 with=post,gate,pre gate_rows=T stream_scale=0.75
op linear_xent out=loss,xlse,sums in=y2,wv,targets gives=loss,lse,sums trans_w=1
op div out=dl in=one,count
op linear_xent_grad out=dy2,dwv in=y2,wv,targets,xlse,dl gives=dx,dw trans_w=1
op residual_norm_grad out=dr1,dm,dgpost2,dgate2,dgpre2 in=m,r2,gpost2,gate2,gpre2,dy2 with=post,gate,pre,dy gives=dx,do,dpost,dgate,dpre gate_rows=T stream_scale=0.75
op matmul out=dw2 in=h,dm ta=1
op matmul out=dh in=dm,w2 tb=1
op silu_grad out=dhpre in=hpre,dh
op matmul out=dw1 in=y1,dhpre ta=1
op matmul out=dy1 in=dhpre,w1 tb=1
op residual_norm_grad out=dr0,dao,dgpost1,dgate1,dgpre1 in=ao,r1,gpost1,gate1,gpre1,dr1,dy1 with=post,gate,pre,dr,dy gives=dx,do,dpost,dgate,dpre branch_scale=0.5
op matmul out=dwo in=ctx,dao ta=1
op matmul out=dctx in=dao,wo tb=1
op attention_grad out=dq,dk,dv in=q,k,v,ctx,dctx,alse batch=B heads=HEADS causal=1 scale=auto
op rotary_grad out=dq,dk in=dq,dk,pos batch=B heads=HEADS rot=8 scaling=parts factor=4 context=64 low=0.5 high=4 magnitude=1.125
op matmul out=dwqkv in=y0,dqkv ta=1
op matmul out=dy0 in=dqkv,wqkv tb=1
op residual_norm_grad out=dx,do0,dgpre0 in=o0,r0,gpre0,dr0,dy0 with=pre,dr,dy gives=dx,do,dpre
"""

GRADS = dict(dx="x", do0="o0", dgpre0="gpre0", dwqkv="wqkv", dwo="wo", dgpost1="gpost1", dgate1="gate1",
             dgpre1="gpre1", dw1="w1", dw2="w2", dgpost2="gpost2", dgate2="gate2", dgpre2="gpre2", dwv="wv")


def inputs(B, T, D, F, V, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, std=1.0: torch.randn(*s, device="cuda", generator=g) * std
    u = lambda *s: torch.rand(*s, device="cuda", generator=g) + 0.5
    t = dict(x=n(B * T, D), o0=n(B * T, D), gpre0=u(D), wqkv=n(D, 3 * D, std=D ** -0.5), wo=n(D, D, std=D ** -0.5),
             gpost1=u(D), gate1=u(1, D), gpre1=u(D), w1=n(D, F, std=D ** -0.5), w2=n(F, D, std=F ** -0.5), gpost2=u(D),
             gate2=u(B, D), gpre2=u(D), wv=n(V, D, std=D ** -0.5))
    t["targets"] = torch.randint(0, V, (B * T,), device="cuda", generator=g, dtype=torch.int32)
    t["targets"][::5] = -1
    t["pos"] = torch.arange(T, device="cuda", dtype=torch.int32) * 3 + 7
    return t


def step64(t, B, T, HEADS):
    """Losses, mean-loss gradients by output name, in 64-bit autograd."""
    from lm64 import rotary64
    p = {k: (v.double().requires_grad_(True) if v.is_floating_point() else v) for k, v in t.items()}
    D = p["x"].shape[1]
    norm = lambda v: v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-5)
    r0 = p["x"] + p["o0"]
    qkv = (norm(r0) * p["gpre0"]) @ p["wqkv"]
    q, k, v = (a.reshape(B, T, HEADS, D // HEADS) for a in qkv.split(D, dim=1))
    pos = p["pos"][None].expand(B, T)
    q, k = (rotary64(a, pos, 8, False, scaling=2, factor=4.0, context=64, low=0.5, high=4.0, magnitude=1.125)[0]
            for a in (q, k))
    heads = lambda a: a.permute(0, 2, 1, 3).contiguous()
    s = heads(q) @ heads(k).transpose(-1, -2).contiguous() * (D // HEADS) ** -0.5
    s = s.masked_fill(~torch.ones(T, T, dtype=torch.bool, device=s.device).tril(), -float("inf"))
    ctx = (torch.softmax(s, dim=-1) @ heads(v)).permute(0, 2, 1, 3).reshape(B * T, D)
    r1 = r0 + 0.5 * p["gate1"] * norm(ctx @ p["wo"]) * p["gpost1"]
    m = torch.nn.functional.silu((norm(r1) * p["gpre1"]) @ p["w1"]) @ p["w2"]
    r2 = 0.75 * r1 + p["gate2"].repeat_interleave(T, dim=0) * norm(m) * p["gpost2"]
    y2 = norm(r2) * p["gpre2"]
    z = y2 @ p["wv"].t()
    live = t["targets"] >= 0
    loss = torch.logsumexp(z, dim=1) - z.gather(1, t["targets"].clamp(min=0).long()[:, None])[:, 0]
    loss = torch.where(live, loss, 0.0)
    (loss.sum() / live.sum()).backward()
    return loss.detach(), y2.detach(), {g: p[n].grad for g, n in GRADS.items()}

"""The operators around a transformer block as a training or scoring program
calls them, over the range of sizes, data types and directions in use, each
also in its plain form (elementary torch operations in 32 bits).

Kinds:

  rotary         rotary positions of the q and k of one attention call
  rotary_grad    their gradient
  norm           the join of a block's branch with the residual stream:
                 post-norm, gate and scales, and the next block's pre-norm
  norm_grad      its gradient, weight and gate gradients among it
  loss           cross entropy of hidden states against a vocabulary
  loss_train     the same, then the gradients of hidden states and weights
"""
import math
import os
import sys

import torch

own = False
_BACKEND = None


def _bwpp():
    path = os.path.join(os.getcwd(), "bluewolf-plus-plus_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bwpp
    return bwpp


def _backend():
    """The handle a program keeps for its lifetime, on torch's stream."""
    global _BACKEND
    if _BACKEND is None:
        _BACKEND = _bwpp().HipBackend(0)
    _BACKEND.set_stream(torch.cuda.current_stream())
    return _BACKEND


# ------------------------------------------------------------------- cases


def listed():
    return [
        # One decoding step of eight sequences far into a long context, by-parts
        # frequency scaling: the smallest call, where latency counts.
        dict(name="rotary_decode_8x1", kind="rotary", dtype="bf16", B=8, S=1, Hq=32, Hk=8, d=128, rot=128,
             layout="half", scaling="parts", positions=True),
        # Training: q and k as they leave the fused projection, four sequences.
        dict(name="rotary_bf16_4x4096", kind="rotary", dtype="bf16", B=4, S=4096, Hq=32, Hk=8, d=128, rot=128,
             layout="half", scaling="none", positions=False),
        # The gradient in fp32 with odd sizes: interleaved pairs over a part of
        # the head, linear scaling, packed sequences with positions of their own.
        dict(name="rotary_grad_f32_3x1001", kind="rotary_grad", dtype="f32", B=3, S=1001, Hq=12, Hk=12, d=80, rot=40,
             layout="interleaved", scaling="linear", positions=True),
        # One decoding step of sixteen sequences.
        dict(name="norm_bf16_16x4096", kind="norm", dtype="bf16", rows=16, cols=4096, pad=0, post=True, gate_rows=0),
        # A full batch of activations between two blocks.
        dict(name="norm_bf16_8192x4096", kind="norm", dtype="bf16", rows=8192, cols=4096, pad=0, post=True,
             gate_rows=0),
        # Its backward, the gate being a row per sequence of 1024 tokens.
        dict(name="norm_grad_bf16_8192x4096", kind="norm_grad", dtype="bf16", rows=8192, cols=4096, pad=0, post=True,
             gate_rows=1024),
        # fp32 with odd sizes and rows at any 4-byte address, no post-norm.
        dict(name="norm_grad_f32_1999x1021", kind="norm_grad", dtype="f32", rows=1999, cols=1021, pad=2, post=False,
             gate_rows=0),
        # Scoring the next token of a few sequences.
        dict(name="loss_bf16_4x1024x16384", kind="loss", dtype="bf16", T=4, D=1024, V=16384, wide="vd"),
        # Evaluating a batch against a vocabulary of odd size.
        dict(name="loss_bf16_2048x4096x50001", kind="loss", dtype="bf16", T=2048, D=4096, V=50001, wide="vd"),
        # A training step's loss, the weights stored as the DSL's x @ w.
        dict(name="loss_train_bf16_4096x2048x32768", kind="loss_train", dtype="bf16", T=4096, D=2048, V=32768,
             wide="dv"),
        # The same in fp32 with odd sizes throughout.
        dict(name="loss_train_f32_777x1021x8003", kind="loss_train", dtype="f32", T=777, D=1021, V=8003, wide="vd"),
        # The largest: a wide model with a large vocabulary.
        dict(name="loss_train_bf16_4096x4096x131072", kind="loss_train", dtype="bf16", T=4096, D=4096, V=131072,
             wide="vd"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, step):
    """Mostly a multiple of `step`, at times any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.35 else max(lo, n // step * step)


def draw(rng):
    kind = rng.choice(["rotary", "rotary_grad", "norm", "norm_grad", "loss", "loss", "loss_train", "loss_train"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind in ("rotary", "rotary_grad"):
        d = rng.choice([32, 64, 80, 96, 128, 192, 256])
        Hk = rng.choice([1, 2, 4, 8, 16])
        Hq = Hk * rng.choice([1, 2, 4])
        B = rng.randint(1, 16)
        S = _log_int(rng, 1, max(1, min(16384, 4 * 4096 * 48 * 128 // (B * (Hq + Hk) * d))))
        return dict(kind=kind, dtype=dtype, B=B, S=S, Hq=Hq, Hk=Hk, d=d, rot=rng.choice([d, d, d // 2]),
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "parts"]),
                    positions=rng.random() < 0.5)
    if kind in ("norm", "norm_grad"):
        cols = _size(rng, 64, 16384 if kind == "norm" else 8192, 64)
        rows = _log_int(rng, 1, min(32768, 8192 * 4096 // cols))
        return dict(kind=kind, dtype=dtype, rows=rows, cols=cols, pad=rng.choice([0, 0, 1, 8]),
                    post=rng.random() < 0.5, gate_rows=rng.choice([0, 1, 7, 512]))
    top = 4096 * 4096 * 131072 // 2 if dtype == "bf16" else 2 ** 34
    D = _size(rng, 128, 4096, 64)
    V = _size(rng, 512, 131072, 64)
    T = _log_int(rng, 1, max(1, min(8192, top // (D * V))))
    return dict(kind=kind, dtype=dtype, T=T, D=D, V=V, wide=rng.choice(["vd", "vd", "dv"]))


# ------------------------------------------------------------------ inputs


class _Inputs:
    """Seeded draws on the GPU; the same (seed, order) gives the same values."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std).add_(mean).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=self.g, device="cuda").mul_(hi - lo).add_(lo)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)


_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}
EPS = 1e-6
BASE = 10000.0
# frequency scaling: (factor, context trained on, low and high turns, magnitude)
_SCALING = {"none": (1.0, 0, 0.0, 0.0, 1.0), "linear": (4.0, 0, 0.0, 0.0, 1.0), "parts": (16.0, 8192, 1.0, 32.0, 1.25)}
_STREAM, _BRANCH = 1.5, 0.25


def _inputs(case, seed):
    """The tensors a pass reads, by name."""
    r = _Inputs(seed)
    k, dt = case["kind"], _TORCH[case["dtype"]]
    if k in ("rotary", "rotary_grad"):
        B, S, Hq, Hk, d = (case[i] for i in ("B", "S", "Hq", "Hk", "d"))
        if k == "rotary":  # q, k and v side by side, as the fused projection leaves them
            qkv = r.normal(B, S, Hq + 2 * Hk, d, dtype=dt)
            t = dict(q=qkv[:, :, :Hq], k=qkv[:, :, Hq:Hq + Hk])
        else:  # what the attention gradient leaves, head by head
            t = dict(q=r.normal(B, Hq, S, d, dtype=dt).transpose(1, 2), k=r.normal(B, Hk, S, d, dtype=dt).transpose(1, 2))
        if case["positions"]:
            top = 131072 if case["scaling"] == "parts" else 32768
            t["positions"] = r.ints(0, top - S, B, 1) + torch.arange(S, device="cuda", dtype=torch.int32)[None, :]
        return t
    if k in ("norm", "norm_grad"):
        rows, cols, ld, gr = case["rows"], case["cols"], case["cols"] + case["pad"], case["gate_rows"]
        ngate = (rows + gr - 1) // gr if gr else 1
        # the stream grows with depth, a branch is of order one
        t = dict(o=r.normal(rows, ld, std=0.7, dtype=dt)[:, :cols], gate=r.normal(ngate, cols, std=0.5, dtype=dt),
                 pre=r.uniform(cols, lo=0.5, hi=1.5).to(dt))
        if case["post"]:
            t["post"] = r.uniform(cols, lo=0.5, hi=1.5).to(dt)
        if k == "norm":
            t["x"] = r.normal(rows, ld, std=4.0, dtype=dt)[:, :cols]
        else:
            t["r"] = r.normal(rows, ld, std=4.0, dtype=dt)[:, :cols]
            t["dr"] = r.normal(rows, ld, std=0.5, dtype=dt)[:, :cols]
            t["dy"] = r.normal(rows, ld, dtype=dt)[:, :cols]
        return t
    T, D, V = case["T"], case["D"], case["V"]
    w = r.normal(V, D, std=1.5 / math.sqrt(D))
    target = r.ints(0, V, T)
    # hidden states that lean to their target, some strongly
    x = r.normal(T, D) + r.uniform(T, 1, lo=0.0, hi=5.0) * w[target.long()]
    t = dict(x=x.to(dt), w=(w if case["wide"] == "vd" else w.t().contiguous()).to(dt))
    # in training a fifth of the rows (prompts, padding) has no target
    live = r.uniform(T) >= 0.2
    live[0] = True
    t["target"] = torch.where(live, target, -1) if k == "loss_train" else target
    t["dloss"] = 1.0 / (t["target"] >= 0).sum().float().reshape(1)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    st = dict(case=case, t=t)
    if not own:
        return st
    bwpp = _bwpp()
    st["be"] = _backend()
    code = int(bwpp.DType.BF16 if case["dtype"] == "bf16" else bwpp.DType.F32)
    k, dt = case["kind"], _TORCH[case["dtype"]]
    new = lambda *s, dtype=dt: torch.zeros(*s, dtype=dtype, device="cuda")
    if k in ("rotary", "rotary_grad"):
        B, S, Hq, Hk, d = (case[i] for i in ("B", "S", "Hq", "Hk", "d"))
        q, kk = t["q"], t["k"]
        st["out"] = dict(q=new(B, S, Hq, d), k=new(B, S, Hk, d))
        factor, context, low, high, magnitude = _SCALING[case["scaling"]]
        scaling = dict(none=bwpp.RotaryScaling.NONE, linear=bwpp.RotaryScaling.LINEAR,
                       parts=bwpp.RotaryScaling.BY_PARTS)[case["scaling"]]
        layout = bwpp.RotaryLayout.HALF if case["layout"] == "half" else bwpp.RotaryLayout.INTERLEAVED
        a, b = ("q", "qo") if k == "rotary" else ("qo", "q")  # the gradient runs from the outputs' side
        c, e = ("k", "ko") if k == "rotary" else ("ko", "k")
        st["p"] = bwpp.RotaryParams(
            batch=B, tokens=S, q_heads=Hq, k_heads=Hk, dim=d, rot_dim=case["rot"], layout=int(layout), dtype=code,
            base=BASE, scaling=int(scaling), factor=factor, context=context, low_turns=low, high_turns=high,
            magnitude=magnitude, pos_batch_stride=S,
            **{f"ld{a}": q.stride(1), f"{a}_head_stride": q.stride(2), f"{a}_batch_stride": q.stride(0),
               f"ld{c}": kk.stride(1), f"{c}_head_stride": kk.stride(2), f"{c}_batch_stride": kk.stride(0),
               f"ld{b}": Hq * d, f"{b}_head_stride": d, f"{b}_batch_stride": S * Hq * d,
               f"ld{e}": Hk * d, f"{e}_head_stride": d, f"{e}_batch_stride": S * Hk * d})
    elif k in ("norm", "norm_grad"):
        rows, cols, ld = case["rows"], case["cols"], case["cols"] + case["pad"]
        st["p"] = bwpp.ResidualNormParams(rows=rows, cols=cols, ldx=ld, ldo=ld, ldy=ld, post_norm=int(case["post"]),
                                          gate_rows=case["gate_rows"], eps=EPS, stream_scale=_STREAM,
                                          branch_scale=_BRANCH, dtype=code)
        if k == "norm":
            st["out"] = dict(r=new(rows, ld)[:, :cols], y=new(rows, ld)[:, :cols])
        else:
            st["out"] = dict(dx=new(rows, ld)[:, :cols], do=new(rows, ld)[:, :cols], dpre=new(cols),
                             dgate=torch.zeros_like(t["gate"]))
            if case["post"]:
                st["out"]["dpost"] = new(cols)
    else:
        T, D, V = case["T"], case["D"], case["V"]
        st["p"] = bwpp.LinearXentParams(rows=T, vocab=V, dim=D, trans_w=int(case["wide"] == "vd"), dtype=code,
                                        dloss_scalar=1)
        st["out"] = dict(loss=new(T, dtype=torch.float32), lse=new(T, dtype=torch.float32),
                         sums=new(2, dtype=torch.float32))
        if k == "loss_train":
            st["out"].update(dx=new(T, D), dw=torch.zeros_like(t["w"]))
    return st


# --------------------------------------------------------------- one pass


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    be, t, o, p, k = st["be"], st["t"], st["out"], st["p"], st["case"]["kind"]
    if k == "rotary":
        be.dispatch_rotary(t["q"], t["k"], t.get("positions"), o["q"], o["k"], p)
    elif k == "rotary_grad":
        be.dispatch_rotary_grad(t["q"], t["k"], t.get("positions"), o["q"], o["k"], p)
    elif k == "norm":
        be.dispatch_residual_norm(t["x"], t["o"], t.get("post"), t["gate"], t["pre"], o["r"], o["y"], p)
    elif k == "norm_grad":
        be.dispatch_residual_norm_grad(t["o"], t["r"], t.get("post"), t["gate"], t["pre"], t["dr"], t["dy"], o["dx"],
                                       o["do"], o.get("dpost"), o["dgate"], o["dpre"], p)
    else:
        be.dispatch_linear_xent(t["x"], t["w"], t["target"], o["loss"], o["lse"], o["sums"], p)
        if k == "loss_train":
            be.dispatch_linear_xent_grad(t["x"], t["w"], t["target"], o["lse"], t["dloss"], o["dx"], o["dw"], p)
    return o


def _angles(case, t):
    """[B or 1, S, rot / 2] angles in 64 bits: far positions lose them in 32."""
    n = case["rot"]
    f = BASE ** (-torch.arange(0, n, 2, device="cuda", dtype=torch.float64) / n)
    factor, context, low, high, magnitude = _SCALING[case["scaling"]]
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "parts":
        c = ((context * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * (c + (1.0 - c) / factor)
    p = t["positions"] if case["positions"] else torch.arange(case["S"], device="cuda")[None, :]
    return p.double()[:, :, None] * f, magnitude


def _rms(v):
    return torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS)


def _rms_grad(v, s, g):
    """Gradient of v * s(v), s = _rms(v), for the upstream gradient g."""
    return s * (g - v * (s * s) * (g * v).mean(dim=1, keepdim=True))


def _gate_sum(case, v):
    gr = case["gate_rows"]
    if gr == 1:
        return v
    if gr == 0:
        return v.sum(dim=0, keepdim=True)
    n = (v.shape[0] + gr - 1) // gr
    return torch.nn.functional.pad(v, (0, 0, 0, n * gr - v.shape[0])).reshape(n, gr, -1).sum(dim=1)


def _gate_rows(case, gate):
    gr = case["gate_rows"]
    return gate if gr < 2 else gate.repeat_interleave(gr, dim=0)[:case["rows"]]


def _run_plain(st):
    case, t = st["case"], st["t"]
    k, dt = case["kind"], _TORCH[case["dtype"]]
    if k in ("rotary", "rotary_grad"):
        a, m = _angles(case, t)
        cos, sin = (a.cos() * m).float()[:, :, None, :], (a.sin() * m).float()[:, :, None, :]
        if k == "rotary_grad":
            sin = -sin
        n, out = case["rot"], {}
        for name in ("q", "k"):
            v = t[name].float()
            if case["layout"] == "half":
                x, y = v[..., :n // 2], v[..., n // 2:n]
                rot = torch.cat([x * cos - y * sin, y * cos + x * sin], dim=-1)
            else:
                x, y = v[..., 0:n:2], v[..., 1:n:2]
                rot = torch.stack([x * cos - y * sin, y * cos + x * sin], dim=-1).flatten(-2)
            out[name] = torch.cat([rot, v[..., n:]], dim=-1).to(dt)
        return out
    if k == "norm":
        u = t["o"].float()
        if case["post"]:
            u = u * _rms(u) * t["post"].float()
        r = _STREAM * t["x"].float() + _BRANCH * (_gate_rows(case, t["gate"]).float() * u)
        return dict(r=r.to(dt), y=(r * _rms(r) * t["pre"].float()).to(dt))
    if k == "norm_grad":
        o, r, dy, g = t["o"].float(), t["r"].float(), t["dy"].float(), _gate_rows(case, t["gate"]).float()
        s = _rms(r)
        dt_ = t["dr"].float() + _rms_grad(r, s, dy * t["pre"].float())
        out = dict(dx=(_STREAM * dt_).to(dt), dpre=(dy * r * s).sum(dim=0).to(dt))
        b = _BRANCH * dt_
        if case["post"]:
            so = _rms(o)
            oh, du = o * so, b * g
            out["dgate"] = _gate_sum(case, b * oh * t["post"].float()).to(dt)
            out["dpost"] = (du * oh).sum(dim=0).to(dt)
            out["do"] = _rms_grad(o, so, du * t["post"].float()).to(dt)
        else:
            out["dgate"] = _gate_sum(case, b * o).to(dt)
            out["do"] = (b * g).to(dt)
        return out
    x, w = t["x"].float(), t["w"].float()
    z = x @ (w.t() if case["wide"] == "vd" else w)
    live = t["target"] >= 0
    at = t["target"].clamp(min=0).long()[:, None]
    top = z.max(dim=1, keepdim=True).values
    zt = z.gather(1, at)
    z = z.sub_(top).exp_()
    total = z.sum(dim=1, keepdim=True)
    lse = top + total.log()
    loss = torch.where(live, (lse - zt)[:, 0], 0.0)
    out = dict(loss=loss, lse=lse[:, 0], sums=torch.stack([loss.sum(), live.sum().float()]))
    if k == "loss_train":
        z.div_(total)
        z.scatter_add_(1, at, torch.full_like(zt, -1.0))
        z.mul_(torch.where(live, t["dloss"], 0.0)[:, None])
        out["dx"] = (z @ (w if case["wide"] == "vd" else w.t())).to(dt)
        out["dw"] = (z.t() @ x if case["wide"] == "vd" else x.t() @ z).to(dt)
    return out


# ------------------------------------------------------- what it must cost


def work(case):
    k, e = case["kind"], _BYTES[case["dtype"]]
    if k in ("rotary", "rotary_grad"):
        rows = case["B"] * case["S"]
        heads = case["Hq"] + case["Hk"]
        return dict(bytes=2 * rows * heads * case["d"] * e + (4 * rows if case["positions"] else 0),
                    flops=rows * (heads * 3 * case["rot"] + 20 * case["rot"] // 2))
    if k in ("norm", "norm_grad"):
        n, cols = case["rows"] * case["cols"], case["cols"]
        gates = (-(-case["rows"] // case["gate_rows"]) if case["gate_rows"] else 1) * cols
        small = cols * (2 if case["post"] else 1) + gates
        if k == "norm":
            return dict(bytes=(4 * n + small) * e, flops=12 * n)
        return dict(bytes=(6 * n + 2 * small) * e, flops=30 * n)
    T, D, V = case["T"], case["D"], case["V"]
    once = (T * D + V * D) * e + 12 * T
    if k == "loss":
        return dict(bytes=once, flops=2.0 * T * D * V)
    # the gradients need two more products; the logits once
    return dict(bytes=once + (T * D + V * D) * e, flops=6.0 * T * D * V)


# -------------------------------------------------- the same in 64 bits


def exact(case, seed):
    t = _inputs(case, seed)
    k = case["kind"]
    if k in ("rotary", "rotary_grad"):
        # a pair as a complex number, turned by e^(i p f)
        n = case["rot"]
        i = torch.arange(n // 2, device="cuda", dtype=torch.float64)
        f = torch.exp(-(2.0 * i / n) * math.log(BASE))
        factor, context, low, high, magnitude = _SCALING[case["scaling"]]
        if case["scaling"] == "linear":
            f = f / factor
        if case["scaling"] == "parts":
            turns = context * f / (2 * math.pi)
            kept = torch.clamp((turns - low) / (high - low), 0.0, 1.0)
            f = kept * f + (1.0 - kept) * (f / factor)
        pos = t["positions"].double() if case["positions"] else torch.arange(
            case["S"], device="cuda", dtype=torch.float64)[None, :]
        a = pos[..., None] * f
        turn = torch.polar(torch.full_like(a, magnitude), a if k == "rotary" else -a)[:, :, None, :]
        out = {}
        for name in ("q", "k"):
            v = t[name].double().clone()
            if case["layout"] == "half":
                z = torch.complex(v[..., :n // 2].contiguous(), v[..., n // 2:n].contiguous()) * turn
                v[..., :n // 2], v[..., n // 2:n] = z.real, z.imag
            else:
                z = torch.complex(v[..., 0:n:2].contiguous(), v[..., 1:n:2].contiguous()) * turn
                v[..., 0:n:2], v[..., 1:n:2] = z.real, z.imag
            out[name] = v
        return out
    if k in ("norm", "norm_grad"):
        v = {n: a.double() for n, a in t.items()}
        rows, gr = case["rows"], case["gate_rows"]
        which = torch.arange(rows, device="cuda") // gr if gr else torch.zeros(rows, device="cuda", dtype=torch.long)
        gate = v["gate"][which]
        inv = lambda a: 1.0 / torch.sqrt(a.pow(2).mean(dim=1, keepdim=True) + EPS)
        post = v.get("post", torch.ones(case["cols"], device="cuda", dtype=torch.float64))
        io = inv(v["o"]) if case["post"] else torch.ones(rows, 1, device="cuda", dtype=torch.float64)
        oh = v["o"] * io
        if k == "norm":
            r = _STREAM * v["x"] + _BRANCH * gate * (oh * post)
            return dict(r=r, y=r * inv(r) * v["pre"])
        ir = inv(v["r"])
        rh = v["r"] * ir
        back = lambda h, i, g: i * (g - h * (h * g).mean(dim=1, keepdim=True))
        d = v["dr"] + back(rh, ir, v["dy"] * v["pre"])
        du = _BRANCH * d * gate
        dgate = torch.zeros_like(v["gate"]).index_add_(0, which, _BRANCH * d * oh * post)
        out = dict(dx=_STREAM * d, do=back(oh, io, du * post) if case["post"] else du, dpre=(v["dy"] * rh).sum(dim=0),
                   dgate=dgate)
        if case["post"]:
            out["dpost"] = (du * oh).sum(dim=0)
        return out
    x = t["x"].double()
    w = t["w"].double() if case["wide"] == "vd" else t["w"].double().t().contiguous()
    target = t["target"].long()
    live = target >= 0
    z = x @ w.t()
    lse = torch.logsumexp(z, dim=1)
    row = torch.arange(case["T"], device="cuda")
    loss = (lse - z[row, target.clamp(min=0)]) * live
    out = dict(loss=loss, lse=lse, sums=torch.stack([loss.sum(), live.sum().double()]))
    if k == "loss_train":
        z.sub_(lse[:, None]).exp_()
        z[row[live], target[live]] -= 1.0
        z.mul_((live * t["dloss"].double())[:, None])
        out["dx"] = z @ w
        dw = z.t() @ x
        out["dw"] = dw if case["wide"] == "vd" else dw.t().contiguous()
    return out

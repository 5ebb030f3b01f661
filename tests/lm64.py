"""Plain 64-bit forms of the operators around the block, for their tests,
and strided device buffers with guard values between the rows."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
PAD = 5.0


def strided(shape, strides, dtype, value=None):
    """A CUDA tensor of `shape` at element `strides` in a buffer of PAD, and the
    buffer; filled with `value` where given."""
    n = 1 + sum((a - 1) * b for a, b in zip(shape, strides))
    buf = torch.full((n + 8,), PAD, device="cuda", dtype=dtype)
    t = torch.as_strided(buf, shape, strides)
    if value is not None:
        t.copy_(value)
    return t, buf


def untouched(t, buf):
    """Whether nothing but t's own elements was written in its buffer."""
    mine = torch.zeros(buf.numel(), device="cuda", dtype=torch.bool)
    torch.as_strided(mine, t.shape, t.stride()).fill_(True)
    return bool((buf[~mine] == PAD).all())


def rotary64(x, positions, rot, interleaved, base=10000.0, scaling=0, factor=1.0, context=0, low=0.0, high=0.0,
             magnitude=1.0, grad=False):
    """x [B, T, H, d] (any float type), positions [B, T]; returns the result and,
    per element, the sum of the magnitudes of its two terms."""
    v = x.double()
    if rot == 0:
        return v, v.abs()
    f = base ** (-torch.arange(0, rot, 2, device=x.device, dtype=torch.float64) / rot)
    if scaling == 1:
        f = f / factor
    if scaling == 2:
        c = ((context * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (c + (1 - c) / factor)
    a = positions.double()[:, :, None, None] * f
    cos, sin = torch.cos(a) * magnitude, torch.sin(a) * (-magnitude if grad else magnitude)
    at = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    p, q = v[..., at[0]], v[..., at[1]]
    out, size = v.clone(), v.abs()
    out[..., at[0]], out[..., at[1]] = p * cos - q * sin, q * cos + p * sin
    both = (p.abs() + q.abs()) * abs(magnitude)
    size[..., at[0]], size[..., at[1]] = both, both
    return out, size


def _rstd(v, eps):
    return 1.0 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps)


def gate_of(gate, rows, gate_rows):
    return gate[torch.arange(rows, device=gate.device) // gate_rows] if gate_rows else gate.expand(rows, -1)


def resnorm64(x, o, post, gate, pre, gate_rows, eps, a, b, post_norm):
    """r, y and the sums of magnitudes behind r."""
    x, o = x.double(), o.double()
    one = torch.ones(1, x.shape[1], dtype=torch.float64, device=x.device)
    u = o * _rstd(o, eps) * (one if post is None else post.double()) if post_norm else o
    g = one if gate is None else gate_of(gate.double(), x.shape[0], gate_rows)
    r = a * x + b * g * u
    size = (a * x).abs() + (b * g * u).abs()
    return r, r * _rstd(r, eps) * (one if pre is None else pre.double()), size


def resnorm_grad64(o, r, post, gate, pre, dr, dy, gate_rows, eps, a, b, post_norm):
    """Gradients by name, each with the sum of the magnitudes of its terms."""
    rows, cols = o.shape
    dev = o.device
    one = torch.ones(1, cols, dtype=torch.float64, device=dev)
    z = torch.zeros(rows, cols, dtype=torch.float64, device=dev)
    o, r = o.double(), r.double()
    dr, dy = (z if v is None else v.double() for v in (dr, dy))
    post, pre = (one if v is None else v.double() for v in (post, pre))
    gv = one if gate is None else gate_of(gate.double(), rows, gate_rows)
    ir = _rstd(r, eps)
    io = _rstd(o, eps) if post_norm else torch.ones_like(ir)
    hr, ho = r * ir, o * io
    m = lambda v: v.mean(dim=1, keepdim=True)
    t = dr + ir * (pre * dy - hr * m(pre * dy * hr))
    ts = dr.abs() + ir * ((pre * dy).abs() + hr.abs() * m((pre * dy * hr).abs()))
    e, es = b * t, abs(b) * ts
    u = ho * post
    ge, ges = gv * e, gv.abs() * es
    do = io * (post * ge - ho * m(post * ge * ho)) if post_norm else ge
    dos = io * ((post.abs() * ges) + ho.abs() * m(post.abs() * ges * ho.abs())) if post_norm else ges
    n = (rows + gate_rows - 1) // gate_rows if gate_rows else 1
    which = torch.arange(rows, device=dev) // gate_rows if gate_rows else torch.zeros(rows, device=dev, dtype=torch.long)
    by_gate = lambda v: torch.zeros(n, cols, dtype=torch.float64, device=dev).index_add_(0, which, v)
    return dict(dx=(a * t, abs(a) * ts), do=(do, dos), dpre=((dy * hr).sum(0), (dy * hr).abs().sum(0)),
                dpost=((ge * ho).sum(0), (ges * ho.abs()).sum(0)),
                dgate=(by_gate(e * u), by_gate(es * u.abs())))


def xent64(x, w_vd, target, scale=1.0, dloss=None):
    """x [T, D], w [V, D]; loss, lse, and with dloss [T] dx and dw [V, D]."""
    x, w = x.double(), w_vd.double()
    z = scale * (x @ w.t().contiguous())
    V = z.shape[1]
    live = (target >= 0) & (target < V)
    at = torch.where(live, target, 0).long()
    rows = torch.arange(z.shape[0], device=z.device)
    lse = torch.logsumexp(z, dim=1)
    loss = torch.where(live, lse - z[rows, at], 0.0)
    if dloss is None:
        return loss, lse
    p = torch.exp(z - lse[:, None])
    p[rows, at] -= 1.0
    p = torch.where(live[:, None], p * dloss.double()[:, None], 0.0)
    xs = torch.where(live[:, None], x, 0.0)
    return loss, lse, scale * (p @ w), scale * (p.t().contiguous() @ xs)

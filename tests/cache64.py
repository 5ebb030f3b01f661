"""A paged cache and what the operators over it give, in 64 bits: builders for
the tests' pools, tables and ragged batches, and plain forms that walk tokens
one by one through the table."""
import math

import torch

import bwpp
from lm64 import HALF_STEP, rotary64, strided

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Cache:
    """Pools in strided buffers of guard values, a table with pages in any
    order, and a ragged batch: `held` and `new` tokens of every sequence."""

    def __init__(self, held, new, Hk=2, d=64, page=16, dtype=F32, by_token=False, pad=0, spare=2, before=0, after=0,
                 ld_table=0, seed=0, max_pages=None):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.held, self.new, self.Hk, self.d, self.page, self.dtype = held, new, Hk, d, page, dtype
        need = [-(-(a + b) // page) for a, b in zip(held, new)]
        self.max_pages = max(need + [1]) if max_pages is None else max_pages
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=self.g, device="cuda").tolist()
        self.ld = ld_table or self.max_pages
        rows, at = [], 0
        for n in need:
            n = min(n, self.max_pages)
            rows.append(order[at:at + n] + [-1] * (self.ld - n))
            at += n
        self.table = i32(rows).reshape(len(held), self.ld)
        shape = (self.pages, page, Hk, d)
        if by_token:
            ts = Hk * d + pad
            strides = (page * ts, ts, d, 1)
        else:
            hs = page * (d + pad)
            strides = (Hk * hs, d + pad, hs, 1)
        self.strides = strides
        self.k, self.kbuf = strided(shape, strides, dtype, self.normal(*shape))
        self.v, self.vbuf = strided(shape, strides, dtype, self.normal(*shape))
        self.before = before
        starts = [before]
        for n in new:
            starts.append(starts[-1] + n)
        self.first = starts
        self.tokens = starts[-1] + after
        self.starts, self.held_t = i32(starts), i32(held)

    def normal(self, *shape, std=1.0):
        return (torch.randn(*shape, generator=self.g, device="cuda") * std).to(self.dtype)

    def params(self, Hq, **kw):
        s = self.strides
        d = dict(pages=self.pages, page_tokens=self.page, heads=self.Hk, dim=self.d, batch=len(self.held),
                 max_pages=self.max_pages, ld_table=self.ld, tokens=self.tokens, q_heads=Hq,
                 dtype=int(self.dtype == BF16), page_stride=s[0], token_stride=s[1], head_stride=s[2])
        d.update(kw)
        return bwpp.CacheParams(**d)

    def slot(self, s, p):
        """(page, place) of a slot, None if it does not exist."""
        if not 0 <= p < self.max_pages * self.page:
            return None
        page = int(self.table_cpu()[s][p // self.page])
        return (page, p % self.page) if 0 <= page < self.pages else None

    def table_cpu(self):
        if not hasattr(self, "_table"):
            self._table = self.table.tolist()
        return self._table

    def gather(self, s, length):
        """Keys and values [length, Hk, d] of a sequence's slots, and which of
        the slots exist."""
        places = [self.slot(s, p) for p in range(length)]
        live = torch.tensor([p is not None for p in places], dtype=torch.bool, device="cuda")
        at = torch.tensor([p or (0, 0) for p in places], device="cuda").reshape(length, 2)
        return self.k[at[:, 0], at[:, 1]], self.v[at[:, 0], at[:, 1]], live


def bits(mask):
    """bool [rows, n] as 32-bit words in int32, the lowest bit first."""
    rows, n = mask.shape
    words = max(1, -(-n // 32))
    m = torch.nn.functional.pad(mask.cpu(), (0, words * 32 - n)).reshape(rows, words, 32).to(torch.int64)
    v = (m << torch.arange(32)).sum(dim=2)
    return torch.where(v >= 2 ** 31, v - 2 ** 32, v).to(torch.int32).cuda()


def tree(n, g, back=4):
    """bool [n, n]: token i sees itself and its ancestors; its parent is one of
    the `back` tokens before it."""
    sees = torch.eye(n, dtype=torch.bool)
    pick = torch.rand(n, generator=g, device=g.device).cpu()
    for i in range(1, n):
        sees[i] |= sees[i - 1 - int(pick[i] * min(i, back))]
    return sees


def attention64(c, q, scale, sees=None):
    """o, lse and their bounds for q [tokens, Hq, d]; sees: per sequence, bool
    [n, n] (None: causal).  Rows outside the sequences are NaN.

    Bounds, u = 2^-24.  A score is a sum of d products in fp32, off by at most
    (d + 4) u S, S = |scale| sum |q k|; its exponential is off by that, by 2 u
    for the instruction and 2 u |score| for its scaling and offset: e.  bf16
    kernels hold a probability in two bf16 terms, 2^-16, or, where a key head has
    more than 32 rows on average, rounded to one bf16 (half a step of 8 significant
    bits: 2^-8 of it) for the weighted sum alone: r.  A sum over n keys
    adds n u to the weights' sum and to the weighted sum (running maxima,
    partial sums and joins rescale: 8 u and u for every 16 keys more, inside n u
    + 64 u).  So o is off by (2 e + r + (2 n + 64) u) sum w |v| and its own
    rounding (e enters twice, by the weights and their sum, r once), lse by e +
    (n + 64) u and 2 u |lse|."""
    T, Hq, d = q.shape
    o = torch.full((T, Hq, d), float("nan"), dtype=torch.float64, device="cuda")
    lse = torch.full((T, Hq), float("nan"), dtype=torch.float64, device="cuda")
    to, tl = torch.zeros_like(o), torch.zeros_like(lse)
    g = Hq // c.Hk
    one = q.dtype == BF16 and -(-T // len(c.held)) * g > 32
    for s, (held, n) in enumerate(zip(c.held, c.new)):
        if n == 0:
            continue
        r = slice(c.first[s], c.first[s] + n)
        L = held + n
        k, v, live = c.gather(s, L)
        ok = torch.ones(n, L, dtype=torch.bool, device="cuda")
        ok[:, held:] = (torch.ones(n, n, dtype=torch.bool).tril() if sees is None else sees[s]).cuda()
        ok &= live[None, :]
        for h in range(Hq):
            qq, kk, vv = q[r, h].double(), k[:, h // g].double(), v[:, h // g].double()
            # a key that a token does not see has no part in it, whatever it holds
            z = (qq[:, None, :] * kk[None, :, :]).sum(dim=2) * scale if L * n * d < 2 ** 27 else qq @ kk.T * scale
            S = (qq.abs() @ kk.abs().T * abs(scale)).nan_to_num(0, 0, 0).masked_fill(~ok, 0).amax(dim=1)
            z = z.masked_fill(~ok, -math.inf)
            top = z.amax(dim=1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            w = (z - top).exp()
            total = w.sum(dim=1)
            p = w / total.clamp(min=1e-300)[:, None]
            vis = torch.where(ok[:, :, None], vv[None], torch.zeros((), dtype=torch.float64, device="cuda"))
            o[r, h] = (p[:, :, None] * vis).sum(dim=1)
            lse[r, h] = torch.where(total == 0, torch.full_like(total, -math.inf), total.log() + top[:, 0])
            e = (d + 4) * U * S + 2 * U + 2 * U * S + (2.0 ** -16 if q.dtype == BF16 else 0.0)
            size = (p[:, :, None] * vis.abs()).sum(dim=1)
            to[r, h] = (2 * e + (2.0 ** -8 if one else 0.0) + (2 * L + 64) * U)[:, None] * size + HALF_STEP[q.dtype] * o[r, h].abs()
            tl[r, h] = e + (L + 64) * U + 2 * U * lse[r, h].abs().nan_to_num(0, 0, 0)
    return o, lse, to, tl


def append64(c, q, k, v, pos, rot, inter, scal, rotate=True):
    """q_out and the pools after an append, and the rotated elements' bounds (those
    of the rotary tests: half a step and 4 u of the two terms' magnitudes)."""
    kw = dict(scaling=scal.get("scaling", 0), factor=scal.get("factor", 1.0), context=scal.get("context", 0),
              low=scal.get("low_turns", 0.0), high=scal.get("high_turns", 0.0), magnitude=scal.get("magnitude", 1.0),
              base=scal.get("base", 10000.0))
    half = HALF_STEP[c.dtype]

    def turn(x):
        if not rotate:
            return x.double(), torch.zeros_like(x, dtype=torch.float64)
        y, size = rotary64(x[None], pos[None], rot, inter, **kw)
        tol = half * y.abs() + 4 * U * (1 + half) * size
        tol[..., rot:] = 0.0
        return y[0], tol[0]

    qo, tq = turn(q)
    ko, tk = turn(k)
    kc, vc, tkc = c.k.double(), c.v.double(), torch.zeros_like(c.k, dtype=torch.float64)
    for s, (held, n) in enumerate(zip(c.held, c.new)):
        for i in range(n):
            at = c.slot(s, held + i)
            if at is not None:
                t = c.first[s] + i
                kc[at], vc[at], tkc[at] = ko[t], v[t].double(), tk[t]
    live = torch.zeros(c.tokens, dtype=torch.bool, device="cuda")
    live[c.first[0]:c.first[-1]] = True
    return qo, tq, kc, tkc, vc, live

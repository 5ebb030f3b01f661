"""A paged cache of keys and values as a serving loop uses it: new tokens are
rotated and appended, attention reads the cache (one token a sequence, a tree
of drafted tokens, a piece of a prompt), accepted drafts are kept, and rules
for the next token are applied to the logits.  Each also in its plain form
(elementary torch operations in 32 bits).

Kinds:

  append  rotary positions of new q and k, keys and values into their pages
  attend  attention of the new tokens over the cache, with its log-sum-exp
  keep    the accepted tokens of drafted trees moved together
  rules   penalties for repeated tokens, biases and a grammar's mask on logits
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
        # One decoding step of eight sequences, by-parts frequency scaling: the
        # smallest call, where latency counts; the pages hold head after head.
        dict(name="append_bf16_8x1", kind="append", dtype="bf16", seqs=8, idle=0, pad=0, new=1, ragged=False,
             held=8000, Hq=32, Hk=8, d=128, page=64, by_token=False, rot=128, layout="half", scaling="parts"),
        # Pieces of prompts in fp32 with odd sizes, interleaved pairs over a part
        # of the head, small pages that hold token after token, one idle sequence.
        dict(name="append_f32_5x333", kind="append", dtype="f32", seqs=5, idle=1, pad=7, new=333, ragged=True,
             held=1001, Hq=12, Hk=12, d=80, page=16, by_token=True, rot=40, layout="interleaved", scaling="linear"),
        # Four whole prompts of different lengths.
        dict(name="append_bf16_4x4096", kind="append", dtype="bf16", seqs=4, idle=0, pad=0, new=4096, ragged=True,
             held=0, Hq=32, Hk=8, d=128, page=64, by_token=False, rot=128, layout="half", scaling="none"),
        # A single conversation: one token over a short cache.
        dict(name="attend_bf16_1x1", kind="attend", dtype="bf16", seqs=1, idle=0, pad=0, new=1, ragged=False,
             held=1000, Hq=32, Hk=8, d=128, page=64, by_token=False, form="step"),
        # A full batch of conversations of very different lengths, the batch
        # padded to a fixed number of rows.
        dict(name="attend_bf16_64x1", kind="attend", dtype="bf16", seqs=64, idle=3, pad=3, new=1, ragged=False,
             held=32768, Hq=32, Hk=8, d=128, page=64, by_token=False, form="step"),
        # Trees of 48 drafted tokens being verified.
        dict(name="attend_bf16_8x48_tree", kind="attend", dtype="bf16", seqs=8, idle=0, pad=0, new=48, ragged=False,
             held=16384, Hq=32, Hk=8, d=128, page=64, by_token=False, form="tree"),
        # The same in fp32, a model of odd sizes without shared heads.
        dict(name="attend_f32_6x13_tree", kind="attend", dtype="f32", seqs=6, idle=1, pad=5, new=13, ragged=True,
             held=2901, Hq=12, Hk=12, d=80, page=16, by_token=True, form="tree"),
        # A piece of a long prompt for two sequences.
        dict(name="attend_bf16_2x2048_prompt", kind="attend", dtype="bf16", seqs=2, idle=0, pad=0, new=2048,
             ragged=False, held=32000, Hq=32, Hk=8, d=128, page=64, by_token=False, form="prompt"),
        # After verifying: the accepted path of each tree.
        dict(name="keep_bf16_64x6of48", kind="keep", dtype="bf16", seqs=64, held=4000, new=48, kept=6, Hk=8, d=128,
             page=64, by_token=False),
        dict(name="keep_f32_5x4of13", kind="keep", dtype="f32", seqs=5, held=901, new=13, kept=4, Hk=12, d=80,
             page=16, by_token=True),
        # The next token of a few sequences, logits as the bf16 product leaves them.
        dict(name="rules_bf16_4x32000", kind="rules", dtype="bf16", rows=4, vocab=32000, history=2000, bias="shared",
             mask=True, penalties=True),
        # A full batch with a large vocabulary, every rule at once.
        dict(name="rules_f32_256x131072", kind="rules", dtype="f32", rows=256, vocab=131072, history=8192,
             bias="shared", mask=True, penalties=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "keep", "rules", "rules"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "rules":
        vocab = _log_int(rng, 256, 131072)
        vocab = vocab if rng.random() < 0.4 else max(256, vocab // 64 * 64)
        return dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, min(256, 2 ** 25 // vocab)), vocab=vocab,
                    history=rng.choice([0, _log_int(rng, 1, 32768)]), bias=rng.choice(["none", "shared", "rows"]),
                    mask=rng.random() < 0.6, penalties=rng.random() < 0.8)
    Hk = rng.choice([1, 2, 4, 8, 12])
    d = rng.choice([64, 80, 96, 128, 128, 128, 160, 256])
    case = dict(kind=kind, dtype=dtype, Hk=Hk, d=d, page=rng.choice([1, 8, 16, 32, 64, 128, 256]),
                by_token=rng.random() < 0.5)
    row = Hk * d * (2 if dtype == "bf16" else 4)  # bytes of a token's keys
    if kind == "keep":
        kept = rng.randint(1, 12)
        return dict(case, seqs=_log_int(rng, 1, 128), held=_log_int(rng, 1, 4000), new=kept * rng.randint(2, 8),
                    kept=kept)
    case.update(Hq=Hk * rng.choice([1, 2, 4, 6, 8]), idle=rng.choice([0, 0, 1, 2]), pad=rng.choice([0, 0, 1, 9]),
                ragged=rng.random() < 0.5)
    if kind == "append":
        form = rng.choice(["step", "piece"])
        seqs = _log_int(rng, 1, 256) if form == "step" else rng.randint(1, 8)
        top = max(2, min(4096, 2 ** 25 // (seqs * row)))
        return dict(case, seqs=seqs + case["idle"], new=1 if form == "step" else _log_int(rng, 2, top),
                    held=rng.choice([0, _log_int(rng, 1, max(2, min(16384, 2 ** 29 // (seqs * row))))]),
                    rot=rng.choice([d, d, d // 2]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "parts"]))
    form = rng.choice(["step", "step", "tree", "prompt"])
    seqs = {"step": _log_int(rng, 1, 128), "tree": _log_int(rng, 1, 32), "prompt": rng.randint(1, 4)}[form]
    # a GiB of keys at most, and no more products than the largest listed case
    pairs = (2 ** 36 if dtype == "bf16" else 2 ** 34) // (seqs * case["Hq"] * d)
    new = {"step": 1, "tree": rng.randint(2, 64),
           "prompt": _log_int(rng, 33, max(64, min(2048, int(math.sqrt(pairs)))))}[form]
    top = min(2 ** 30 // (seqs * row), pairs // new)
    held = rng.choice([0, 1, 1, 1]) * _log_int(rng, 1, max(2, min(65536, top)))
    return dict(case, seqs=seqs + case["idle"], new=new, held=held, form=form)


def _spread(n, lo, hi):
    """n whole numbers between lo and hi, even over their logarithm, in no order."""
    if hi <= lo:
        return [hi] * n
    step = (math.sqrt(5.0) - 1.0) / 2.0
    f = [((i + 1) * step) % 1.0 for i in range(n)]
    return [max(lo, min(hi, int(round(max(lo, 1) * (hi / max(lo, 1)) ** x)))) for x in f]


def _sizes(case):
    """Tokens held and new of each sequence; idle ones come last."""
    n, idle = case["seqs"], case.get("idle", 0)
    held = _spread(n, case["held"] // 64, case["held"])
    new = _spread(n, max(1, case["new"] // 4), case["new"]) if case.get("ragged") else [case["new"]] * n
    return held, [0 if i >= n - idle else new[i] for i in range(n)]


# ------------------------------------------------------------------ inputs


class _Inputs:
    """Seeded draws on the GPU; the same (seed, order) gives the same values."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=dtype).mul_(std)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=self.g, device="cuda").mul_(hi - lo).add_(lo)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}
BASE = 10000.0
# frequency scaling: (factor, context trained on, low and high turns, magnitude)
_SCALING = {"none": (1.0, 0, 0.0, 0.0, 1.0), "linear": (4.0, 0, 0.0, 0.0, 1.0), "parts": (16.0, 8192, 1.0, 32.0, 1.25)}


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _tree(r, seqs, n):
    """Which drafted tokens each drafted token sees (its ancestors and itself),
    bool [seqs, n, n], and its depth: every token's parent is one of the eight
    before it."""
    back = r.uniform(seqs, n)
    sees = torch.zeros(seqs, n, n, dtype=torch.bool, device="cuda")
    depth = torch.zeros(seqs, n, dtype=torch.int32, device="cuda")
    row = torch.arange(seqs, device="cuda")
    sees[:, 0, 0] = True
    for i in range(1, n):
        parent = i - 1 - (back[:, i] * min(i, 8)).long().clamp(max=min(i, 8) - 1)
        sees[:, i] = sees[row, parent]
        sees[:, i, i] = True
        depth[:, i] = depth[row, parent] + 1
    return sees, depth


def _bits(mask):
    """bool [rows, n] as 32-bit words, the lowest bit first."""
    rows, n = mask.shape
    words = (n + 31) // 32
    m = torch.nn.functional.pad(mask, (0, words * 32 - n)).reshape(rows, words, 32).to(torch.int64)
    v = (m << torch.arange(32, device="cuda")).sum(dim=2)
    return torch.where(v >= 2 ** 31, v - 2 ** 32, v).to(torch.int32)


def _cache(r, case, held, new):
    """A pool whose pages lie in any order, some of them nobody's, and the table."""
    Hk, d, page, dt = case["Hk"], case["d"], case["page"], _TORCH[case["dtype"]]
    need = [(a + b + page - 1) // page for a, b in zip(held, new)]
    pages = sum(need) + 3
    shape = (pages, page, Hk, d) if case["by_token"] else (pages, Hk, page, d)
    t = dict(k_cache=r.normal(*shape, dtype=dt), v_cache=r.normal(*shape, dtype=dt))
    order, width, at = r.order(pages), max(max(need), 1), 0
    t["table"] = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    for s, n in enumerate(need):
        t["table"][s, :n] = order[at:at + n]
        at += n
    t["held"] = _int32(held)
    return t


def _inputs(case, seed):
    """The tensors a pass reads, by name."""
    r, k, dt = _Inputs(seed), case["kind"], _TORCH[case["dtype"]]
    if k == "rules":
        rows, vocab = case["rows"], case["vocab"]
        t = dict(x=r.normal(rows, vocab, std=3.0, dtype=dt))
        lengths = _spread(rows, case["history"] // 16, case["history"])
        # what a model writes repeats itself: half of a history is of 200 tokens
        often, n = r.ints(0, vocab, 200), sum(lengths)
        t["history"] = torch.where(r.uniform(n) < 0.5, often[r.ints(0, 200, n).long()], r.ints(0, vocab, n))
        t["starts"], t["prompt"] = _int32(_starts(lengths)), _int32([i // 2 for i in lengths])
        if case["penalties"]:
            t["repetition"] = r.uniform(rows, lo=1.0, hi=1.5)
            t["presence"], t["frequency"] = r.uniform(rows, lo=-0.5, hi=1.0), r.uniform(rows, lo=0.0, hi=0.5)
        if case["bias"] != "none":
            n = 1 if case["bias"] == "shared" else rows
            t["bias"] = torch.where(r.uniform(n, vocab) < 0.01, r.normal(n, vocab, std=5.0), 0.0)
        if case["mask"]:
            t["mask"] = r.ints(-2 ** 31, 2 ** 31 - 1, rows, (vocab + 31) // 32)
        return t
    if k == "keep":
        held = _spread(case["seqs"], case["held"] // 64, case["held"])
        new, kept = [case["new"]] * case["seqs"], case["kept"]
        t = _cache(r, case, held, new)
        # the root, and then a path behind the first `kept` tokens of a wide tree
        pick = torch.rand(case["seqs"], case["new"] - kept, generator=r.g, device="cuda").argsort(dim=1)[:, :kept - 1]
        root = torch.zeros(case["seqs"], 1, dtype=torch.long, device="cuda")
        t["kept"] = torch.cat([root, (pick + kept).sort(dim=1).values], dim=1).to(torch.int32)
        counts = [max(1, kept - i % 3) for i in range(case["seqs"])]
        t["counts"] = _int32(counts)
        return t
    held, new = _sizes(case)
    t = _cache(r, case, held, new)
    T, Hq, Hk, d = sum(new) + case["pad"], case["Hq"], case["Hk"], case["d"]
    t["starts"] = _int32(_starts(new))
    if k == "append":  # q, k and v side by side, as the fused projection leaves them
        qkv = r.normal(T, Hq + 2 * Hk, d, dtype=dt)
        t.update(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hk], v=qkv[:, Hq + Hk:])
        return t
    # queries that look for something: scores of a few units
    t["q"] = r.normal(T, Hq, d, std=2.5, dtype=dt)
    if case["form"] == "tree":
        n = case["new"]
        sees, _ = _tree(r, case["seqs"], n)
        rows = [sees[s, :m] for s, m in enumerate(new)]
        rows.append(torch.zeros(case["pad"], n, dtype=torch.bool, device="cuda"))
        t["mask"] = _bits(torch.cat(rows))
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    st = dict(case=case, t=t)
    k, dt = case["kind"], _TORCH[case["dtype"]]
    if k in ("append", "attend"):
        st["held"], st["new"] = _sizes(case)
    elif k == "keep":
        st["kept"] = t["counts"].tolist()
    if not own:
        return st
    bwpp = _bwpp()
    st["be"] = _backend()
    code = int(bwpp.DType.BF16 if case["dtype"] == "bf16" else bwpp.DType.F32)
    new = lambda *s, dtype=dt: torch.zeros(*s, dtype=dtype, device="cuda")
    if k == "rules":
        st["out"] = dict(y=new(case["rows"], case["vocab"], dtype=torch.float32))
        st["p"] = bwpp.LogitRulesParams(rows=case["rows"], vocab=case["vocab"], dtype_x=code,
                                        history=t["history"].numel(),
                                        ld_bias=case["vocab"] if case["bias"] == "rows" else 0,
                                        ld_mask=(case["vocab"] + 31) // 32)
        return st
    kc, Hk, d = t["k_cache"], case["Hk"], case["d"]
    token, head = (1, 2) if case["by_token"] else (2, 1)
    cache = bwpp.CacheParams(pages=kc.shape[0], page_tokens=case["page"], heads=Hk, dim=d, batch=case["seqs"],
                             max_pages=t["table"].shape[1], dtype=code, page_stride=kc.stride(0),
                             token_stride=kc.stride(token), head_stride=kc.stride(head))
    if k == "keep":
        st["p"] = bwpp.CacheKeepParams(cache=cache, max_kept=case["kept"])
        return st
    q, Hq = t["q"], case["Hq"]
    cache.tokens, cache.q_heads = q.shape[0], Hq
    st["out"] = dict(o=new(q.shape[0], Hq, d))
    if k == "attend":
        st["out"]["lse"] = new(q.shape[0], Hq, dtype=torch.float32)
        st["p"] = bwpp.CacheAttentionParams(cache=cache, scale=d ** -0.5,
                                            mask_words=t["mask"].shape[1] if "mask" in t else 0)
        return st
    factor, context, low, high, magnitude = _SCALING[case["scaling"]]
    scaling = dict(none=bwpp.RotaryScaling.NONE, linear=bwpp.RotaryScaling.LINEAR,
                   parts=bwpp.RotaryScaling.BY_PARTS)[case["scaling"]]
    layout = bwpp.RotaryLayout.HALF if case["layout"] == "half" else bwpp.RotaryLayout.INTERLEAVED
    st["p"] = bwpp.CacheAppendParams(cache=cache, ldq=q.stride(0), ldk=t["k"].stride(0), ldv=t["v"].stride(0),
                                     rot_dim=case["rot"], layout=int(layout), base=BASE, scaling=int(scaling),
                                     factor=factor, context=context, low_turns=low, high_turns=high,
                                     magnitude=magnitude)
    return st


# --------------------------------------------------------------- one pass


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    be, t, p, k = st["be"], st["t"], st["p"], st["case"]["kind"]
    if k == "rules":
        be.dispatch_logit_rules(t["x"], t["history"], t["starts"], t["prompt"], t.get("repetition"), t.get("presence"),
                                t.get("frequency"), t.get("bias"), t.get("mask"), st["out"]["y"], p)
        return st["out"]
    if k == "keep":
        be.dispatch_cache_keep(t["k_cache"], t["v_cache"], t["table"], t["held"], t["kept"], t["counts"], p)
        return dict(k_cache=t["k_cache"], v_cache=t["v_cache"])
    if k == "attend":
        be.dispatch_cache_attention(t["q"], t["k_cache"], t["v_cache"], t["table"], t["starts"], t["held"],
                                    t.get("mask"), st["out"]["o"], st["out"]["lse"], p)
        return st["out"]
    be.dispatch_cache_append(t["q"], t["k"], t["v"], None, t["table"], t["starts"], t["held"], st["out"]["o"],
                             t["k_cache"], t["v_cache"], p)
    return dict(q=st["out"]["o"], k_cache=t["k_cache"], v_cache=t["v_cache"])


def _turn(case, x, positions):
    """x [T, H, d] in 32 bits with rotary positions; the angles in 64 bits, since
    far positions lose them in 32."""
    n = case["rot"]
    f = BASE ** (-torch.arange(0, n, 2, device="cuda", dtype=torch.float64) / n)
    factor, context, low, high, magnitude = _SCALING[case["scaling"]]
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "parts":
        c = ((context * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * (c + (1.0 - c) / factor)
    a = positions.double()[:, None, None] * f
    cos, sin = (a.cos() * magnitude).float(), (a.sin() * magnitude).float()
    if case["layout"] == "half":
        u, v = x[..., :n // 2], x[..., n // 2:n]
        y = torch.cat([u * cos - v * sin, v * cos + u * sin], dim=-1)
    else:
        u, v = x[..., 0:n:2], x[..., 1:n:2]
        y = torch.stack([u * cos - v * sin, v * cos + u * sin], dim=-1).flatten(-2)
    return torch.cat([y, x[..., n:]], dim=-1)


def _places(case, t, st):
    """For every new token: its row, its page and its place in the page."""
    T = sum(st["new"])
    row = torch.arange(T, device="cuda")
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), _int32(st["new"]).long(), output_size=T)
    slot = t["held"].long()[seq] + row - t["starts"].long()[seq]
    return slot, t["table"].long()[seq, slot // case["page"]], slot % case["page"]


def _put(case, cache, page, at, rows):
    if case["by_token"]:
        cache[page, at] = rows
    else:
        cache[page, :, at] = rows


def _sequence(case, t, name, s, length):
    """Keys or values [Hk, length, d] of sequence s, out of their pages."""
    pages = t["table"][s, :(length + case["page"] - 1) // case["page"]].long()
    rows = t[name][pages]
    rows = rows.permute(2, 0, 1, 3) if case["by_token"] else rows.permute(1, 0, 2, 3)
    return rows.reshape(case["Hk"], -1, case["d"])[:, :length]


def _visible(case, t, first, n):
    """bool [n, n]: which of its sequence's new tokens each new token sees."""
    if case["form"] != "tree":
        return torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    words = t["mask"][first:first + n].long()
    j = torch.arange(n, device="cuda")
    return (words[:, j // 32] >> (j % 32)) & 1 != 0


def _run_plain(st):
    case, t = st["case"], st["t"]
    k, dt = case["kind"], _TORCH[case["dtype"]]
    if k == "rules":
        z, rows, n = t["x"].float(), case["rows"], t["history"].numel()
        if case["penalties"] and n:
            seq = torch.searchsorted(t["starts"][1:], torch.arange(n, device="cuda", dtype=torch.int32), right=True)
            written = torch.arange(n, device="cuda") - t["starts"].long()[seq] >= t["prompt"][seq]
            at = seq * case["vocab"] + t["history"]
            count = torch.zeros(z.numel(), device="cuda").index_add_(0, at, written.float()).view_as(z)
            seen = torch.zeros(z.numel(), dtype=torch.bool, device="cuda")
            seen[at] = True
            rho = t["repetition"][:, None]
            z = torch.where(seen.view_as(z), torch.where(z > 0, z / rho, z * rho), z)
            z = z - (t["frequency"][:, None] * count + t["presence"][:, None] * (count > 0))
        if "bias" in t:
            z = z + t["bias"]
        if "mask" in t:
            j = torch.arange(case["vocab"], device="cuda")
            z = torch.where((t["mask"][:, j // 32] >> (j % 32).int()) & 1 != 0, z, -math.inf)
        return dict(y=z)
    if k == "keep":
        page = case["page"]
        i = torch.arange(case["kept"], device="cuda")[None, :]
        live = i < t["counts"][:, None]
        seq = torch.arange(case["seqs"], device="cuda")[:, None].expand_as(live)[live]
        to, frm = (t["held"][:, None] + i)[live].long(), (t["held"][:, None] + t["kept"])[live].long()
        for name in ("k_cache", "v_cache"):
            c, a, b = t[name], t["table"].long()[seq, frm // page], t["table"].long()[seq, to // page]
            rows = c[a, frm % page] if case["by_token"] else c[a, :, frm % page]
            _put(case, c, b, to % page, rows)
        return dict(k_cache=t["k_cache"], v_cache=t["v_cache"])
    if k == "append":
        slot, page, at = _places(case, t, st)
        T = slot.numel()
        q = torch.zeros(t["q"].shape, dtype=dt, device="cuda")
        q[:T] = _turn(case, t["q"][:T].float(), slot).to(dt)
        _put(case, t["k_cache"], page, at, _turn(case, t["k"][:T].float(), slot).to(dt))
        _put(case, t["v_cache"], page, at, t["v"][:T])
        return dict(q=q, k_cache=t["k_cache"], v_cache=t["v_cache"])
    o = torch.zeros(t["q"].shape, dtype=dt, device="cuda")
    lse = torch.zeros(t["q"].shape[:2], device="cuda")
    first, Hk, d = 0, case["Hk"], case["d"]
    for s, (held, n) in enumerate(zip(st["held"], st["new"])):
        if n == 0:
            continue
        keys, values = (_sequence(case, t, c, s, held + n).float() for c in ("k_cache", "v_cache"))
        q = t["q"][first:first + n].float().reshape(n, Hk, -1, d).transpose(0, 1)  # [Hk, n, group, d]
        g = q.shape[2]
        z = (q.reshape(Hk, n * g, d) @ keys.transpose(1, 2)).mul_(d ** -0.5).view(Hk, n, g, held + n)
        z[..., held:].masked_fill_(~_visible(case, t, first, n)[None, :, None, :], -math.inf)
        top = z.max(dim=-1, keepdim=True).values
        z = z.sub_(top).exp_()
        total = z.sum(dim=-1, keepdim=True)
        out = (z.view(Hk, n * g, -1) @ values).view(Hk, n, g, d) / total
        o[first:first + n] = out.transpose(0, 1).reshape(n, Hk * g, d).to(dt)
        lse[first:first + n] = (top + total.log())[..., 0].transpose(0, 1).reshape(n, Hk * g)
        first += n
    return dict(o=o, lse=lse)


# ------------------------------------------------------- what it must cost


def work(case):
    k, e = case["kind"], _BYTES[case["dtype"]]
    if k == "rules":
        n = case["rows"] * case["vocab"]
        small = 4 * sum(_spread(case["rows"], case["history"] // 16, case["history"]))
        if case["bias"] != "none":
            small += 4 * case["vocab"] * (case["rows"] if case["bias"] == "rows" else 1)
        if case["mask"]:
            small += 4 * case["rows"] * ((case["vocab"] + 31) // 32)
        return dict(bytes=n * (e + 4) + small, flops=5 * n)
    row = case["Hk"] * case["d"] * e
    if k == "keep":
        moved = sum(max(1, case["kept"] - i % 3) - 1 for i in range(case["seqs"]))
        return dict(bytes=4 * row * moved + 12 * case["seqs"], flops=0)
    held, new = _sizes(case)
    T, qrow = sum(new), case["Hq"] * case["d"] * e
    if k == "append":
        return dict(bytes=2 * T * (qrow + 2 * row) + 8 * T,
                    flops=T * ((case["Hq"] + case["Hk"]) * 3 * case["rot"] + 10 * case["rot"]))
    keys = sum(a + n for a, n in zip(held, new) if n)
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(held, new))
    return dict(bytes=2 * keys * row + 2 * T * qrow + 4 * T * case["Hq"], flops=4.0 * pairs * case["Hq"] * case["d"])


# -------------------------------------------------- the same in 64 bits


def exact(case, seed):
    t = _inputs(case, seed)
    k = case["kind"]
    if k == "rules":
        z = t["x"].double()
        starts, prompt = t["starts"].tolist(), t["prompt"].tolist()
        for r in range(case["rows"]):
            if case["penalties"]:
                past = t["history"][starts[r]:starts[r + 1]].long()
                said = torch.bincount(past[prompt[r]:], minlength=case["vocab"]).double()
                any_ = torch.bincount(past, minlength=case["vocab"]) > 0
                rho = t["repetition"][r].double()
                z[r] = torch.where(any_, torch.minimum(z[r] * rho, z[r] / rho), z[r])  # rho >= 1: always downwards
                z[r] -= said * t["frequency"][r].double() + (said > 0) * t["presence"][r].double()
            if "bias" in t:
                z[r] += t["bias"][r if case["bias"] == "rows" else 0].double()
        if "mask" in t:
            bit = (t["mask"][:, :, None].long() >> torch.arange(32, device="cuda")) % 2
            z[bit.flatten(1)[:, :case["vocab"]] == 0] = -math.inf
        return dict(y=z)
    token_at = lambda c, page, at: c[page, at] if case["by_token"] else c[page, :, at]
    kc, vc = t["k_cache"].double(), t["v_cache"].double()
    if k == "keep":
        new = [kc.clone(), vc.clone()]
        table, held = t["table"].tolist(), t["held"].tolist()
        for s, (kept, n) in enumerate(zip(t["kept"].tolist(), t["counts"].tolist())):
            for i in range(n):
                a, b = held[s] + kept[i], held[s] + i
                pa, pb = table[s][a // case["page"]], table[s][b // case["page"]]
                for old, c in zip((kc, vc), new):
                    token_at(c, pb, b % case["page"])[...] = token_at(old, pa, a % case["page"])
        return dict(k_cache=new[0], v_cache=new[1])
    held, new = _sizes(case)
    if k == "append":
        n = case["rot"]
        i = torch.arange(n // 2, device="cuda", dtype=torch.float64)
        f = torch.exp(-(2.0 * i / n) * math.log(BASE))
        factor, context, low, high, magnitude = _SCALING[case["scaling"]]
        if case["scaling"] == "linear":
            f = f / factor
        if case["scaling"] == "parts":
            kept = torch.clamp((context * f / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
            f = kept * f + (1.0 - kept) * (f / factor)

        def turned(x, pos):  # a pair as a complex number, turned by e^(i p f)
            a = pos[:, None] * f
            turn = torch.polar(torch.full_like(a, magnitude), a)[:, None, :]
            v = x.double().clone()
            if case["layout"] == "half":
                z = torch.complex(v[..., :n // 2].contiguous(), v[..., n // 2:n].contiguous()) * turn
                v[..., :n // 2], v[..., n // 2:n] = z.real, z.imag
            else:
                z = torch.complex(v[..., 0:n:2].contiguous(), v[..., 1:n:2].contiguous()) * turn
                v[..., 0:n:2], v[..., 1:n:2] = z.real, z.imag
            return v

        q, first = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda"), 0
        for s, m in enumerate(new):
            if m == 0:
                continue
            pos = torch.arange(held[s], held[s] + m, device="cuda")
            rows = slice(first, first + m)
            q[rows] = turned(t["q"][rows], pos.double())
            pages = t["table"][s].long()[torch.div(pos, case["page"], rounding_mode="floor")]
            at = torch.remainder(pos, case["page"])
            _put(case, kc, pages, at, turned(t["k"][rows], pos.double()))
            _put(case, vc, pages, at, t["v"][rows].double())
            first += m
        return dict(q=q, k_cache=kc, v_cache=vc)
    Hk, d, first = case["Hk"], case["d"], 0
    g = case["Hq"] // Hk
    o = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(t["q"].shape[:2], dtype=torch.float64, device="cuda")
    for s, m in enumerate(new):
        if m == 0:
            continue
        pos = torch.arange(held[s] + m, device="cuda")
        pages, at = t["table"][s].long()[pos // case["page"]], pos % case["page"]
        unseen = torch.ones(m, m, dtype=torch.bool, device="cuda").triu(1)
        if case["form"] == "tree":
            bit = (t["mask"][first:first + m, :, None].long() >> torch.arange(32, device="cuda")) % 2
            unseen = bit.flatten(1)[:, :m] == 0
        for h in range(Hk):
            keys, values = (c[pages, at, h] if case["by_token"] else c[pages, h, at] for c in (kc, vc))
            q = t["q"][first:first + m, h * g:(h + 1) * g].double()
            z = (q.reshape(m * g, d) @ keys.t() / math.sqrt(d)).view(m, g, -1)
            z[:, :, held[s]:] = z[:, :, held[s]:].masked_fill(unseen[:, None, :], -math.inf)
            l = torch.logsumexp(z, dim=2)
            lse[first:first + m, h * g:(h + 1) * g] = l
            o[first:first + m, h * g:(h + 1) * g] = (z.sub_(l[:, :, None]).exp_().view(m * g, -1) @ values).view(m, g, d)
        first += m
    return dict(o=o, lse=lse)

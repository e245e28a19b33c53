"""A paged key-value cache of a language model in the framework's exact integer arithmetic, as timed cases.

  plan     block tables and slot maps from request lengths
  rows     keys and values of tokens quantised into pages at their slots, and read back
  attend   attention of one new token a sequence over the cache
  select   beam search's selection over beams and vocabulary
  reorder  beam search's reordering: block tables and lengths by parent, partly filled pages copied

Values are Q16 integers (65536 stands for 1.0); q e means q * 2^e. Every output is a whole number and has to be equal.
Where `own` is false, run() computes in elementary torch operations (64-bit integers, and products in float64, where every
partial sum is a whole number below 2^53); where it is true, it calls the framework.
"""
from __future__ import annotations

import math

import torch

own = False

ONE = 65536                    # 1.0 of the Q16 values
DEV = "cuda"
SPAN = 256                     # positions of the cache whose weights share a maximum
VSPAN = 4096                   # entries of the vocabulary that do
LOW = -(1 << 31)               # a logit that bans its token
NONE = -(1 << 63)              # the score of a beam that is not there


def _up(v, a):
    return (v + a - 1) // a * a


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one decode step of sixteen sequences: the smallest call
        {"name": "plan_16x1", "kind": "plan", "R": 16, "most": 1, "ctx": 4000, "page": 16},
        # a batch of prompts of ragged lengths behind cached prefixes, large pages
        {"name": "plan_300x400", "kind": "plan", "R": 300, "most": 400, "ctx": 8000, "page": 64},
        # keys and values of a decode step's 24 sequences, one token each, 8 bits
        {"name": "rows_24x8x128", "kind": "rows", "M": 24, "heads": 8, "D": 128, "bits": 8, "page": 16, "run": 1},
        # those of a prompt, 16 bits
        {"name": "rows_5000x8x128", "kind": "rows", "M": 5000, "heads": 8, "D": 128, "bits": 16, "page": 64, "run": 5000},
        # one short sequence of a small model, every head its own keys, 16 bits: latency
        {"name": "attend_1x500", "kind": "attend", "R": 1, "most": 500, "Hq": 16, "heads": 16, "D": 64, "bits": 16, "page": 16, "window": 0, "even": True},
        # a serving batch of ragged lengths, four queries a key, some slots idle
        {"name": "attend_37x4096", "kind": "attend", "R": 37, "most": 4096, "Hq": 32, "heads": 8, "D": 128, "bits": 8, "page": 16, "window": 0, "even": False},
        # two documents of 131072 tokens: few rows, a long axis
        {"name": "attend_2x131072", "kind": "attend", "R": 2, "most": 131072, "Hq": 32, "heads": 8, "D": 128, "bits": 8, "page": 64, "window": 0, "even": True},
        # a sliding window, six queries a key, heads of an odd size
        {"name": "attend_16x9000w", "kind": "attend", "R": 16, "most": 9000, "Hq": 12, "heads": 2, "D": 96, "bits": 16, "page": 32, "window": 1024, "even": False},
        # four beams of one request; twice as many candidates as beams, so that ended ones can be taken out
        {"name": "select_1x4x32000", "kind": "select", "G": 1, "beams": 4, "V": 32000, "n": 8},
        # a batch of requests over a large vocabulary of an odd size
        {"name": "select_40x5x100003", "kind": "select", "G": 40, "beams": 5, "V": 100003, "n": 10},
        # four beams of one request
        {"name": "reorder_1x4", "kind": "reorder", "R": 4, "beams": 4, "ctx": 1000, "heads": 8, "D": 128, "bits": 8, "page": 16},
        # a batch of requests of eight beams, large pages, 16 bits
        {"name": "reorder_48x8", "kind": "reorder", "R": 384, "beams": 8, "ctx": 2000, "heads": 8, "D": 128, "bits": 16, "page": 64},
    ]


def _log(rng, lo, hi, step=1):
    """A whole multiple of `step` between lo and hi, even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step))


def draw(rng):
    kind = rng.choice(["plan", "rows", "attend", "attend", "attend", "select", "reorder"])
    page, bits = rng.choice([16, 32, 64, 128, 256]), rng.choice([8, 16])
    if kind == "plan":
        while True:
            R, most = _log(rng, 1, 2048), _log(rng, 1, 4096)
            if R * most <= 300 * 400:
                return {"kind": kind, "R": R, "most": most, "ctx": _log(rng, 16, 8000), "page": page}
    if kind == "rows":
        while True:
            M, heads, D = _log(rng, 1, 8192), _log(rng, 1, 32), rng.choice([16, 64, 80, 96, 128, 192, 256])
            if M * heads * D <= 5000 * 8 * 128:
                return {"kind": kind, "M": M, "heads": heads, "D": D, "bits": bits, "page": page, "run": rng.choice([1, M, _log(rng, 1, M)])}
    if kind == "attend":
        while True:
            R, most, heads, D = _log(rng, 1, 128), _log(rng, 1, 131072), _log(rng, 1, 32), rng.choice([16, 64, 80, 96, 128, 192, 256])
            group = rng.choice([1, 1, 2, 4, 5, 8, 16, 24])
            if heads * group <= 128 and R * most * heads * D * bits <= 2 * 131072 * 8 * 128 * 8 and R * most * heads * group <= 2 * 131072 * 32:
                return {"kind": kind, "R": R, "most": most, "Hq": heads * group, "heads": heads, "D": D, "bits": bits, "page": page,
                        "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]), "even": rng.random() < 0.3}
    if kind == "select":
        while True:
            G, beams, V = _log(rng, 1, 64), rng.randint(1, 16), _log(rng, 1000, 200000)
            if G * beams * V <= 40 * 5 * 100003:
                return {"kind": kind, "G": G, "beams": beams, "V": V, "n": rng.choice([beams, 2 * beams])}
    while True:
        beams = rng.randint(1, 16)
        R, heads, D = beams * _log(rng, 1, 64), _log(rng, 1, 16), rng.choice([64, 96, 128])
        if R <= 384 and R * heads * D * page * bits <= 384 * 8 * 128 * 64 * 16:
            return {"kind": kind, "R": R, "beams": beams, "ctx": _log(rng, 16, 2000), "heads": heads, "D": D, "bits": bits, "page": page}


# ---------------------------------------------------------------- inputs

class Draws:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)

    def ints(self, shape, lo, hi, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV, dtype=dtype)

    def heads(self, M, H, D, scale=ONE):
        """Q16 rows [M, H, D] whose size varies from row to row, with a few loud channels."""
        x = torch.randn((M, H, D), generator=self.g, device=DEV)
        x *= torch.exp(0.4 * torch.randn((M, H, 1), generator=self.g, device=DEV)) * scale
        x *= torch.exp(0.4 * torch.randn((1, H, D), generator=self.g, device=DEV))
        return x.round_().to(torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=DEV).to(torch.int32)

    def lengths(self, R, most, even):
        """Lengths from 0 to `most`, spread over their logarithm, in any order; all near `most` where `even`."""
        x = (1 + self.order(R)).double() / R
        n = most * (1 - (1 - x) / 50) if even else (1 + most) ** ((R * x - 1) / (R - 1) if R > 1 else x) - 1
        return n.round().to(torch.int32)


def tables(d, n, page, width, spare=0):
    """Block tables [R, width] of n tokens each, pages in random order, -1 behind them; the pages not used, and how many there are."""
    need = (n + page - 1) // page
    total = int(need.sum())
    pages = d.order(total + spare)
    at = torch.cumsum(need, 0) - need
    j = torch.arange(width, device=DEV)
    t = torch.where(j < need[:, None], pages[(at[:, None] + j).clamp(max=total + spare - 1)], -1).to(torch.int32)
    return t.contiguous(), pages[total:].contiguous(), total + spare


def scale_of(D):
    """m 2^-s = 2^-16 / sqrt(D): what turns a product of two Q16 rows into a Q16 score."""
    s = 15 + 16 + int(math.log2(math.sqrt(D)))
    return round(2.0**(s - 16) / math.sqrt(D)), s


def inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    d = Draws(seed)
    P = case.get("page")
    if case["kind"] == "plan":
        R = case["R"]
        n = d.lengths(R, case["ctx"], False)
        add = torch.ones_like(n) if case["most"] == 1 else d.lengths(R, case["most"], False)
        width = (case["ctx"] + case["most"] + P - 1) // P
        table, free, pages = tables(d, n, P, width, R * (case["most"] // P + 2))
        tokens = _up(int(add.sum()), 8)                        # the token rows a batch is padded to
        return {"len": n, "add": add, "table": table, "free": free, "nfree": torch.tensor([free.numel()], dtype=torch.int32, device=DEV),
                "pages": pages, "width": width, "tokens": tokens}
    if case["kind"] == "rows":
        M, H, D = case["M"], case["heads"], case["D"]
        k, v = d.heads(M, H, D), d.heads(M, H, D)
        run = case["run"]                                      # tokens of one sequence, one after the other from some place on
        seqs = (M + run - 1) // run
        per = (run + P - 1) // P + 1
        first = d.ints((seqs,), 0, P).to(torch.int64) if run < M or run == 1 else torch.zeros((seqs,), dtype=torch.int64, device=DEV)
        own_pages = d.order(seqs * per).reshape(seqs, per).to(torch.int64)
        t = torch.arange(M, device=DEV)
        pos = first[t // run] + t % run
        slot = (own_pages[t // run, pos // P] * P + pos % P).to(torch.int32)
        slot[d.ints((M,), 0, 24) == 0] = -1                    # rows of a padded batch, written nowhere
        return {"k": k.reshape(M, H * D), "v": v.reshape(M, H * D), "slot": slot, "pages": seqs * per}
    if case["kind"] == "attend":
        R, H, D = case["R"], case["heads"], case["D"]
        n = d.lengths(R, case["most"], case["even"])
        table, _, pages = tables(d, n, P, (case["most"] + P - 1) // P)
        kv = d.heads(pages * P, H, D), d.heads(pages * P, H, D)
        return {"q": d.heads(R, case["Hq"], D, 2 * ONE).reshape(R, -1), "len": n, "table": table, "pages": pages, "k": kv[0], "v": kv[1], "lexp": exp_table()}
    if case["kind"] == "select":
        rows, V = case["G"] * case["beams"], case["V"]
        z = torch.randn((rows, V), generator=d.g, device=DEV) * (2.5 * ONE)
        z = z.round_().to(torch.int32)
        z[:, d.ints((7,), 0, V).to(torch.int64)] = LOW         # tokens that may not follow
        score = -d.ints((rows,), 0, 40 * ONE).to(torch.int64)
        score[d.ints((rows,), 0, 16) == 0] = NONE              # beams that have ended
        score[:: case["beams"]] = -ONE
        return {"z": z, "score": score, "lexp": exp_table(), "lln": ln_table()}
    R, B = case["R"], case["beams"]
    n = d.lengths(R // B, case["ctx"], False).repeat_interleave(B)
    width = (case["ctx"] + P - 1) // P
    table, fresh, pages = tables(d, n, P, width, R)
    parent = (torch.arange(R, device=DEV) // B * B + d.ints((R,), 0, B)).to(torch.int32)
    words = case["heads"] * case["D"] * P * 2 * case["bits"] // 32
    return {"parent": parent, "len": n, "table": table, "fresh": fresh, "pages": pages, "width": width,
            "kv": d.ints((pages, words), LOW, 1 << 31), "sh": d.ints((pages, P * case["heads"] // 2), LOW, 1 << 31)}


def exp_table():
    """exp(-i / 64) with 2^30 for 1, as the attention's table."""
    return (torch.exp(-torch.arange(1025, dtype=torch.float64) / 64) * 2.0**30).round().to(torch.int64).to(DEV)


def ln_table():
    """ln(1 + i / 1024) with 2^30 for 1."""
    return (torch.log1p(torch.arange(1025, dtype=torch.float64) / 1024) * 2.0**30).round().to(torch.int64).to(DEV)


# ---------------------------------------------------------------- what a program has in hand

def new(shape, dt=torch.int32):
    return torch.empty(shape, dtype=dt, device=DEV)


def prepare(case, seed):
    s = inputs(case, seed)
    s["case"] = case
    kind, P = case["kind"], case.get("page")
    if kind == "attend" and not own:
        s["k"], s["ek"] = quant(s["k"], case["bits"])           # the cache as plain rows, [slots, heads, D] with shifts
        s["v"], s["ev"] = quant(s["v"], case["bits"])
    if not own:
        return s
    from vela_amd import beam as vb
    from vela_amd import gemm as vg
    from vela_amd import kv as vk
    if kind == "plan":
        R = case["R"]
        s.update(new_len=new(R), start=new(R + 1), slot=new(s["tokens"]), pos=new(s["tokens"]), used=new(1))
        s["P"] = vk.KvPlan(R=R, tokens=s["tokens"], pages=s["pages"], page=P, width=s["width"], ldt=s["width"], len=vg.ptr(s["len"]), add=vg.ptr(s["add"]),
                           table=vg.ptr(s["table"]), free=vg.ptr(s["free"]), nfree=vg.ptr(s["nfree"]), new_len=vg.ptr(s["new_len"]), start=vg.ptr(s["start"]),
                           slot=vg.ptr(s["slot"]), pos=vg.ptr(s["pos"]), used=vg.ptr(s["used"]))
    elif kind == "rows":
        s["cache"] = vk.KvCache(s["pages"], P, case["heads"], case["D"], case["bits"])
        s["ko"], s["vo"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    elif kind == "attend":
        R, H, D, Hq = case["R"], case["heads"], case["D"], case["Hq"]
        s["cache"] = vk.KvCache(s["pages"], P, H, D, case["bits"])
        slots = torch.arange(s["pages"] * P, dtype=torch.int32, device=DEV)
        vk.k_kv_write(s["cache"], s.pop("k"), s.pop("v"), H * D, slots, slots.numel())
        nb = vk.kv_attention_workspace_bytes(R, Hq, D, case["most"])
        s.update(out=new((R, Hq * D)), rowmax=new(R), ws=new(max(nb, 16) // 4))
        m, sh = scale_of(D)
        s["A"] = vk.KvAttn(Q=vg.ptr(s["q"]), ldq=Hq * D, rows=R, Hq=Hq, table=vg.ptr(s["table"]), ldt=s["table"].shape[1], width=s["table"].shape[1],
                           len=vg.ptr(s["len"]), max_len=case["most"], window=case["window"], m=m, s=sh, Lexp=vg.ptr(s["lexp"]), out=vg.ptr(s["out"]),
                           ldo=Hq * D, rowmax=vg.ptr(s["rowmax"]), ws=vg.ptr(s["ws"]), ws_bytes=nb)
    elif kind == "select":
        G, n = case["G"], case["n"]
        nb = vb.beam_workspace_bytes(G, case["beams"], case["V"], n)
        s.update(oscore=new((G, n), torch.int64), parent=new((G, n)), token=new((G, n)), ws=new(nb // 4))
        s["B"] = vb.BeamSelect(groups=G, beams=case["beams"], V=case["V"], n=n, logits=vg.ptr(s["z"]), ldz=case["V"], score=vg.ptr(s["score"]),
                               Lexp=vg.ptr(s["lexp"]), Lln=vg.ptr(s["lln"]), out_score=vg.ptr(s["oscore"]), parent=vg.ptr(s["parent"]), token=vg.ptr(s["token"]),
                               ws=vg.ptr(s["ws"]), ws_bytes=nb)
    else:
        R = case["R"]
        s["cache"] = vk.KvCache(s["pages"], P, case["heads"], case["D"], case["bits"])
        s["cache"].data.view(torch.int32).copy_(s["kv"].reshape(-1))
        s["cache"].shift.view(torch.int32).copy_(s["sh"].reshape(-1))
        s.update(otable=new((R, s["width"])), olen=new(R), src=new(R), dst=new(R))
        s["T"] = vb.BeamTables(rows=R, page=P, width=s["width"], ldt=s["width"], parent=vg.ptr(s["parent"]), len=vg.ptr(s["len"]), table=vg.ptr(s["table"]),
                               fresh=vg.ptr(s["fresh"]), out_len=vg.ptr(s["olen"]), out_table=vg.ptr(s["otable"]), src=vg.ptr(s["src"]), dst=vg.ptr(s["dst"]))
    return s


# ---------------------------------------------------------------- the plain form

def sat32(v):
    return v.clamp(-(1 << 31), (1 << 31) - 1)


def bits_over(m, base):
    """How many powers of two from 2^base on (up to 2^31) m reaches: the shift to `base` bits."""
    e = torch.zeros_like(m)
    for i in range(base, 32):
        e += m >= 1 << i
    return e


def shift_round(v, s):
    """v 2^-s rounded half up, s >= 0."""
    return (v + ((torch.ones_like(s) << s) >> 1)) >> s


def quant(x, bits):
    """Rows [.., D] in `bits` bits: q (int16) and the shift of each row."""
    top = (1 << bits - 1) - 1
    e = bits_over(x.abs().amax(-1).to(torch.int64), bits - 1)
    q = torch.empty(x.shape, dtype=torch.int16, device=x.device)
    for i in range(0, x.shape[0], 65536):                       # in parts: 64 bits a value at a time
        q[i:i + 65536] = shift_round(x[i:i + 65536].to(torch.int64), e[i:i + 65536, ..., None]).clamp(-top, top)
    return q, e


def between(lexp, d):
    """The exp table at d >= 0 in Q16, 0 from 16 on."""
    c = d.clamp(max=16 * ONE - 1)
    i, f = c >> 10, c & 1023
    return torch.where(d >= 16 * ONE, 0, lexp[i] + (((lexp[i + 1] - lexp[i]) * f) >> 10))


def whole_div(a, b):
    return torch.div(a + (b >> 1), b, rounding_mode="floor")


def plain_plan(s):
    case, P, W = s["case"], s["case"]["page"], s["width"]
    n, add = s["len"].to(torch.int64), s["add"].to(torch.int64)
    R = n.numel()
    have, need = (n + P - 1) // P, ((n + add + P - 1) // P).clamp(max=W)
    more = (need - have).clamp(min=0)
    at = torch.cumsum(more, 0) - more
    j = torch.arange(W, device=DEV)
    i = at[:, None] + j - have[:, None]
    nf = s["nfree"].to(torch.int64)
    fresh = torch.where(i < nf, s["free"].to(torch.int64)[i.clamp(0, s["free"].numel() - 1)], -1)
    table = torch.where((j >= have[:, None]) & (j < (have + more)[:, None]), fresh, s["table"].to(torch.int64))
    start = torch.zeros(R + 1, dtype=torch.int64, device=DEV)
    start[1:] = torch.cumsum(add, 0)
    t = torch.arange(s["tokens"], device=DEV)
    r = (torch.searchsorted(start, t, right=True) - 1).clamp(max=R - 1)
    pos = n[r] + t - start[r]
    page = table[r, (pos // P).clamp(max=W - 1)]
    ok = (t < start[R]) & (pos < W * P) & (page >= 0) & (page < s["pages"])
    to = lambda v: v.to(torch.int32)  # noqa: E731
    return {"table": to(table), "len": to(n + add), "start": to(start), "slot": to(torch.where(ok, page * P + pos % P, -1)),
            "pos": to(torch.where(t < start[R], pos, -1)), "used": to(more.sum().reshape(1))}


def plain_rows(s):
    case = s["case"]
    out = []
    for x in (s["k"], s["v"]):
        q, e = quant(x.reshape(case["M"], case["heads"], case["D"]), case["bits"])
        cache = torch.zeros((s["pages"] * case["page"], *q.shape[1:]), dtype=torch.int16, device=DEV)
        shift = torch.zeros(cache.shape[:2], dtype=torch.int64, device=DEV)
        at, there = s["slot"].to(torch.int64), s["slot"] >= 0
        cache[at[there]], shift[at[there]] = q[there], e[there]
        back = cache[at.clamp(min=0)].to(torch.int64) << shift[at.clamp(min=0)][..., None]
        out.append(torch.where(there[:, None, None], back, 0).reshape(case["M"], -1).to(torch.int32))
    return {"k": out[0], "v": out[1]}


def plain_attend(s):
    case = s["case"]
    R, H, D, P = case["R"], case["heads"], case["D"], case["page"]
    group = case["Hq"] // H
    m, sh = scale_of(D)
    lexp = s["lexp"]
    out = torch.zeros((R, H, group, D), dtype=torch.int64, device=DEV)
    x = s["q"].to(torch.int64).reshape(R, H, group, D)
    eq = bits_over(x.abs().amax(-1), 14)
    q = shift_round(x, eq[..., None])
    for r, n in enumerate(s["len"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        j = torch.arange(first // SPAN * SPAN, _up(n, SPAN), device=DEV)              # whole spans
        ok = (j >= first) & (j < n)
        slot = s["table"][r].to(torch.int64)[(j // P).clamp(max=s["table"].shape[1] - 1)] * P + j % P
        slot = torch.where(ok, slot, 0)
        k = s["k"][slot].permute(1, 2, 0).double().contiguous()                      # [H, D, T]
        S = torch.matmul(q[r].double(), k).to(torch.int64)                           # [H, group, T]
        score = sat32(shift_round(S * m, sh - eq[r][..., None] - s["ek"][slot].t()[:, None]))
        score = score.reshape(H, group, -1, SPAN)
        ok = ok.reshape(-1, SPAN)
        mx = torch.where(ok, score, -(1 << 40)).amax(-1)                             # [H, group, U]
        p = torch.where(ok, (((between(lexp, (mx[..., None] - score).clamp(min=0)) + (1 << 14)) >> 15).clamp(max=32767)), 0)
        L = p.sum(-1)
        v = (s["v"][slot].to(torch.int64) << s["ev"][slot][..., None]).double().reshape(-1, SPAN, H, D).permute(2, 0, 1, 3).contiguous()   # [H, U, SPAN, D]
        O = torch.matmul(p.permute(0, 2, 1, 3).double().contiguous(), v).to(torch.int64)                                                # [H, U, group, D]
        A = whole_div(O, L.transpose(1, 2)[..., None])
        G = ((between(lexp, mx.amax(-1, keepdim=True) - mx) + (1 << 6)) >> 7) * L
        down = bits_over64(G.sum(-1, keepdim=True), 30)
        g = (G + ((torch.ones_like(down) << down) >> 1)) >> down
        out[r] = whole_div((A * g.transpose(1, 2)[..., None]).sum(1), g.sum(-1)[..., None])
    out = out.reshape(R, -1)
    return {"out": out.to(torch.int32), "rowmax": out.abs().amax(1).clamp(max=(1 << 31) - 1).to(torch.int32)}


def bits_over64(m, base):
    e = torch.zeros_like(m)
    for i in range(base, 63):
        e += m >= 1 << i
    return e


def plain_select(s):
    case = s["case"]
    G, B, V, n = case["G"], case["beams"], case["V"], case["n"]
    z = s["z"].to(torch.int64)
    off = s["z"] == LOW
    pad = _up(V, VSPAN) - V
    zs = torch.nn.functional.pad(z, (0, pad), value=LOW).reshape(G * B, -1, VSPAN)
    mxc = zs.amax(-1)
    S = torch.where(zs == LOW, 0, between(s["lexp"], mxc[..., None] - zs)).sum(-1)
    mx = mxc.amax(-1, keepdim=True)
    S = ((between(s["lexp"], mx - mxc) * ((S + (1 << 11)) >> 12) + (1 << 17)) >> 18).sum(-1, keepdim=True).clamp(min=1)
    top = bits_over64(S, 1)                                     # floor(log2 S)
    f = (torch.where(top >= 30, S >> (top - 30).clamp(min=0), S << (30 - top).clamp(min=0))) - (1 << 30)
    i, fr = f >> 20, f & ((1 << 20) - 1)
    lln = s["lln"]
    logz = ((top - 30) * lln[1024] + lln[i] + (((lln[i + 1] - lln[i]) * fr) >> 20) + (1 << 13)) >> 14
    c = s["score"][:, None] + z - mx - logz
    c = torch.where(off | (s["score"][:, None] == NONE), NONE, c).reshape(G, B * V)
    # equal ones by their place: a stable sort of the few that reach the n-th largest value of all
    least = torch.topk(c, n, dim=1).values[:, -1:]
    score, parent, token = (torch.full((G, n), v, dtype=torch.int64, device=DEV) for v in (NONE, -1, -1))
    for g in range(G):
        at = torch.nonzero((c[g] >= least[g]) & (c[g] > NONE))[:, 0]
        o = torch.sort(c[g, at], descending=True, stable=True).indices[:n]
        k = o.numel()
        score[g, :k], parent[g, :k], token[g, :k] = c[g, at[o]], g * B + at[o] // V, at[o] % V
    return {"score": score, "parent": parent.to(torch.int32), "token": token.to(torch.int32)}


def plain_reorder(s):
    P, W = s["case"]["page"], s["width"]
    p = s["parent"].to(torch.int64)
    n = s["len"][p].to(torch.int64)
    j = torch.arange(W, device=DEV)
    old = s["table"][p].to(torch.int64)
    part = n % P != 0
    last = (n // P).clamp(max=W - 1)
    table = torch.where(j < ((n + P - 1) // P)[:, None], old, -1)
    table = torch.where(part[:, None] & (j == (n // P)[:, None]), s["fresh"].to(torch.int64)[:, None], table)
    src = torch.where(part, old.gather(1, last[:, None])[:, 0], -1)
    dst = torch.where(part, s["fresh"].to(torch.int64), -1)
    s["kv"][dst[part]], s["sh"][dst[part]] = s["kv"][src[part]], s["sh"][src[part]]
    to = lambda v: v.to(torch.int32)  # noqa: E731
    return {"table": to(table), "len": to(n), "src": to(src), "dst": to(dst), "kv": s["kv"], "sh": s["sh"]}


# ---------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    if not own:
        return {"plan": plain_plan, "rows": plain_rows, "attend": plain_attend, "select": plain_select, "reorder": plain_reorder}[case["kind"]](s)
    from vela_amd import beam as vb
    from vela_amd import gemm as vg
    from vela_amd import kv as vk
    if case["kind"] == "plan":
        vk.k_kv_plan(s["P"])
        return {"table": s["table"], "len": s["new_len"], "start": s["start"], "slot": s["slot"], "pos": s["pos"], "used": s["used"]}
    if case["kind"] == "rows":
        ld = case["heads"] * case["D"]
        vk.k_kv_write(s["cache"], s["k"], s["v"], ld, s["slot"], case["M"])
        vk.k_kv_read(s["cache"], s["slot"], case["M"], s["ko"], s["vo"], ld)
        return {"k": s["ko"], "v": s["vo"]}
    if case["kind"] == "attend":
        vg.fill_u32(s["rowmax"])                               # row maxima are gathered onto the caller's zeros
        vk.k_kv_attention(s["cache"], s["A"])
        return {"out": s["out"], "rowmax": s["rowmax"]}
    if case["kind"] == "select":
        vb.k_beam_select(s["B"])
        return {"score": s["oscore"], "parent": s["parent"], "token": s["token"]}
    vb.k_beam_tables(s["T"])
    vk.k_kv_copy(s["cache"], s["src"], s["dst"], case["R"])
    return {"table": s["otable"], "len": s["olen"], "src": s["src"], "dst": s["dst"],
            "kv": s["cache"].data.view(torch.int32).view(s["pages"], -1), "sh": s["cache"].shift.view(torch.int32).view(s["pages"], -1)}


def work(case):
    kind, P = case["kind"], case.get("page")
    ragged = lambda most: most if most <= 1 else (most / math.log(1 + most) - 1)  # noqa: E731  the mean of the ragged lengths
    if kind == "plan":
        tokens = case["R"] * ragged(case["most"])
        # lengths in and out, the new table entries and the free list's, two words a token
        return {"bytes": 16.0 * case["R"] + 8 * tokens / P + 8 * tokens, "flops": 4.0 * tokens}
    if kind == "rows":
        n = 2.0 * case["M"] * case["heads"] * case["D"]
        # int32 rows read, written to the pages, read from them, int32 rows written
        return {"bytes": n * (8 + 2 * case["bits"] / 8), "flops": 4 * n}
    if kind == "attend":
        most = case["most"]
        n = most * 0.99 if case["even"] else (most + (case["R"] - 1) * ragged(most)) / case["R"]
        if case["window"]:
            n = min(n, case["window"])
        keys = case["R"] * n
        return {"bytes": keys * case["heads"] * (2 * case["D"] * case["bits"] / 8 + 2) + 8.0 * case["R"] * case["Hq"] * case["D"] + 4 * keys / P,
                "flops": 4.0 * keys * case["Hq"] * case["D"]}
    if kind == "select":
        return {"bytes": 4.0 * case["G"] * case["beams"] * case["V"] + 16 * case["G"] * case["n"], "flops": 4.0 * case["G"] * case["beams"] * case["V"]}
    n = case["R"] * ragged(case["ctx"])
    # a page and its shifts a row, read and written; the tables' entries likewise
    page = case["heads"] * P * (2 * case["D"] * case["bits"] / 8 + 2)
    return {"bytes": 2.0 * case["R"] * page * (P - 1) / P + 8 * n / P + 8 * case["R"], "flops": 1.0 * case["R"] * page}


# ---------------------------------------------------------------- the definition, in 64-bit integers

def x_len(v, bits):
    """The least e >= 0 with v < 2^(bits + e), v a list of Python integers."""
    return [max(0, int(m).bit_length() - bits) for m in v]


def x_exp(lexp, d):
    inside = (d >= 0) & (d < 1048576)
    i = torch.where(inside, torch.div(d, 1024, rounding_mode="floor"), 0)
    lo, hi = lexp[i], lexp[i + 1]
    return torch.where(inside, lo + torch.div((hi - lo) * (d - 1024 * i), 1024, rounding_mode="floor"), 0)


def x_near(a, b):
    """a / b to the nearest whole number, halves up, b > 0."""
    return torch.div(2 * a + b, 2 * b, rounding_mode="floor")


def x_round(v, s):
    """floor(v / 2^s + 1/2) of 64-bit integers; s a tensor of whole numbers >= 0."""
    p = torch.ones_like(v) << s.expand_as(v)
    return torch.where(s > 0, torch.div(v + torch.div(p, 2, rounding_mode="floor"), p, rounding_mode="floor"), v)


def x_quant(x, bits):
    """Rows [M, D] in `bits` bits and their shifts."""
    e = torch.tensor(x_len(x.abs().max(1).values.tolist(), bits - 1), device=DEV)[:, None]
    top = 2 ** (bits - 1) - 1
    return x_round(x, e).clamp(-top, top), e


def x_attend(case, s):
    R, H, D, P = case["R"], case["heads"], case["D"], case["page"]
    group = case["Hq"] // H
    m, sh = scale_of(D)
    out = torch.zeros((R, case["Hq"] * D), dtype=torch.int64, device=DEV)
    n = s["len"].tolist()
    for r in range(R):
        first = n[r] - min(n[r], case["window"] or n[r])
        if n[r] == 0:
            continue
        j = torch.arange(first, n[r], device=DEV)
        slot = s["table"][r, torch.div(j, P, rounding_mode="floor")].to(torch.int64) * P + j % P
        for h in range(H):
            k, ek = x_quant(s["k"][slot, h].to(torch.int64), case["bits"])
            v, ev = x_quant(s["v"][slot, h].to(torch.int64), case["bits"])
            v = v * (1 << ev)
            for a in range(group):
                at = (h * group + a) * D
                x = s["q"][r, at:at + D].to(torch.int64)
                eq = x_len([int(x.abs().max())], 14)[0]
                q = x_round(x, torch.full((1,), eq, device=DEV))
                z = x_round((k * q).sum(1) * m, sh - eq - ek[:, 0])
                means, weights, tops = [], [], []
                for b in range(first // SPAN * SPAN, n[r], SPAN):
                    i = slice(max(b, first) - first, min(b + SPAN, n[r]) - first)
                    top = z[i].max()
                    w = torch.div(x_exp(s["lexp"], top - z[i]) + 16384, 32768, rounding_mode="floor").clamp(max=32767)
                    means.append(x_near((w[:, None] * v[i]).sum(0), w.sum()))
                    weights.append(w.sum())
                    tops.append(top)
                tops, weights = torch.stack(tops), torch.stack(weights)
                G = torch.div(x_exp(s["lexp"], tops.max() - tops) + 64, 128, rounding_mode="floor") * weights
                down = x_len([int(G.sum())], 30)[0]
                g = x_round(G, torch.full((1,), down, device=DEV))
                out[r, at:at + D] = x_near((g[:, None] * torch.stack(means)).sum(0), g.sum())
    return {"out": out, "rowmax": out.abs().max(1).values}


def exact(case, seed):
    kind, P = case["kind"], case.get("page")
    if kind == "attend":
        if case["R"] * case["Hq"] * (min(case["most"], case["window"] or case["most"]) / SPAN + 4) > 40000:
            return None                                        # head by head and span by span: too long
        return x_attend(case, inputs(case, seed))
    s = inputs(case, seed)
    if kind == "plan":
        n, add, table, free = s["len"].tolist(), s["add"].tolist(), s["table"].tolist(), s["free"].tolist()
        start, slot, pos, used = [0], [-1] * s["tokens"], [-1] * s["tokens"], 0
        for r in range(case["R"]):
            for i in range(add[r]):
                at = n[r] + i
                if at % P == 0 and at // P < s["width"]:       # the first token of a new page
                    table[r][at // P] = free[used] if used < len(free) else -1
                    used += 1
                t = start[r] + i
                pos[t] = at
                if at // P < s["width"] and 0 <= table[r][at // P] < s["pages"]:
                    slot[t] = table[r][at // P] * P + at % P
            start.append(start[r] + add[r])
        return {"table": torch.tensor(table), "len": torch.tensor(n) + torch.tensor(add), "start": torch.tensor(start), "slot": torch.tensor(slot),
                "pos": torch.tensor(pos), "used": torch.tensor([used])}
    if kind == "rows":
        M, out = case["M"], {}
        for name in ("k", "v"):
            q, e = x_quant(s[name].to(torch.int64).reshape(M * case["heads"], case["D"]), case["bits"])
            out[name] = (q * (1 << e)).reshape(M, -1) * (s["slot"] >= 0)[:, None]
        return out
    if kind == "select":
        B, V, lln = case["beams"], case["V"], s["lln"].tolist()
        score, parent, token = [], [], []
        for g in range(case["G"]):
            best = []
            for row in range(g * B, g * B + B):
                if int(s["score"][row]) == NONE:
                    continue
                z = s["z"][row].to(torch.int64)
                live = torch.nonzero(z > LOW)[:, 0]
                parts = []
                for b in range(0, V, VSPAN):
                    part = z[b:b + VSPAN]
                    part = part[part > LOW]
                    if part.numel():
                        parts.append((int(part.max()), int(x_exp(s["lexp"], part.max() - part).sum())))
                mx = max(p[0] for p in parts)
                S = max(1, sum((int(x_exp(s["lexp"], torch.tensor(mx - a, device=DEV))) * ((b + 2048) // 4096) + 131072) // 262144 for a, b in parts))
                top = S.bit_length() - 1
                f = (S * 2**30 >> top) - 2**30
                i, fr = f >> 20, f % 1048576
                logz = ((top - 30) * lln[1024] + lln[i] + (((lln[i + 1] - lln[i]) * fr) >> 20) + 8192) >> 14
                c = z[live] + (int(s["score"][row]) - mx - logz)
                keep = torch.sort(c, descending=True, stable=True).indices[:case["n"]]
                best += [(-v, row, t) for v, t in zip(c[keep].tolist(), live[keep].tolist())]
            best = sorted(best)[:case["n"]]
            best += [(-NONE, -1, -1)] * (case["n"] - len(best))
            score.append([-b[0] for b in best])
            parent.append([b[1] for b in best])
            token.append([b[2] for b in best])
        return {"score": torch.tensor(score), "parent": torch.tensor(parent), "token": torch.tensor(token)}
    n, table, fresh = s["len"].tolist(), s["table"].tolist(), s["fresh"].tolist()
    rows, src, dst = [], [], []
    for r, p in enumerate(s["parent"].tolist()):
        full, part = divmod(n[p], P)
        row = table[p][:full] + ([fresh[r]] if part else [])
        rows.append(row + [-1] * (s["width"] - len(row)))
        src.append(table[p][full] if part else -1)
        dst.append(fresh[r] if part else -1)
        if part:
            s["kv"][fresh[r]], s["sh"][fresh[r]] = s["kv"][table[p][full]], s["sh"][table[p][full]]
    return {"table": torch.tensor(rows), "len": torch.tensor([n[p] for p in s["parent"].tolist()]), "src": torch.tensor(src), "dst": torch.tensor(dst),
            "kv": s["kv"], "sh": s["sh"]}

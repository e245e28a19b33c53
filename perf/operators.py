"""Operators of a language model's decode step in the framework's exact integer arithmetic, as timed cases.

  norm   residual addition, root-mean-square norm and 8-bit rows with a shift per row
  w4     a product of few rows with 4-bit weights, group scales and zero points
  moe    a mixture-of-experts layer for few tokens: router, the chosen experts' 4-bit feed-forward, combination

Values are Q16 integers (65536 stands for 1.0); q e means q * 2^e. Every output is a whole number and has to be equal.
Where `own` is false, run() computes in elementary torch operations (64-bit integers, and products in float64, where every
partial sum is a whole number below 2^53); where it is true, it calls the framework.
"""
from __future__ import annotations

import math

import torch

own = False

ONE = 65536                    # 1.0 of the Q16 values
EPS_DEN = 100000               # 1 / epsilon of the norm
DEV = "cuda"


def _up(v, a):
    return (v + a - 1) // a * a


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # the norm before a layer's products while one token is decoded: the smallest call
        {"name": "norm_1x2048", "kind": "norm", "M": 1, "C": 2048},
        # the same for a batch of 37 sequences, one token each, in a wide model
        {"name": "norm_37x5120", "kind": "norm", "M": 37, "C": 5120},
        # the norm over a prompt of 4096 tokens
        {"name": "norm_4096x4096", "kind": "norm", "M": 4096, "C": 4096},
        # one token through a square projection of a small model
        {"name": "w4_1x2048x2048", "kind": "w4", "M": 1, "K": 2048, "N": 2048, "group": 128, "src": "q8", "epi": "plain", "res": True},
        # one token through a merged query, key and value projection; 16-bit rows
        {"name": "w4_1x4096x12288", "kind": "w4", "M": 1, "K": 4096, "N": 12288, "group": 64, "src": "q16", "epi": "plain", "res": False},
        # sixteen sequences through a gated up-projection, with the row maxima that the next product reads
        {"name": "w4_geglu_16x4096x22016", "kind": "w4", "M": 16, "K": 4096, "N": 22016, "group": 128, "src": "q8", "epi": "geglu", "res": False},
        # the down-projection behind it for five sequences: int32 rows quantised from their maxima, residual
        {"name": "w4_down_5x11008x4096", "kind": "w4", "M": 5, "K": 11008, "N": 4096, "group": 128, "src": "x32", "epi": "plain", "res": True},
        # drafted tokens of many sequences, fine groups, sizes off every tile
        {"name": "w4_51x2600x9999", "kind": "w4", "M": 51, "K": 2600, "N": 9999, "group": 32, "src": "q16", "epi": "plain", "res": False},
        # one token through a layer of eight experts, two chosen
        {"name": "moe_1_8x2", "kind": "moe", "M": 1, "experts": 8, "topk": 2, "D": 1024, "F": 2048, "group": 128, "renorm": True},
        # four sequences, many narrow experts, six chosen
        {"name": "moe_4_64x6", "kind": "moe", "M": 4, "experts": 64, "topk": 6, "D": 2048, "F": 1408, "group": 128, "renorm": False},
        # sixteen sequences, 128 experts, eight chosen: most experts are read
        {"name": "moe_16_128x8", "kind": "moe", "M": 16, "experts": 128, "topk": 8, "D": 2048, "F": 768, "group": 64, "renorm": True},
        # more tokens than a tile of sixteen has rows, wide experts, fine groups
        {"name": "moe_43_8x2", "kind": "moe", "M": 43, "experts": 8, "topk": 2, "D": 2048, "F": 5504, "group": 32, "renorm": True},
    ]


def _log(rng, lo, hi, step=1):
    """A whole multiple of `step` between lo and hi, even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step))


def draw(rng):
    kind = rng.choice(["norm", "w4", "w4", "moe", "moe"])
    if kind == "norm":
        while True:
            M, C = _log(rng, 1, 4096), _log(rng, 256, 8192, 4)
            if M * C <= 4096 * 4096:
                return {"kind": kind, "M": M, "C": C}
    if kind == "w4":
        while True:
            M, K, N = _log(rng, 1, 64), _log(rng, 512, 11008, 4), _log(rng, 512, 22016)
            if K * N <= 4096 * 22016 and M * K * N <= 16 * 4096 * 22016:
                break
        epi = rng.choice(["plain", "plain", "geglu"])
        return {"kind": kind, "M": M, "K": K, "N": N // 2 * 2 if epi == "geglu" else N, "group": rng.choice([32, 64, 128]),
                "src": rng.choice(["q8", "q16", "x32"]), "epi": epi, "res": epi == "plain" and rng.random() < 0.5}
    while True:
        M, E, D, F = _log(rng, 1, 48), _log(rng, 4, 128), _log(rng, 512, 4096, 16), _log(rng, 256, 5504, 4)
        if E * D * F <= 128 * 2048 * 768 and M * D * F <= 16 * 2048 * 5504:
            return {"kind": kind, "M": M, "experts": E, "topk": rng.randint(1, min(8, E)), "D": D, "F": F,
                    "group": rng.choice([32, 64, 128]), "renorm": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs

class Draws:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)

    def ints(self, shape, lo, hi, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV, dtype=dtype)

    def rows(self, M, C, scale=ONE):
        """Q16 rows whose size varies from row to row, with a few loud channels."""
        x = torch.randn((M, C), generator=self.g, device=DEV)
        x *= torch.exp(0.3 * torch.randn((M, 1), generator=self.g, device=DEV))
        x *= torch.exp(0.4 * torch.randn((1, C), generator=self.g, device=DEV))
        return (x * scale).round().to(torch.int32)

    def q8(self, M, C, ld):
        """8-bit rows [M, ld] with their shifts, as the norm writes them (columns from C on hold 0)."""
        q = torch.zeros((M, ld), dtype=torch.int8, device=DEV)
        q[:, :C] = (torch.randn((M, C), generator=self.g, device=DEV) * 30).round().clamp(-127, 127).to(torch.int8)
        return q, self.ints((M,), 9, 13)

    def q16(self, M, C, ld):
        """16-bit rows as int8 planes, q = 256 hi + lo + 128, with their shifts."""
        q = torch.zeros((M, ld), dtype=torch.int32, device=DEV)
        q[:, :C] = (torch.randn((M, C), generator=self.g, device=DEV) * 7000).round().clamp(-32767, 32767).to(torch.int32)
        return (q >> 8).to(torch.int8), ((q & 255) - 128).to(torch.int8), self.ints((M,), 1, 5)

    def w4(self, N, K, group, qrms, count=None):
        """4-bit weights two a byte (even columns in the low half), group scales and zero points, and the columns' {m, s, b, 0}; the outputs keep the inputs' scale."""
        lead = () if count is None else (count,)
        groups = _up(K, group) // group
        nib = self.ints((*lead, N, (K + 1) // 2), 0, 256, torch.uint8)   # uniform codes: every value of the 4 bits
        if K % 2:
            nib[..., -1] &= 15
        sc = self.ints((*lead, N, groups), 800, 4096).to(torch.int16)
        z = self.ints((*lead, N, groups), 6, 11, torch.uint8)
        c = torch.zeros((*lead, N, 4), dtype=torch.int32, device=DEV)
        c[..., 0] = self.ints((*lead, N), 1 << 14, 1 << 15)
        c[..., 1] = round(math.log2(24000 * 4.8 * 2500 * math.sqrt(K)))
        c[..., 2] = self.ints((*lead, N), -5000, 5000)
        return nib, sc, z, c


def inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    d = Draws(seed)
    M = case["M"]
    if case["kind"] == "norm":
        C = case["C"]
        return {"x": d.rows(M, C, 2 * ONE), "r": d.rows(M, C, ONE), "g": d.ints((C,), 40000, 90000)}
    if case["kind"] == "w4":
        K, N = case["K"], case["N"]
        s = {}
        if case["src"] == "q8":
            s["hi"], s["e"] = d.q8(M, K, _up(K, 16))
        elif case["src"] == "q16":
            s["hi"], s["lo"], s["e"] = d.q16(M, K, _up(K, 16))
        else:
            s["x"] = d.rows(M, K)
            s["rowmax"] = s["x"].abs().amax(1).to(torch.int32)
        s["nib"], s["sc"], s["z"], s["cst"] = d.w4(N, K, case["group"], 30)
        if case["res"]:
            s["res"] = d.rows(M, N)
        if case["epi"] == "geglu":
            s["lut"] = gate_table()
        return s
    E, D, F = case["experts"], case["D"], case["F"]
    s = {"lut": gate_table(), "lexp": exp_table()}
    s["hi"], s["e"] = d.q8(M, D, D)
    s["rw"] = (torch.randn((E, D), generator=d.g, device=DEV) * 40).round().clamp(-127, 127).to(torch.int8)
    c = torch.zeros((E, 4), dtype=torch.int32, device=DEV)
    c[:, 0] = d.ints((E,), 1 << 14, 1 << 15)
    c[:, 1] = round(math.log2(24000 * 40 * math.sqrt(D))) - 1
    c[:, 2] = d.ints((E,), -20000, 20000)
    c[:, 3] = s["rw"].sum(1, dtype=torch.int32)
    s["rcst"] = c
    s["up"] = d.w4(2 * F, D, case["group"], 30, E)
    s["down"] = d.w4(D, F, case["group"], 7000, E)
    s["res"] = d.rows(M, D)
    return s


def gate_table():
    """The Q16 sigmoid over [-16, 16) in steps of 1/64: with it the gated product is a * (g sigmoid(g))."""
    x = (torch.arange(2049, dtype=torch.float64) - 1024) / 64
    return (65536 * torch.sigmoid(x)).round().to(torch.int32).to(DEV)


def exp_table():
    """exp(-i / 64) with 2^30 for 1, as the attention's table."""
    return (torch.exp(-torch.arange(1025, dtype=torch.float64) / 64) * 2.0**30).round().to(torch.int64).to(DEV)


# ---------------------------------------------------------------- what a program has in hand

def new(shape, dt=torch.int32):
    return torch.empty(shape, dtype=dt, device=DEV)


def prepare(case, seed):
    s = inputs(case, seed)
    s["case"] = case
    if own:                    # the weights laid out once, output buffers and argument blocks: a serving program keeps these
        from vela_amd import gemm as vg
        from vela_amd import moe as vm
        from vela_amd import w4 as vw
        M = case["M"]
        if case["kind"] == "norm":
            s["h"], s["q"], s["eq"] = new((M, case["C"])), new((M, case["C"]), torch.int8), new(M)
        elif case["kind"] == "w4":
            K, N, out = case["K"], case["N"], case["N"] // 2 if case["epi"] == "geglu" else case["N"]
            s["W"] = vw.W4Weights(N, K, case["group"])
            s["W"].pack(s["nib"], s["sc"], s["z"], s["cst"])
            s["y"] = new((M, out))
            if case["src"] == "x32":
                s["A"] = vg.ASrc(src=vg.SRC_X32, x=vg.ptr(s["x"]), ldx=K, rowmax=vg.ptr(s["rowmax"]), K=K)
            else:
                s["A"] = vg.ASrc(src=vg.SRC_I8, hi=vg.ptr(s["hi"]), lo=vg.ptr(s.get("lo")), ld8=_up(K, 16), e=vg.ptr(s["e"]), K=K)
            s["E"] = vg.AEpi(epi=vg.EPI_GEGLU if case["epi"] == "geglu" else vg.EPI_PLAIN, Y=vg.ptr(s["y"]), ldy=out, residual=vg.ptr(s.get("res")), Lphi=vg.ptr(s.get("lut")))
            if case["epi"] == "geglu":
                s["rm"] = new(M)
                s["E"].rowmax = vg.ptr(s["rm"])
        else:
            E, D, F, k = case["experts"], case["D"], case["F"], case["topk"]
            s["A"] = vg.ASrc(src=vg.SRC_I8, hi=vg.ptr(s["hi"]), ld8=D, e=vg.ptr(s["e"]), K=D)
            s["idx"], s["p"], s["y"] = new((M, k)), new((M, k)), new((M, D))
            s["R"] = vm.MoeRoute(W=vg.ptr(s["rw"]), ldw=D, cst=vg.ptr(s["rcst"]), experts=E, topk=k, renorm=int(case["renorm"]), Lexp=vg.ptr(s["lexp"]), idx=vg.ptr(s["idx"]), p=vg.ptr(s["p"]))
            s["U"], s["V"] = vw.W4Weights(2 * F, D, case["group"], count=E), vw.W4Weights(D, F, case["group"], count=E)
            for w, parts in ((s["U"], s["up"]), (s["V"], s["down"])):
                w.pack(*parts)
            s["ws"] = new(vm.moe_workspace_bytes(M, k, F) // 4)
            s["P"] = vm.MoeArgs(up=s["U"].desc, down=s["V"].desc, topk=k, idx=vg.ptr(s["idx"]), p=vg.ptr(s["p"]), Lphi=vg.ptr(s["lut"]), Y=vg.ptr(s["y"]), ldy=D,
                                residual=vg.ptr(s["res"]), ws=vg.ptr(s["ws"]), ws_bytes=s["ws"].numel() * 4)
    return s


# ---------------------------------------------------------------- the plain form

def sat32(v):
    return v.clamp(-(1 << 31), (1 << 31) - 1)


def shift_round(v, s):
    """v 2^-s rounded half up and saturated to 32 bits (s from 0 to 62; left shifts do not occur in these cases)."""
    return sat32((v + ((torch.ones_like(s) << s) >> 1)) >> s)


def bits_over(m, base):
    """How many powers of two from 2^base on (below 2^32) m reaches: the shift to `base` bits."""
    return (m[..., None] >= (1 << torch.arange(base, 32, device=m.device))).sum(-1)


def view16(y):
    """Rows in 16 bits: q, and the shift of each row."""
    e = bits_over(y.abs().amax(-1), 15)
    return shift_round(y, e[..., None]).clamp(-32767, 32767), e


def table16(x, lut):
    """The Q16 table between its points, 0 below -16 and 1 from 16 on."""
    z = x + 16 * ONE
    i, f = (z >> 10).clamp(0, 2047), z & 1023
    a, b = lut[i].to(torch.int64), lut[i + 1].to(torch.int64)
    return torch.where(z < 0, 0, torch.where(z >= 32 * ONE, ONE, a + (((b - a) * f) >> 10)))


def gated(y, lut):
    """a * (g table(g)) of interleaved columns (a, g)."""
    a, g = y[..., 0::2], y[..., 1::2]
    sixteen = torch.full_like(g, 16)
    return shift_round(a * shift_round(g * table16(g, lut), sixteen), sixteen)


def whole_weights(nib, sc, z, K, group):
    """(u - z) * scale, in float64 [..., N, K]."""
    u = torch.stack((nib & 15, nib >> 4), -1).flatten(-2)[..., :K].to(torch.int16)
    wide = lambda t: t.to(torch.int16).repeat_interleave(group, -1)[..., :K]  # noqa: E731
    return (u - wide(z)).double() * wide(sc).double()


def requant(acc, cst, e):
    """sat32(rshr(acc m, s - e) + b): acc whole numbers in float64, cst [..., N, 4], e [..., 1]."""
    c = cst.to(torch.int64)
    return sat32(shift_round(acc.to(torch.int64) * c[..., 0], c[..., 1] - e) + c[..., 2])


def plain_norm(s):
    h = sat32(s["x"].to(torch.int64) + s["r"].to(torch.int64))
    C = h.shape[1]
    ex = (bits_over(h.abs().amax(1), 15) - 5).clamp(min=0)[:, None]
    dev = shift_round(h, ex)
    var = (dev * dev).sum(1, keepdim=True) // C
    v = (var + ((torch.ones_like(ex) << (32 - 2 * ex)) + EPS_DEN // 2) // EPS_DEN) << 16
    sd = v.double().sqrt().to(torch.int64)
    sd = sd - (sd * sd > v).to(torch.int64)
    sd = sd + ((sd + 1) * (sd + 1) <= v).to(torch.int64)
    yy = torch.div((h << (25 - ex)) + sd, 2 * sd, rounding_mode="floor")
    y = shift_round(yy * s["g"].to(torch.int64), torch.full_like(ex, 16))
    e = bits_over(y.abs().amax(1), 7)
    q = shift_round(y, e[:, None]).clamp(-127, 127)
    return {"h": h.to(torch.int32), "q": (q << e[:, None]).to(torch.int32), "e": e.to(torch.int32)}


def plain_rows(s, case):
    """The rows' whole numbers (int64) and their shifts."""
    if case["kind"] == "w4" and case["src"] == "x32":
        return view16(s["x"].to(torch.int64))
    hi = s["hi"].to(torch.int64)[:, : case.get("K", case.get("D"))]
    if "lo" in s:
        hi = 256 * hi + s["lo"].to(torch.int64)[:, : case["K"]] + 128
    return hi, s["e"].to(torch.int64)


def plain_w4(s):
    case = s["case"]
    q, e = plain_rows(s, case)
    w = whole_weights(s["nib"], s["sc"], s["z"], case["K"], case["group"])
    y = requant(q.double() @ w.t(), s["cst"], e[:, None])
    if case["epi"] == "geglu":
        v = gated(y, s["lut"])
        return {"y": v.to(torch.int32), "rowmax": v.abs().amax(1).clamp(max=(1 << 31) - 1).to(torch.int32)}
    if case["res"]:
        y = sat32(y + s["res"].to(torch.int64))
    return {"y": y.to(torch.int32)}


def plain_route(s, case):
    """The experts of each token, the largest logits first (equal ones by their index), and their Q15 shares."""
    q, e = plain_rows(s, case)
    z = requant(q.double() @ s["rw"].double().t(), s["rcst"], e[:, None])
    order = torch.sort(z, dim=1, descending=True, stable=True)
    top, idx = order.values[:, : case["topk"]], order.indices[:, : case["topk"]]
    off = top[:, :1] - (top if case["renorm"] else z)
    share = lambda d: torch.where(d >= 16 * ONE, 0, between(s["lexp"], d.clamp(max=16 * ONE - 1)))  # noqa: E731
    total = share(off).sum(1, keepdim=True)
    r = torch.full_like(total, 1 << 62) // total
    p = ((share(top[:, :1] - top) * r + (1 << 46)) >> 47).clamp(max=32767)
    return idx, p


def between(lexp, d):
    i, f = d >> 10, d & 1023
    return lexp[i] + (((lexp[i + 1] - lexp[i]) * f) >> 10)


def plain_moe(s):
    case = s["case"]
    M, E, D, F = case["M"], case["experts"], case["D"], case["F"]
    idx, p = plain_route(s, case)
    q, e = plain_rows(s, case)
    up = whole_weights(*s["up"][:3], D, case["group"]).reshape(E * 2 * F, D)
    acc = (q.double() @ up.t()).reshape(M, E, 2 * F)
    v = gated(requant(acc, s["up"][3], e[:, None, None]), s["lut"])         # [M, E, F]: every expert for every token
    q2, e2 = view16(v)
    down = whole_weights(*s["down"][:3], F, case["group"]).transpose(1, 2).contiguous()
    y = requant(torch.matmul(q2.double().transpose(0, 1).contiguous(), down), s["down"][3][:, None], e2.t()[..., None])   # [E, M, D]
    y = y.transpose(0, 1).gather(1, idx[..., None].expand(-1, -1, D))       # the chosen ones, [M, topk, D]
    out = shift_round((y * p[..., None]).sum(1), torch.full((1, 1), 15, device=DEV))
    return {"y": sat32(out + s["res"].to(torch.int64)).to(torch.int32), "idx": idx.to(torch.int32), "p": p.to(torch.int32)}


# ---------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    if not own:
        return {"norm": plain_norm, "w4": plain_w4, "moe": plain_moe}[case["kind"]](s)
    from vela_amd import gemm as vg
    from vela_amd import moe as vm
    from vela_amd import norms as vn
    from vela_amd import w4 as vw
    if case["kind"] == "norm":
        vn.k_rmsnorm_q(s["x"], s["r"], case["M"], case["C"], s["g"], EPS_DEN, s["h"], s["q"], None, s["eq"], case["C"])
        return {"h": s["h"], "q": torch.bitwise_left_shift(s["q"], s["eq"][:, None]), "e": s["eq"]}   # 8 bits as the values they stand for
    if case["kind"] == "w4":
        if "rm" in s:
            vg.fill_u32(s["rm"])                   # row maxima are gathered onto the caller's zeros
        vw.k_gemm_w4(s["A"], case["M"], s["W"], s["E"])
        return {"y": s["y"], "rowmax": s["rm"]} if "rm" in s else {"y": s["y"]}
    vm.k_moe_route(s["A"], case["M"], s["R"])
    vm.k_moe(s["A"], case["M"], s["P"])
    return {"y": s["y"], "idx": s["idx"], "p": s["p"]}


def work(case):
    M = case["M"]
    if case["kind"] == "norm":
        C = case["C"]
        # rows and residual read, their sum and the 8-bit rows written; the weights once; a square, a sum and a scaling a value
        return {"bytes": 13.0 * M * C + 4 * C + 4 * M, "flops": 4.0 * M * C}
    g = case["group"]
    w4 = lambda n, k: n * k * 0.5 + 2.0 * n * (_up(k, g) // g) + 16 * n  # noqa: E731  4 bits each, 2 bytes of scale and zero point a group, 16 of requantisation a column
    if case["kind"] == "w4":
        K, N = case["K"], case["N"]
        rows = M * K * {"q8": 1, "q16": 2, "x32": 4}[case["src"]]
        out = 4 * M * (N // 2 if case["epi"] == "geglu" else N)
        return {"bytes": w4(N, K) + rows + out + (4 * M * N if case["res"] else 0), "flops": 2.0 * M * N * K}
    E, D, F, k = case["experts"], case["D"], case["F"], case["topk"]
    used = E * (1 - (1 - k / E) ** M)              # distinct experts of M tokens, on average
    return {"bytes": E * D + used * (w4(2 * F, D) + w4(D, F)) + M * D * 9, "flops": 2.0 * M * (E * D + k * 3 * F * D)}


# ---------------------------------------------------------------- the definition, in 64-bit integers

def x_round(v, s):
    """Rounding right shift by the definition floor(v / 2^s + 1/2), saturated; s a tensor or a number."""
    half = torch.where(torch.as_tensor(s, device=v.device) > 0, torch.ones_like(v) << (torch.as_tensor(s, device=v.device) - 1).clamp(min=0), 0)
    r = (v + half) >> s
    return torch.minimum(torch.maximum(r, torch.tensor(-2147483648, device=v.device)), torch.tensor(2147483647, device=v.device))


def x_shift(rows, bits):
    """Per row the least e >= 0 with every |value| below 2^(bits + e)."""
    return torch.tensor([max(0, int(m).bit_length() - bits) for m in rows.abs().max(-1).values.reshape(-1).tolist()], device=rows.device).reshape(rows.shape[:-1])


def x_codes(nib, K):
    out = torch.empty((*nib.shape[:-1], 2 * nib.shape[-1]), dtype=torch.int64, device=nib.device)
    out[..., 0::2], out[..., 1::2] = nib % 16, torch.div(nib, 16, rounding_mode="floor")
    return out[..., :K]


def x_product(q, parts, e, group):
    """One row of whole numbers q [K] against 4-bit weights [N, K]: group by group, then the columns' requantisation."""
    nib, sc, z, cst = parts
    K = q.shape[0]
    pad = _up(K, group) - K
    u = torch.nn.functional.pad(x_codes(nib, K), (0, pad)).reshape(nib.shape[0], -1, group)
    qg = torch.nn.functional.pad(q, (0, pad)).reshape(1, -1, group)
    part = (u * qg).sum(-1) - z.to(torch.int64) * qg.sum(-1)
    acc = (part * sc.to(torch.int64)).sum(-1)
    c = cst.to(torch.int64)
    return x_round(x_round(acc * c[:, 0], c[:, 1] - e) + c[:, 2], 0)


def x_gate(y, lut):
    a, g = y.reshape(-1, 2).unbind(1)
    pos = g + 1048576
    i = torch.div(pos, 1024, rounding_mode="floor")
    inside = (i >= 0) & (i < 2048)
    lo, hi = lut[i.clamp(0, 2047)].to(torch.int64), lut[i.clamp(0, 2047) + 1].to(torch.int64)
    t = lo + torch.div((hi - lo) * (pos - 1024 * i), 1024, rounding_mode="floor")
    t = torch.where(inside, t, torch.where(i < 0, 0, 65536))
    return x_round(a * x_round(g * t, 16), 16)


def exact(case, seed):
    s = inputs(case, seed)
    M = case["M"]
    if case["kind"] == "norm":
        h = x_round(s["x"].to(torch.int64) + s["r"], 0)
        ex = (x_shift(h, 15) - 5).clamp(min=0)
        dev = x_round(h, ex[:, None])
        ss = (dev * dev).sum(1).tolist()
        sd = torch.tensor([math.isqrt((ss[i] // case["C"] + ((1 << (32 - 2 * t)) + EPS_DEN // 2) // EPS_DEN) << 16) for i, t in enumerate(ex.tolist())], device=DEV)[:, None]
        top = h * (1 << (25 - ex))[:, None] + sd
        yy = torch.div(top - top % (2 * sd), 2 * sd, rounding_mode="trunc")
        y = x_round(yy * s["g"].to(torch.int64), 16)
        e = x_shift(y, 7)
        q = x_round(y, e[:, None]).clamp(-127, 127)
        return {"h": h, "q": q * (1 << e)[:, None], "e": e}
    if case["kind"] == "w4" and case["src"] == "x32":
        e = x_shift(s["x"].to(torch.int64), 15)
        q = x_round(s["x"].to(torch.int64), e[:, None]).clamp(-32767, 32767)
    else:
        q, e = s["hi"].to(torch.int64), s["e"].to(torch.int64)
        q = q * 256 + s["lo"] + 128 if "lo" in s else q
    if case["kind"] == "w4":
        y = torch.stack([x_product(q[t, : case["K"]], (s["nib"], s["sc"], s["z"], s["cst"]), e[t], case["group"]) for t in range(M)])
        if case["epi"] == "geglu":
            v = torch.stack([x_gate(y[t], s["lut"]) for t in range(M)])
            return {"y": v, "rowmax": v.abs().max(1).values.clamp(max=2147483647)}
        return {"y": x_round(y + s["res"], 0) if case["res"] else y}
    ys, ids, ps = [], [], []
    lexp = s["lexp"].tolist()
    share = lambda d: 0 if d >= 1048576 else lexp[d // 1024] + (lexp[d // 1024 + 1] - lexp[d // 1024]) * (d % 1024) // 1024  # noqa: E731
    for t in range(M):
        c = s["rcst"].to(torch.int64)
        z = x_round(x_round((s["rw"].to(torch.int64) * q[t]).sum(1) * c[:, 0], c[:, 1] - e[t]) + c[:, 2], 0).tolist()
        chosen = sorted(range(len(z)), key=lambda j: (-z[j], j))[: case["topk"]]
        total = sum(share(max(z) - z[j]) for j in (chosen if case["renorm"] else range(len(z))))
        r = (1 << 62) // total
        p = [min(32767, (share(max(z) - z[j]) * r + (1 << 46)) >> 47) for j in chosen]
        acc = torch.zeros(case["D"], dtype=torch.int64, device=DEV)
        for j, pj in zip(chosen, p):
            v = x_gate(x_product(q[t], [w[j] for w in s["up"]], e[t], case["group"]), s["lut"])
            e2 = x_shift(v[None], 15)
            acc += pj * x_product(x_round(v, e2).clamp(-32767, 32767), [w[j] for w in s["down"]], e2[0], case["group"])
        ys.append(x_round(x_round(acc, 15) + s["res"][t], 0))
        ids.append(chosen)
        ps.append(p)
    return {"y": torch.stack(ys), "idx": torch.tensor(ids), "p": torch.tensor(ps)}

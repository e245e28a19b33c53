"""The language-model operators (include/vgemm_lm.h) by their formulas in Python and numpy 64-bit integers, and seeded inputs
for their tests. int64 arithmetic wraps as the formulas say; the square root and the floor divisions are Python's."""
import math

import numpy as np

I64 = np.int64


def up(v, a):
    return (v + a - 1) // a * a


def sat32(v):
    return np.clip(v, -(1 << 31), (1 << 31) - 1)


def rshr(v, s):
    """Rounding right shift for s >= 0, saturating left shift for s < 0, saturated to 32 bits (src/intops.cuh:11-17)."""
    v, s = np.broadcast_arrays(np.asarray(v, I64), np.asarray(s, I64))
    p = np.clip(s, 0, 62)
    with np.errstate(over="ignore"):
        right = (v + ((I64(1) << p) >> 1)) >> p
        neg = np.clip(-s, 0, 31)
        lim = I64(1) << (62 - neg)
        left = np.clip(v, -lim, lim) * (I64(1) << neg)
    return sat32(np.where(s >= 0, right, left))


def shift_to(m, bits):
    """The least e >= 0 with m < 2^(bits + e), m below 2^32."""
    return np.array([max(0, int(v).bit_length() - bits) for v in np.asarray(m).reshape(-1)], I64).reshape(np.shape(m))


def quant(y, bits):
    """Rows in `bits` + 1 bits: q and the shift of each row."""
    e = shift_to(np.abs(y).max(-1), bits)
    lim = (1 << bits) - 1
    return np.clip(rshr(y, e[..., None]), -lim, lim), e


def lut16i(x, L):
    z = x + (16 << 16)
    i, f = np.clip(z >> 10, 0, 2047), z & 1023
    a, b = L.astype(I64)[i], L.astype(I64)[i + 1]
    return np.where(z < 0, 0, np.where(z >= (32 << 16), 65536, a + (((b - a) * f) >> 10)))


def geglu(y, L):
    a, g = y[..., 0::2], y[..., 1::2]
    return rshr(a * rshr(g * lut16i(g, L), 16), 16)


def rmsnorm(x, r, g, den):
    """h, y (int64) of vgemm_rmsnorm_q."""
    h = sat32(x.astype(I64) + (0 if r is None else r.astype(I64)))
    y = np.zeros_like(h)
    C = h.shape[1]
    for t in range(h.shape[0]):
        ex = max(0, int(shift_to(np.abs(h[t]).max(), 15)) - 5)
        ss = int((rshr(h[t], ex) ** 2).sum())
        sd = math.isqrt((ss // C + ((1 << (32 - 2 * ex)) + den // 2) // den) << 16)
        yy = [((int(v) << (25 - ex)) + sd) // (2 * sd) if sd else 0 for v in h[t]]
        y[t] = rshr(np.array(yy, I64) * g.astype(I64), 16)
    return h, y


class Weights:
    """`count` random N x K matrices of 4-bit codes with group scales and zero points and their column constants."""

    def __init__(self, rng, N, K, group, count=None, zeros=True, s=None, scale=(1, 4096), m=(1, 1 << 15), b=60000, pad=0):
        lead = () if count is None else (count,)
        self.N, self.K, self.group, self.groups, self.count = N, K, group, up(K, group) // group, count
        self.u = rng.integers(0, 16, (*lead, N, K), dtype=np.uint8)
        self.sc = rng.integers(*scale, (*lead, N, self.groups + pad), dtype=np.int16)
        self.z = rng.integers(0, 16, (*lead, N, self.groups + pad), dtype=np.uint8) if zeros else None
        u = np.concatenate([self.u, np.zeros((*lead, N, K % 2), np.uint8)], -1)
        self.nib = np.concatenate([u[..., 0::2] | u[..., 1::2] << 4, rng.integers(0, 256, (*lead, N, pad), dtype=np.uint8)], -1)
        self.msb = np.zeros((*lead, N, 4), np.int32)
        self.msb[..., 0] = rng.integers(*m, (*lead, N))
        if s is None:
            s = 14 + 11 + 13 + int(math.log2(K) / 2)
        self.msb[..., 1] = rng.integers(s - 2, s + 2, (*lead, N))
        self.msb[..., 2] = rng.integers(-b, b + 1, (*lead, N))
        self.msb[..., 3] = rng.integers(-9, 9, (*lead, N))     # not read

    def dense(self):
        """(u - z) sc, int64 [..., N, K]."""
        z = np.repeat((self.z if self.z is not None else np.full_like(self.sc, 8)).astype(I64)[..., :self.groups], self.group, -1)[..., :self.K]
        sc = np.repeat(np.minimum(self.sc.view(np.uint16).astype(I64), 4095)[..., :self.groups], self.group, -1)[..., :self.K]
        return (self.u.astype(I64) - z) * sc


def product(q, e, w, msb):
    """PLAIN rows of one matrix: q int64 [M, K], e [M], w int64 [N, K]."""
    # exact in float64: |acc| <= 2^15 * 15 * 4095 * 2^15 < 2^46
    acc = np.rint(q.astype(np.float64) @ w.T.astype(np.float64)).astype(I64)
    with np.errstate(over="ignore"):
        v = acc * msb[:, 0].astype(I64)
    return sat32(rshr(v, msb[:, 1].astype(I64) - np.asarray(e, I64)[:, None]) + msb[:, 2])


def lutexp(z, L):
    return 0 if z >= 1 << 20 else int(L[z >> 10]) + (((int(L[(z >> 10) + 1]) - int(L[z >> 10])) * (z & 1023)) >> 10)


def route(q, e, w, cst, topk, renorm, L):
    """idx, p, logits of vgemm_moe_route."""
    acc = q.astype(I64) @ w.astype(I64).T
    with np.errstate(over="ignore"):
        z = sat32(rshr(acc * cst[:, 0].astype(I64), cst[:, 1].astype(I64) - np.asarray(e, I64)[:, None]) + cst[:, 2])
    idx, p = [], []
    for row in z.tolist():
        top = sorted(range(len(row)), key=lambda j: (-row[j], j))[:topk]
        tot = sum(lutexp(row[top[0]] - row[j], L) for j in (top if renorm else range(len(row))))
        r = (1 << 62) // tot if tot else 0
        idx.append(top)
        p.append([min(32767, (lutexp(row[top[0]] - row[j], L) * r + (1 << 46)) >> 47) for j in top])
    return np.array(idx), np.array(p), z


def moe(q, e, idx, p, up_w: Weights, down_w: Weights, lut, res):
    """Y of vgemm_moe."""
    out = np.zeros((q.shape[0], down_w.N), I64)
    du, dd = up_w.dense(), down_w.dense()
    for t in range(q.shape[0]):
        for x, share in zip(idx[t], p[t]):
            if not 0 <= x < up_w.count:
                continue
            v = geglu(product(q[t:t + 1], e[t:t + 1], du[x], up_w.msb[x]), lut)
            q2, e2 = quant(v, 15)
            out[t] += int(share) * product(q2, e2, dd[x], down_w.msb[x])[0]
    out = rshr(out, 15)
    return out if res is None else sat32(out + res)


def sigmoid_table():
    x = (np.arange(2049) - 1024) / 64.0
    return np.round(65536 / (1 + np.exp(-x))).astype(np.int32)


def exp_table():
    return np.round(np.exp(-np.arange(1025) / 64.0) * 2.0**30).astype(np.int64)


def rows8(rng, M, K, ld=None, full=False):
    """8-bit rows [M, ld] (columns past K hold junk, which nothing may use) and shifts."""
    q = rng.integers(-127, 128, (M, ld or up(K, 16)), dtype=np.int8)
    if full:
        q[...] = np.where(rng.random(q.shape) < 0.5, -128, 127)
    return q, rng.integers(0, 14, M, dtype=np.int32)


def rows16(rng, M, K, ld=None, full=False):
    """16-bit rows as planes hi, lo [M, ld], their values [M, K] and shifts."""
    v = rng.integers(-32767, 32768, (M, ld or up(K, 16)))
    if full:
        v = np.where(rng.random(v.shape) < 0.5, -32768, 32767)
    return (v >> 8).astype(np.int8), ((v & 255) - 128).astype(np.int8), v[:, :K].astype(I64), rng.integers(0, 6, M, dtype=np.int32)

"""The paged key-value cache and its operators (include/vgemm_kv.h) by their formulas in Python and numpy 64-bit integers."""
import numpy as np

from tests import lm_math as lm

I64 = np.int64
SPAN, VSPAN = 256, 4096
LOW, NONE = -(1 << 31), -(1 << 63)


def lutexp(d, L):
    d = np.asarray(d, I64)
    c = np.minimum(d, (1 << 20) - 1)
    L = L.astype(I64)
    i, f = c >> 10, c & 1023
    return np.where(d >= 1 << 20, 0, L[i] + (((L[i + 1] - L[i]) * f) >> 10))


def ln_table():
    return np.round(np.log1p(np.arange(1025) / 1024.0) * 2.0**30).astype(np.int64)


def quant(x, bits):
    """Rows [.., D] as the cache holds them: q and the shift of each row."""
    return lm.quant(np.asarray(x, I64), bits - 1)


def scale_of(D):
    s = 31 + int(np.log2(np.sqrt(D)))
    return round(2.0**(s - 16) / np.sqrt(D)), s


def plan(length, add, table, free, pages, page, width, tokens):
    """table (a copy), new_len, start, slot, pos, used."""
    table = table.copy()
    start, slot, pos, used = [0], np.full(tokens, -1, I64), np.full(tokens, -1, I64), 0
    new = []
    for r, (n, a) in enumerate(zip(length, add)):
        n, a = min(max(int(n), 0), 1 << 23), min(max(int(a), 0), 1 << 23)
        have, need = -(-n // page), min(-(-(n + a) // page), width)
        for j in range(have, need):
            p = int(free[used]) if used < len(free) else -1
            table[r, j] = p if 0 <= p < pages else -1
            used += 1
        for i in range(a):
            t, at = start[-1] + i, n + i
            if t >= tokens:
                break
            pos[t] = at
            if at // page < width and 0 <= table[r, at // page] < pages:
                slot[t] = table[r, at // page] * page + at % page
        start.append(start[-1] + a)
        new.append(n + a)
    return table, np.array(new, I64), np.array(start, I64), slot, pos, used


def attend(q, k, ek, v, ev, ok, heads, m, s, L):
    """One sequence: q [Hq, D] int32 values, k and v [n, heads, D] with shifts [n, heads] (position by position), ok [n]: the tokens
    that count. Returns [Hq, D]."""
    Hq, D = q.shape
    n = len(ok)
    out = np.zeros((Hq, D), I64)
    at = np.nonzero(ok)[0]
    if at.size == 0:
        return out
    for h in range(Hq):
        g = h // (Hq // heads)
        x, eq = quant14(q[h].astype(I64))
        # whole numbers below 2^53: exact in float64
        S = np.rint(k[at, g].astype(np.float64) @ x.astype(np.float64)).astype(I64)
        z = lm.rshr(S * m, s - eq - ek[at, g].astype(I64))
        mx, Ls, As = [], [], []
        ends = np.flatnonzero(np.diff(at // SPAN, append=-1)) + 1
        for i in map(slice, np.concatenate([[0], ends[:-1]]), ends):
            top = z[i].max()
            P = np.minimum(32767, (lutexp(top - z[i], L) + (1 << 14)) >> 15)
            w = int(P.sum())
            num = (P[:, None] * (v[at[i], g].astype(I64) << ev[at[i], g].astype(I64)[:, None])).sum(0)
            As.append((num + (w >> 1)) // w if w else np.zeros(D, I64))
            mx.append(int(top))
            Ls.append(w)
        mx, Ls, As = np.array(mx, I64), np.array(Ls, I64), np.array(As, I64)
        live = mx[Ls > 0]
        if live.size == 0:
            continue
        G = np.maximum((lutexp(np.maximum(live.max() - mx, 0), L) + 64) >> 7, mx == live.max()) * Ls
        down = max(0, int(G.sum()).bit_length() - 30)
        w = (G + ((1 << down) >> 1)) >> down
        T = int(w.sum())
        out[h] = lm.sat32(((w[:, None] * lm.sat32(As)).sum(0) + (T >> 1)) // T) if T else 0
    return out


def quant14(x):
    """The query in 15 bits and its shift: no value needs to be clamped."""
    e = int(lm.shift_to(np.abs(x).max(), 14))
    return lm.rshr(x, e), e


def logz(z, L, Lln):
    """max and log of the sum of one row's weights; None where every token is banned."""
    parts = []
    for b in range(0, len(z), VSPAN):
        p = z[b:b + VSPAN].astype(I64)
        p = p[p > LOW]
        if p.size:
            parts.append((int(p.max()), int(lutexp(p.max() - p, L).sum())))
    if not parts:
        return None
    mx = max(p[0] for p in parts)
    S = max(1, sum((int(lutexp(mx - a, L)) * ((b + 2048) >> 12) + (1 << 17)) >> 18 for a, b in parts))
    t = S.bit_length() - 1
    f = (S << 30 >> t) - (1 << 30)
    i, fr = f >> 20, f & ((1 << 20) - 1)
    lz = ((t - 30) * int(Lln[1024]) + int(Lln[i]) + (((int(Lln[i + 1]) - int(Lln[i])) * fr) >> 20) + (1 << 13)) >> 14
    return mx, lz


def select(z, score, groups, beams, n, L, Lln):
    """score, parent, token [groups, n] as Python integers."""
    out = []
    for g in range(groups):
        best = []
        for r in range(g * beams, (g + 1) * beams):
            if int(score[r]) == NONE:
                continue
            st = logz(z[r], L, Lln)
            if st is None:
                continue
            row = z[r].astype(I64)
            keep = np.argsort(-row, kind="stable")[:n]
            best += [(-(int(score[r]) + int(row[t]) - st[0] - st[1]), r, int(t)) for t in keep if row[t] > LOW]
        best = sorted(best)[:n]
        best += [(-NONE, -1, -1)] * (n - len(best))
        out.append(best)
    return (np.array([[-b[0] for b in o] for o in out], I64), np.array([[b[1] for b in o] for o in out]), np.array([[b[2] for b in o] for o in out]))


def beam_tables(parent, length, table, fresh, page, width):
    rows = len(parent)
    out, src, dst, new = np.full((rows, width), -1, I64), np.full(rows, -1, I64), np.full(rows, -1, I64), np.zeros(rows, I64)
    for r, p in enumerate(parent):
        n = min(max(int(length[p]), 0), width * page) if 0 <= p < rows else 0
        full, part = divmod(n, page)
        new[r] = n
        if full:
            out[r, :full] = table[p, :full]
        if part:
            out[r, full], src[r], dst[r] = fresh[r], table[p, full], fresh[r]
    return out, new, src, dst

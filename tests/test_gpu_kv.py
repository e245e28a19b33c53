"""The paged key-value cache's operators on the GPU: every result is a whole number and has to be equal to the formulas in 64-bit
integers (tests/kv_math.py)."""
import numpy as np
import pytest
import torch

from tests import kv_math as km
from tests import lm_math as lm
from tests.conftest import assert_equal, to_np
from vela_amd import beam as vb
from vela_amd import gemm as vg
from vela_amd import kv as vk

pytestmark = pytest.mark.gpu
JUNK = -123456789


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def full(shape, v=JUNK, dt=torch.int32):
    return torch.full((shape,) if isinstance(shape, int) else shape, v, dtype=dt, device="cuda")


# ---------------------------------------------------------------- block tables and slot maps

def run_plan(length, add, table, free, nfree, pages, page, width, tokens, optional=True, stream=None):
    d = {k: dev(np.asarray(v, np.int32)) for k, v in dict(len=length, add=add, table=table, free=free, nfree=[nfree]).items()}
    R = len(length)
    out = dict(new_len=full(R + 1), start=full(R + 2), slot=full(tokens + 1), pos=full(tokens + 1), used=full(2))
    if not optional:
        out = {"slot": out["slot"]}
    P = vk.KvPlan(R=R, tokens=tokens, pages=pages, page=page, width=width, ldt=table.shape[1] if table.ndim == 2 else width,
                  **{k: vg.ptr(v) if v.numel() else None for k, v in {**d, **out}.items()})
    vk.k_kv_plan(P, stream)
    return {"table": to_np(d["table"]), **{k: to_np(v) for k, v in out.items()}}


def check_plan(length, add, table, free, pages, page, width, tokens, nfree=None, **kw):
    nfree = len(free) if nfree is None else nfree
    got = run_plan(length, add, table, free, nfree, pages, page, width, tokens, **kw)
    want = km.plan(length, add, table, free[:nfree], pages, page, width, tokens)
    R = len(length)
    for name, w in zip(("table", "new_len", "start", "slot", "pos", "used"), want):
        if name not in got:
            continue
        g = got[name]
        if name == "table":
            assert_equal(g, w, name)
        else:
            size = {"new_len": R, "start": R + 1, "used": 1}.get(name, tokens)
            assert_equal(g[:size], np.reshape(w, -1), name)
            assert (g[size:] == JUNK).all(), f"{name}: written past its end"


def random_plan(rng, R, most, ctx, page, ldt=0):
    length, add = rng.integers(0, ctx + 1, R), rng.integers(0, most + 1, R)
    width = max(1, -(-(ctx + most) // page))
    need = -(-length // page)
    pages = int(need.sum()) + int((-(-(length + add) // page) - need).sum()) + 3
    order = rng.permutation(pages)
    table = np.full((R, width + ldt), JUNK, np.int32)
    at = 0
    for r in range(R):
        table[r, :need[r]] = order[at:at + need[r]]
        at += need[r]
    return length, add, table, order[at:].astype(np.int32), pages, width


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("R,most,ctx", [(1, 1, 0), (1, 700, 300), (5, 40, 60), (255, 1, 900), (256, 3, 40), (257, 9, 500), (1000, 2, 33), (4096, 1, 20)])
def test_plan(gpu, page, R, most, ctx):
    rng = np.random.default_rng(R + page)
    length, add, table, free, pages, width = random_plan(rng, R, most, ctx, page, ldt=3)
    check_plan(length, add, table, free, pages, page, width, int(add.sum()) + 5)


def test_plan_of_no_requests_and_no_rows(gpu):
    got = run_plan([], [], np.zeros((0, 4), np.int32), np.zeros(0, np.int32), 0, 8, 16, 4, 7)
    assert (got["slot"][:7] == -1).all() and (got["pos"][:7] == -1).all() and got["start"][0] == 0 and got["used"][0] == 0
    rng = np.random.default_rng(3)
    length, add, table, free, pages, width = random_plan(rng, 6, 50, 90, 16)
    check_plan(length, add, table, free, pages, 16, width, 0)        # the tables alone
    check_plan(length, add, table, free, pages, 16, width, 40, optional=False)


@pytest.mark.parametrize("rows", [1, 30, 100])
def test_plan_with_fewer_rows_than_tokens(gpu, rows):
    """Pages and lengths do not depend on the token rows there are."""
    length, add, table, free, pages, width = random_plan(np.random.default_rng(4), 9, 60, 90, 16)
    check_plan(length, add, table, free, pages, 16, width, rows)


def test_plan_of_the_most_rows(gpu):
    """2^31 - 1 of them: the rows behind the tokens get -1 by all blocks."""
    tokens, length, add = (1 << 31) - 1, [3, 20], [40, 7]
    table, free = np.array([[5, -1, -1], [2, 0, -1]], np.int32), np.array([1, 7, 3], np.int32)
    d = [dev(np.asarray(v, np.int32)) for v in (length, add, table, free, [3])]
    slot = full(tokens + 1)
    P = vk.KvPlan(R=2, tokens=tokens, pages=8, page=16, width=3, ldt=3, len=vg.ptr(d[0]), add=vg.ptr(d[1]), table=vg.ptr(d[2]), free=vg.ptr(d[3]), nfree=vg.ptr(d[4]),
                  slot=vg.ptr(slot))
    vk.k_kv_plan(P)
    want = km.plan(length, add, table, free, 8, 16, 3, 50)
    assert_equal(to_np(d[2]), want[0])
    assert_equal(to_np(slot[:50]), want[3])
    assert int(slot[50:tokens].amax()) == int(slot[50:tokens].amin()) == -1 and int(slot[tokens]) == JUNK


@pytest.mark.parametrize("nfree", [0, 1, 5, -4])
def test_plan_past_the_free_list(gpu, nfree):
    length, add, table, free, pages, width = random_plan(np.random.default_rng(5), 12, 70, 90, 16)
    check_plan(length, add, table, free, pages, 16, width, int(add.sum()) + 2, nfree=max(nfree, 0)) if nfree >= 0 else None
    got = run_plan(length, add, table, free, nfree, pages, 16, width, int(add.sum()))
    want = km.plan(length, add, table, free[:max(nfree, 0)], pages, 16, width, int(add.sum()))
    assert_equal(got["table"], want[0])
    assert_equal(got["slot"][:-1], want[3])
    assert got["used"][0] == want[5] > max(nfree, 0)


def test_plan_of_bad_numbers(gpu):
    """Lengths below zero count as zero, tokens past the table's width and on entries that are no pages have no slot, free numbers that are
    no pages become -1."""
    table = np.array([[4, -1, JUNK], [99, -1, JUNK], [JUNK, -1, JUNK], [2, 6, JUNK]], np.int32)
    check_plan([10, 10, -5, 31], [30, 3, 18, 40], table, np.array([7, 12, -3, 5], np.int32), 10, 16, 2, 100)
    check_plan([10, 10, 7, 31], [30, 3, -18, 1 << 30], table, np.array([7, 12, -3, 5], np.int32), 10, 16, 2, 100)
    check_plan([500, 10, 0, 0], [30, 3, 0, 2], table, np.array([7, 8, 9, 5], np.int32), 10, 16, 2, 100)   # more tokens than the table's width


# ---------------------------------------------------------------- rows

class Cache:
    """A cache of junk, with what was written by position of slot."""

    def __init__(self, pages, page, heads, D, bits, seed=0):
        self.c = vk.KvCache(pages, page, heads, D, bits)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.c.data.copy_(torch.randint(-128, 128, self.c.data.shape, generator=g, device="cuda", dtype=torch.int8))
        self.c.shift.copy_(torch.randint(0, 256, self.c.shift.shape, generator=g, device="cuda", dtype=torch.uint8))

    def values(self):
        """q of keys and of values [slots, heads, D], their shifts [slots, heads], from the layout of the header."""
        c = self.c
        n, g = c.bits // 8, c.page // 16
        d = to_np(c.data).reshape(c.pages, c.heads, 2, g, n, 16 * c.D).astype(np.int64)
        out = []
        for half in range(2):
            if half == 0:
                x = d[:, :, 0].reshape(c.pages, c.heads, g, n, 4, c.D // 16, 4, 16).transpose(0, 2, 4, 6, 1, 3, 5, 7)
            else:
                x = d[:, :, 1].reshape(c.pages, c.heads, g, n, c.D, 16).transpose(0, 2, 5, 1, 3, 4)
            x = x.reshape(c.pages * c.page, c.heads, n, c.D)
            out.append(x[:, :, 0] if n == 1 else 256 * x[:, :, 0] + x[:, :, 1] + 128)
        s = to_np(c.shift).reshape(c.pages, c.heads, 2, c.page).astype(np.int64).transpose(2, 0, 3, 1).reshape(2, -1, c.heads)
        return out[0], s[0], out[1], s[1]


def rows_of(rng, M, heads, D, extreme=False):
    x = np.round(rng.standard_normal((M, heads, D)) * 65536 * np.exp(rng.standard_normal((M, heads, 1)))).astype(np.int64)
    if extreme:
        x = rng.integers(-(1 << 31), 1 << 31, (M, heads, D)) >> rng.integers(0, 32, (M, heads, 1))
        kind = rng.integers(0, 6, (M, heads))
        x[kind == 0] = 0
        x[kind == 1] = -(1 << 31)
        x[kind == 2] = (1 << 31) - 1
        x[kind == 3] = np.where(rng.random((int((kind == 3).sum()), D)) < 0.5, 127, -128)
    return x.astype(np.int32)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("page,heads,D,M", [(16, 1, 16, 1), (16, 8, 128, 24), (32, 3, 80, 33), (64, 2, 64, 200), (128, 5, 96, 17), (256, 2, 256, 300), (16, 1, 192, 15),
                                            (64, 1024, 16, 3)])
@pytest.mark.parametrize("extreme", [False, True])
def test_rows_into_pages_and_back(gpu, bits, page, heads, D, M, extreme):
    rng = np.random.default_rng(M + D)
    pages = -(-M // page) + 2
    C = Cache(pages, page, heads, D, bits)
    before = C.values()
    slot = rng.permutation(pages * page)[:M].astype(np.int32) if M < 100 else np.arange(7, 7 + M, dtype=np.int32)
    if M > 2:
        slot[1], slot[2] = -1, pages * page
    pad = 8
    k, v = (np.concatenate([rows_of(rng, M, heads, D, extreme).reshape(M, -1), rng.integers(-9, 9, (M, pad)).astype(np.int32)], 1) for _ in range(2))
    dk, dv, ds = dev(k), dev(v), dev(slot)
    vk.k_kv_write(C.c, dk, dv, heads * D + pad, ds, M)
    after = C.values()
    there = (slot >= 0) & (slot < pages * page)
    for x, b0, s0, b1, s1, name in ((k, before[0], before[1], after[0], after[1], "keys"), (v, before[2], before[3], after[2], after[3], "values")):
        q, e = km.quant(x[:, :heads * D].reshape(M, heads, D), bits)
        b0[slot[there]], s0[slot[there]] = q[there], e[there]
        assert_equal(b1, b0, name)
        assert_equal(s1, s0, f"{name}: shifts")
    ko, vo = full((M, heads * D + pad)), full((M, heads * D + pad))
    vk.k_kv_read(C.c, ds, M, ko, vo, heads * D + pad)
    only_k, only_v = full((M, heads * D + pad)), full((M, heads * D + pad))
    vk.k_kv_read(C.c, ds, M, only_k, None, heads * D + pad)
    vk.k_kv_read(C.c, ds, M, None, only_v, heads * D + pad)
    for x, o, o1, name in ((k, ko, only_k, "keys"), (v, vo, only_v, "values")):
        q, e = km.quant(x[:, :heads * D].reshape(M, heads, D), bits)
        want = np.where(there[:, None], lm.sat32(q << e[..., None]).reshape(M, -1), 0)
        assert_equal(to_np(o)[:, :heads * D], want, name)
        assert (to_np(o)[:, heads * D:] == JUNK).all()
        assert torch.equal(o, o1)


def test_rows_of_a_merged_projection(gpu):
    """K and V as parts of the same rows, queries before them."""
    rng = np.random.default_rng(8)
    M, heads, D, Hq = 37, 2, 64, 6
    x = rows_of(rng, M, Hq + 2 * heads, D)
    dx, C = dev(x.reshape(M, -1)), Cache(3, 16, heads, D, 8)
    ds = torch.arange(M, dtype=torch.int32, device="cuda")
    ld = (Hq + 2 * heads) * D
    vk.k_kv_write(C.c, vg.ptr(dx) + 4 * Hq * D, vg.ptr(dx) + 4 * (Hq + heads) * D, ld, ds, M)
    got = C.values()
    for (q, e), (g, s) in zip((km.quant(x[:, Hq:Hq + heads], 8), km.quant(x[:, Hq + heads:], 8)), (got[:2], got[2:])):
        assert_equal(g[:M], q)
        assert_equal(s[:M], e)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("page,heads,D,n", [(16, 1, 16, 1), (16, 8, 128, 7), (64, 3, 80, 40), (256, 16, 256, 3)])
def test_copies_of_pages(gpu, bits, page, heads, D, n):
    rng = np.random.default_rng(n)
    pages = 2 * n + 3
    C = Cache(pages, page, heads, D, bits)
    data, shift = to_np(C.c.data).reshape(pages, -1).copy(), to_np(C.c.shift).reshape(pages, -1).copy()
    order = rng.permutation(pages)
    src, dst = order[:n].astype(np.int32), order[n:2 * n].astype(np.int32)
    if n > 3:
        src[0], dst[1], src[2], dst[3], src[4] = -1, -1, pages, pages + 5, src[5]
    ok = (src >= 0) & (src < pages) & (dst >= 0) & (dst < pages)
    vk.k_kv_copy(C.c, dev(src), dev(dst), n)
    data[dst[ok]], shift[dst[ok]] = data[src[ok]], shift[src[ok]]
    assert_equal(to_np(C.c.data).reshape(pages, -1), data)
    assert_equal(to_np(C.c.shift).reshape(pages, -1), shift)


# ---------------------------------------------------------------- attention

class Attend:
    """Sequences of given lengths in a cache of shuffled pages."""

    def __init__(self, rng, lens, page, heads, D, bits, Hq, extreme=False, width=0, kvscale=None):
        self.rng, self.page, self.heads, self.D, self.bits, self.Hq, self.lens = rng, page, heads, D, bits, Hq, np.asarray(lens)
        R = len(lens)
        need = -(-np.maximum(self.lens, 0) // page)
        self.width = max(int(need.max(initial=0)), 1) + width
        pages = int(need.sum()) + 2
        order = rng.permutation(pages)
        self.table = np.full((R, self.width + 3), -1, np.int32)
        at = 0
        for r in range(R):
            self.table[r, :need[r]] = order[at:at + need[r]]
            at += need[r]
        C = self.cache = Cache(pages, page, heads, D, bits)
        slots = np.concatenate([self.slots(r) for r in range(R)]).astype(np.int32) if need.sum() else np.zeros(0, np.int32)
        k, v = rows_of(rng, len(slots), heads, D, extreme), rows_of(rng, len(slots), heads, D, extreme)
        if kvscale is not None:
            k, v = kvscale(k), kvscale(v)
        if len(slots):
            vk.k_kv_write(C.c, dev(k.reshape(len(slots), -1)), dev(v.reshape(len(slots), -1)), heads * D, dev(slots), len(slots))
        self.q = rows_of(rng, R, Hq, D, extreme)
        self.lexp = lm.exp_table()
        self.m, self.s = km.scale_of(D)

    def slots(self, r):
        j = np.arange(max(self.lens[r], 0))
        return self.table[r, j // self.page] * self.page + j % self.page

    def want(self, window=0, max_len=1 << 23):
        kq, ek, vq, ev = self.cache.values()
        out = []
        for r in range(len(self.lens)):
            n = min(max(int(self.lens[r]), 0), max_len, self.width * self.page)
            j = np.arange(n)
            page = self.table[r, j // self.page]
            ok = (page >= 0) & (page < self.cache.c.pages) & (j >= (n - window if window else 0))
            at = np.where(ok, page * self.page + j % self.page, 0)
            out.append(km.attend(self.q[r], kq[at], ek[at], vq[at], ev[at], ok, self.heads, self.m, self.s, self.lexp))
        return np.array(out).reshape(len(self.lens), -1)

    def args(self, window=0, max_len=None, ldq=None, ldo=None, rowmax=None):
        R, C = len(self.lens), self.Hq * self.D
        max_len = max(int(self.lens.max(initial=0)), 1) if max_len is None else max_len
        ldq, ldo = ldq or C, ldo or C
        d = self.d = dict(q=full((R, ldq)), out=full((R, ldo)), table=dev(self.table), len=dev(self.lens.astype(np.int32)), lexp=dev(self.lexp))
        d["q"][:, :C] = dev(self.q.reshape(R, -1))
        nb = vk.kv_attention_workspace_bytes(R, self.Hq, self.D, max_len)
        d["ws"] = full((nb // 4 + 4,))
        d["rowmax"] = rowmax
        return vk.KvAttn(Q=vg.ptr(d["q"]), ldq=ldq, rows=R, Hq=self.Hq, table=vg.ptr(d["table"]), ldt=self.table.shape[1], width=self.width, len=vg.ptr(d["len"]), max_len=max_len,
                         window=window, m=self.m, s=self.s, Lexp=vg.ptr(d["lexp"]), out=vg.ptr(d["out"]), ldo=ldo, rowmax=vg.ptr(rowmax), ws=vg.ptr(d["ws"]), ws_bytes=nb)

    def check(self, window=0, max_len=None, pad=0):
        R, C = len(self.lens), self.Hq * self.D
        rowmax = full(R, 5)
        A = self.args(window, max_len, C + pad, C + 2 * pad, rowmax)
        vk.k_kv_attention(self.cache.c, A)
        got, want = to_np(self.d["out"]), self.want(window, A.max_len)
        assert_equal(got[:, :C], want, "out")
        assert (got[:, C:] == JUNK).all()
        assert (to_np(self.d["ws"])[A.ws_bytes // 4:] == JUNK).all(), "written past the workspace"
        assert_equal(to_np(rowmax).view(np.uint32), np.maximum(np.abs(want).max(1), 5), "rowmax")


SHAPES = [  # page, heads, D, Hq
    (16, 1, 16, 1), (16, 2, 64, 2), (16, 2, 128, 8), (32, 3, 80, 15), (64, 1, 96, 16), (128, 2, 192, 12), (256, 1, 256, 4), (64, 1, 64, 17), (16, 1, 128, 40)]


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("page,heads,D,Hq", SHAPES)
def test_attention(gpu, bits, page, heads, D, Hq):
    rng = np.random.default_rng(D + Hq)
    Attend(rng, [1, 0, 5, 255, 256, 257, 700, 64, 1023], page, heads, D, bits, Hq).check()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 511, 512, 513, 5000])
def test_attention_lengths(gpu, bits, n):
    Attend(np.random.default_rng(n), [n], 16, 2, 64, bits, 6).check()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D,heads,Hq", [(16, 2, 2), (64, 1, 5), (128, 2, 4), (256, 1, 1)])
def test_attention_of_extreme_rows(gpu, bits, D, heads, Hq):
    """Rows of the type's lowest and highest values and of zeros, shifts from 0 to the most side by side: six digits."""
    Attend(np.random.default_rng(D), [300, 256, 40, 1, 2], 32, heads, D, bits, Hq, extreme=True).check(pad=4)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("spread", [0, 1, 7, 8, 9, 15, 16, 17, 24])
def test_attention_of_shifts_apart(gpu, bits, spread):
    """Every number of digits the weights can take, at both ends of its range."""
    rng = np.random.default_rng(spread)
    top = 31 - spread - (1 if spread < 24 else 0)

    def scale(x):
        up = rng.integers(0, 2, x.shape[:2])[..., None] * spread
        return (np.sign(x) * (np.abs(x.astype(np.int64)) % 64 + 64 << up) << min(top - 7, 3)).astype(np.int32)

    Attend(rng, [256, 100, 600], 16, 2, 64, bits, 4, kvscale=scale).check()


@pytest.mark.parametrize("window", [1, 2, 100, 255, 256, 257, 300, 512, 5000])
def test_attention_windows(gpu, window):
    Attend(np.random.default_rng(window), [1, 0, 256, 300, 777, 1024, 1025], 16, 2, 64, 8, 4).check(window=window)


def test_attention_of_absent_pages(gpu):
    """Entries that are no pages mask their tokens, up to whole spans and whole rows; a table narrower than the length bounds it, as does max_len."""
    a = Attend(np.random.default_rng(9), [1000, 1000, 600, 300, 20], 16, 2, 64, 8, 4)
    a.table[0, 3], a.table[0, 20], a.table[0, 62] = -1, a.cache.c.pages, -(1 << 31)
    a.table[1, 16:32] = -1                      # a whole span
    a.table[2, :38] = 1 << 30                   # the whole row
    a.table[3, 16:] = -1                        # the last span
    a.check()
    a.check(window=300)
    a.check(max_len=700)
    a.check(max_len=256)
    a.check(max_len=1)
    a.width = 40
    a.check(max_len=4000)
    a.width = 0
    a.check()


def test_attention_without_tokens(gpu):
    a = Attend(np.random.default_rng(10), [0, -7, 0], 16, 2, 64, 8, 4)
    a.check()
    a.check(max_len=0)


@pytest.mark.parametrize("table", ["zero", "one", "most", "steps", "rising"])
def test_attention_tables(gpu, table):
    """Other tables than exp's, down to one of zeros (nothing counts) and up to the largest entries."""
    a = Attend(np.random.default_rng(11), [700, 200, 256], 16, 2, 64, 8, 4)
    a.lexp = {"zero": np.zeros(1025), "one": np.ones(1025), "most": np.full(1025, 2**31 - 1), "steps": (np.arange(1025) % 2) * (2**31 - 1),
              "rising": np.arange(1025) * 2097151}[table].astype(np.int64)
    a.check()


@pytest.mark.parametrize("m,s", [(1, -64), (32768, -64), (32768, 128), (1, 128), (32768, 0), (20000, 60), (1, 15)])
@pytest.mark.parametrize("bits", [8, 16])
def test_attention_scales(gpu, m, s, bits):
    """Scores that saturate, that are all equal, that need every bit."""
    a = Attend(np.random.default_rng(12), [300, 64, 700], 16, 1, 256, bits, 3, extreme=bits == 16)
    a.m, a.s = m, s
    a.check()


def test_attention_of_many_rows(gpu):
    """More spans than blocks: a block takes several, one after the other."""
    rng = np.random.default_rng(13)
    a = Attend(rng, rng.integers(0, 800, 300), 16, 40, 16, 8, 40)
    a.check()


@pytest.mark.parametrize("n", [70000, 270000])
def test_attention_of_long_sequences(gpu, n):
    """More spans than the join holds weights of at a time."""
    Attend(np.random.default_rng(14), [n, 3000], 256, 1, 16, 8, 2).check()


def test_attention_past_four_gigabytes(gpu):
    """Pages whose offsets pass 32 bits, in bytes of data and in elements."""
    page, heads, D = 256, 16, 256
    nb = vk.kv_page_bytes(page, heads, D, 16)
    pages = (5 << 30) // nb
    C = vk.KvCache(pages, page, heads, D, 16)
    rng = np.random.default_rng(15)
    n, used = 400, [pages - 1, pages - 3]
    slot = np.concatenate([np.arange(256) + used[0] * page, np.arange(144) + used[1] * page]).astype(np.int32)
    k, v = rows_of(rng, n, heads, D), rows_of(rng, n, heads, D)
    vk.k_kv_write(C, dev(k.reshape(n, -1)), dev(v.reshape(n, -1)), heads * D, dev(slot), n)
    ko, vo = full((n, heads * D)), full((n, heads * D))
    vk.k_kv_read(C, dev(slot), n, ko, vo, heads * D)
    (kq, ek), (vq, ev) = km.quant(k, 16), km.quant(v, 16)
    assert_equal(to_np(ko), (kq << ek[..., None]).reshape(n, -1))
    assert_equal(to_np(vo), (vq << ev[..., None]).reshape(n, -1))
    q, lexp, out = rows_of(rng, 1, heads, D), lm.exp_table(), full((1, heads * D))
    m, s = km.scale_of(D)
    ws = full((vk.kv_attention_workspace_bytes(1, heads, D, n) // 4,))
    vk.k_kv_copy(C, dev(np.array([used[1]], np.int32)), dev(np.array([pages - 2], np.int32)), 1)
    for t in ([used[0], used[1]], [used[0], pages - 2]):
        d = dict(q=dev(q.reshape(1, -1)), t=dev(np.array([t], np.int32)), n=dev(np.array([n], np.int32)), L=dev(lexp))
        vk.k_kv_attention(C, vk.KvAttn(Q=vg.ptr(d["q"]), ldq=heads * D, rows=1, Hq=heads, table=vg.ptr(d["t"]), ldt=2, width=2, len=vg.ptr(d["n"]), max_len=n, m=m, s=s,
                                       Lexp=vg.ptr(d["L"]), out=vg.ptr(out), ldo=heads * D, ws=vg.ptr(ws), ws_bytes=ws.numel() * 4))
        assert_equal(to_np(out)[0], km.attend(q[0], kq, ek, vq, ev, np.ones(n, bool), heads, m, s, lexp).reshape(-1))


# ---------------------------------------------------------------- beam search

def check_select(z, score, groups, beams, n, pad=0, lexp=None):
    V = z.shape[1]
    L, Ln = lm.exp_table() if lexp is None else lexp, km.ln_table()
    want = km.select(z, score, groups, beams, n, L, Ln)
    zp = np.concatenate([z, np.full((len(z), pad), (1 << 31) - 1, np.int32)], 1)
    d = [dev(zp), dev(score), dev(L), dev(Ln)]
    out = [full((groups * n + 1,), JUNK, torch.int64), full((groups * n + 1,)), full((groups * n + 1,))]
    nb = vb.beam_workspace_bytes(groups, beams, V, n)
    ws = full((nb // 4 + 1,))
    vb.k_beam_select(vb.BeamSelect(groups=groups, beams=beams, V=V, n=n, logits=vg.ptr(d[0]), ldz=V + pad, score=vg.ptr(d[1]), Lexp=vg.ptr(d[2]), Lln=vg.ptr(d[3]),
                                   out_score=vg.ptr(out[0]), parent=vg.ptr(out[1]), token=vg.ptr(out[2]), ws=vg.ptr(ws), ws_bytes=nb))
    for g, w, name in zip(out, want, ("score", "parent", "token")):
        assert_equal(to_np(g)[:-1].reshape(groups, n), w, name)
        assert to_np(g)[-1] == JUNK
    assert to_np(ws)[-1] == JUNK


def logits(rng, rows, V, scale=3):
    return np.round(rng.standard_normal((rows, V)) * scale * 65536).astype(np.int32)


def scores(rng, rows, dead=0.1):
    s = -rng.integers(0, 1 << 40, rows)
    s[rng.random(rows) < dead] = km.NONE
    return s.astype(np.int64)


@pytest.mark.parametrize("V", [1, 2, 63, 255, 256, 1000, 4095, 4096, 4097, 8191, 32000, 100003, 1 << 18])
@pytest.mark.parametrize("groups,beams,n", [(1, 1, 1), (1, 4, 8), (3, 5, 10)])
def test_select(gpu, V, groups, beams, n):
    rng = np.random.default_rng(V + n)
    check_select(logits(rng, groups * beams, V), scores(rng, groups * beams, 0.1), groups, beams, n, pad=V % 3)


@pytest.mark.parametrize("beams,n", [(32, 64), (32, 1), (1, 64), (2, 63), (17, 34)])
@pytest.mark.parametrize("V", [50, 9000])
def test_select_widest(gpu, beams, n, V):
    rng = np.random.default_rng(beams + n)
    check_select(logits(rng, 2 * beams, V), -rng.integers(0, 1 << 17, 2 * beams), 2, beams, n)


def test_select_most_lists(gpu):
    rng = np.random.default_rng(20)
    check_select(logits(rng, 32, 1 << 18), -rng.integers(0, 1 << 16, 32), 1, 32, 64)


@pytest.mark.parametrize("kind", ["equal", "two", "banned", "few", "lowest", "highest", "first", "lane", "last"])
@pytest.mark.parametrize("V", [300, 9001])
def test_select_of_ties_and_bans(gpu, kind, V):
    """Equal logits go by beam and token; banned tokens are never chosen; rows where nothing, or less than n, is left; the best ones all in one
    lane of a wave, or in one span."""
    rng = np.random.default_rng(V)
    groups, beams, n = 3, 4, 20
    z = logits(rng, groups * beams, V)
    if kind == "equal":
        z[...] = 77
    if kind == "two":
        z[...] = np.where(rng.random(z.shape) < 0.5, 5, 6)
    if kind == "banned":
        z[rng.random(z.shape) < 0.5] = km.LOW
        z[1] = z[4:8] = km.LOW
    if kind == "few":
        z[rng.random(z.shape) < 0.99] = km.LOW
    if kind == "lowest":
        z[...] = km.LOW + 1
        z[:, 7] = km.LOW
    if kind == "highest":
        z[:, ::3] = (1 << 31) - 1
        z[:, 1::3] = km.LOW + 1
    if kind == "first":
        z[:, :30] = 1 << 28
    if kind == "lane":
        z[:, 5::64] += 1 << 24
    if kind == "last":
        z[:, -5:] = 1 << 29
    check_select(z, np.zeros(groups * beams, np.int64), groups, beams, n)
    check_select(z, scores(rng, groups * beams, 0.4), groups, beams, n)


def test_select_of_beams_that_are_not_there(gpu):
    rng = np.random.default_rng(21)
    s = np.full(8, km.NONE, np.int64)
    z = logits(rng, 8, 5000)
    check_select(z, s, 2, 4, 8)
    s[4] = 0                       # the first step: one beam of a group
    check_select(z, s, 2, 4, 8)
    s[5], s[6] = (1 << 61) - 1, -(1 << 61) + 1
    check_select(z, s, 2, 4, 8)


@pytest.mark.parametrize("table", ["zero", "one", "most"])
def test_select_tables(gpu, table):
    rng = np.random.default_rng(22)
    lexp = {"zero": np.zeros(1025), "one": np.ones(1025), "most": np.full(1025, 2**31 - 1)}[table].astype(np.int64)
    check_select(logits(rng, 6, 9001), scores(rng, 6), 2, 3, 6, lexp=lexp)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("rows,ctx", [(1, 5), (4, 1000), (37, 300), (300, 40)])
def test_tables_by_parent(gpu, page, rows, ctx):
    rng = np.random.default_rng(rows + page)
    width, ldt = -(-ctx // page), -(-ctx // page) + 2
    length = rng.integers(0, ctx + 1, rows)
    parent = rng.integers(0, rows, rows)
    if rows > 4:
        parent[2], parent[3], length[1], length[4] = -1, rows, -5, ctx + 10 * page
    table, fresh = rng.integers(0, 99999, (rows, ldt)), rng.integers(0, 99999, rows)
    d = {k: dev(np.asarray(v, np.int32)) for k, v in dict(parent=parent, len=length, table=table, fresh=fresh).items()}
    o = dict(out_len=full(rows + 1), out_table=full((rows, ldt)), src=full(rows + 1), dst=full(rows + 1))
    vb.k_beam_tables(vb.BeamTables(rows=rows, page=page, width=width, ldt=ldt, **{k: vg.ptr(v) for k, v in {**d, **o}.items()}))
    want = km.beam_tables(parent, length, table, fresh, page, width)
    got = to_np(o["out_table"])
    assert_equal(got[:, :width], want[0], "table")
    assert (got[:, width:] == JUNK).all()
    for name, w in (("out_len", want[1]), ("src", want[2]), ("dst", want[3])):
        assert_equal(to_np(o[name])[:-1], w, name)
        assert to_np(o[name])[-1] == JUNK


# ---------------------------------------------------------------- together

class Beams:
    """Steps of beam search over a paged cache: `groups` requests of `beams` beams, prompts of different lengths shared by a group's
    beams, and the same with every beam's keys and values in plain arrays."""

    page, heads, D, bits, Hq, V, groups, beams, most = 16, 2, 64, 8, 6, 5000, 3, 4, 96

    def __init__(self, seed):
        self.rng = np.random.default_rng(seed)
        rng, B = self.rng, self.groups * self.beams
        self.width = self.most // self.page
        self.pages = 60 + B * 24
        self.cache = Cache(self.pages, self.page, self.heads, self.D, self.bits, seed)
        self.free = list(rng.permutation(self.pages))
        self.lexp, self.lln = lm.exp_table(), km.ln_table()
        self.m, self.s = km.scale_of(self.D)
        self.length = np.zeros(B, np.int64)
        self.score = np.full(B, km.NONE, np.int64)
        self.score[::self.beams] = 0                   # a group begins with one beam
        self.k = [np.zeros((0, self.heads, self.D), np.int32) for _ in range(B)]
        self.v = [np.zeros((0, self.heads, self.D), np.int32) for _ in range(B)]
        self.rows = B
        i32 = dict(len=B, add=B, new_len=B, start=B + 1, slot=512, pos=512, used=1, nfree=1, free=self.pages, parent=B, fresh=B, src=B, dst=B, out_len=B, rowmax=B)
        self.d = {k: full(n) for k, n in i32.items()}
        self.d.update(table=full((B, self.width), -1), out_table=full((B, self.width), -1), lexp=dev(self.lexp), lln=dev(self.lln), qkv=full((512, (self.Hq + 2 * self.heads) * self.D)),
                      out=full((B, self.Hq * self.D)), z=full((B, self.V)), score=full(B, 0, torch.int64), oscore=full((self.groups, self.beams), 0, torch.int64),
                      oparent=full((self.groups, self.beams)), otoken=full((self.groups, self.beams)))
        self.ws = full((vk.kv_attention_workspace_bytes(B, self.Hq, self.D, self.most) // 4 + 4,))
        self.bws = full((vb.beam_workspace_bytes(self.groups, self.beams, self.V, self.beams) // 4,))

    def set(self, **kw):
        for k, v in kw.items():
            self.d[k].view(-1)[:np.size(v)] = dev(np.asarray(v).astype(to_np(self.d[k]).dtype).reshape(-1))

    def plan_args(self, tokens):
        p = {k: vg.ptr(self.d[k]) for k in ("len", "add", "table", "free", "nfree", "new_len", "start", "slot", "pos", "used")}
        return vk.KvPlan(R=self.rows, tokens=tokens, pages=self.pages, page=self.page, width=self.width, ldt=self.width, **p)

    def attn_args(self):
        C = self.Hq * self.D
        return vk.KvAttn(Q=vg.ptr(self.d["qkv"]), ldq=(self.Hq + 2 * self.heads) * self.D, rows=self.rows, Hq=self.Hq, table=vg.ptr(self.d["table"]), ldt=self.width, width=self.width,
                         len=vg.ptr(self.d["new_len"]), max_len=self.most, m=self.m, s=self.s, Lexp=vg.ptr(self.d["lexp"]), out=vg.ptr(self.d["out"]), ldo=C, rowmax=vg.ptr(self.d["rowmax"]),
                         ws=vg.ptr(self.ws), ws_bytes=self.ws.numel() * 4)

    def launch(self, tokens, stream=None):
        """Plan, rows, attention, selection, tables and copies of one step."""
        d, C, kvD = self.d, self.Hq * self.D, self.heads * self.D
        ld = C + 2 * kvD
        vk.k_kv_plan(self.plan_args(tokens), stream)
        vk.k_kv_write(self.cache.c, vg.ptr(d["qkv"]) + 4 * C, vg.ptr(d["qkv"]) + 4 * (C + kvD), ld, d["slot"], tokens, stream)
        vg.fill_u32(d["rowmax"], stream=stream)
        vk.k_kv_attention(self.cache.c, self.attn_args(), stream)
        vb.k_beam_select(vb.BeamSelect(groups=self.groups, beams=self.beams, V=self.V, n=self.beams, logits=vg.ptr(d["z"]), ldz=self.V, score=vg.ptr(d["score"]), Lexp=vg.ptr(d["lexp"]),
                                       Lln=vg.ptr(d["lln"]), out_score=vg.ptr(d["oscore"]), parent=vg.ptr(d["oparent"]), token=vg.ptr(d["otoken"]), ws=vg.ptr(self.bws),
                                       ws_bytes=self.bws.numel() * 4), stream)
        vb.k_beam_tables(vb.BeamTables(rows=self.rows, page=self.page, width=self.width, ldt=self.width, parent=vg.ptr(d["oparent"]), len=vg.ptr(d["new_len"]), table=vg.ptr(d["table"]),
                                       fresh=vg.ptr(d["fresh"]), out_len=vg.ptr(d["out_len"]), out_table=vg.ptr(d["out_table"]), src=vg.ptr(d["src"]), dst=vg.ptr(d["dst"])), stream)
        vk.k_kv_copy(self.cache.c, d["src"], d["dst"], self.rows, stream)

    def step(self, run, tokens):
        """One step of one token a row through `run`, checked against the plain arrays."""
        rng, B = self.rng, self.rows
        add = np.where(self.score != km.NONE, 1, 0)
        qkv = rows_of(rng, tokens, self.Hq + 2 * self.heads, self.D)
        z = logits(rng, B, self.V)
        fresh, self.free = self.free[:B], self.free[B:]
        listed = self.free[:B]
        self.set(len=self.length, add=add, free=listed, nfree=[len(listed)], z=z, score=self.score, fresh=fresh, qkv=qkv)
        run(self, tokens)
        live = np.nonzero(add)[0]
        used = int(to_np(self.d["used"])[0])
        self.free = self.free[used:]
        for t, r in enumerate(live):
            self.k[r], self.v[r] = np.concatenate([self.k[r], qkv[t:t + 1, self.Hq:self.Hq + self.heads]]), np.concatenate([self.v[r], qkv[t:t + 1, self.Hq + self.heads:]])
        n = self.length + add
        want = []
        for r in range(B):      # row r of the queries belongs to sequence r
            (kq, ek), (vq, ev) = km.quant(self.k[r], self.bits) if n[r] else (self.k[r], np.zeros((0, self.heads))), km.quant(self.v[r], self.bits) if n[r] else (self.v[r], np.zeros((0, self.heads)))
            want.append(km.attend(qkv[r, :self.Hq], kq, ek, vq, ev, np.ones(n[r], bool), self.heads, self.m, self.s, self.lexp).reshape(-1))
        assert_equal(to_np(self.d["out"]), np.array(want), "attention")
        assert_equal(to_np(self.d["rowmax"]), np.abs(np.array(want)).max(1), "rowmax")
        score, parent, token = km.select(z, self.score, self.groups, self.beams, self.beams, self.lexp, self.lln)
        for name, w in (("oscore", score), ("oparent", parent), ("otoken", token)):
            assert_equal(to_np(self.d[name]), w, name)
        parent = parent.reshape(-1)
        self.score = score.reshape(-1)
        self.length = n[parent]
        assert_equal(to_np(self.d["out_len"]), self.length, "lengths")
        self.k, self.v = [self.k[p].copy() for p in parent], [self.v[p].copy() for p in parent]
        self.d["table"].copy_(self.d["out_table"])


def test_beam_search(gpu):
    """Twenty steps, across page ends, of three requests of four beams that begin with one."""
    b = Beams(30)
    for _ in range(20):
        b.step(lambda s, t: s.launch(t), 16)


def test_beam_search_captured(gpu):
    """The same launches captured once and replayed, with the step's work of the program between the replays."""
    b = Beams(31)
    b.step(lambda s, t: s.launch(t), 16)
    st = torch.cuda.Stream()
    g = vg.Graph(st)
    torch.cuda.synchronize()
    g.begin()
    b.launch(16, stream=st)
    g.end()

    def replay(s, t):
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()

    for _ in range(18):
        b.step(replay, 16)


def test_two_streams_at_once(gpu):
    """Two decoders on streams of their own, with caches and workspaces of their own."""
    a = [Attend(np.random.default_rng(40 + i), [900, 20, 512], 16, 2, 64, 8 + 8 * i, 8) for i in range(2)]
    want = [x.want() for x in a]
    args = [x.args() for x in a]
    streams = [torch.cuda.Stream() for _ in a]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, A, st in zip(a, args, streams):
            vk.k_kv_attention(x.cache.c, A, st)
    torch.cuda.synchronize()
    for x, w in zip(a, want):
        assert_equal(to_np(x.d["out"]), w)


# ---------------------------------------------------------------- every form of the kernels

DEALT = 1 << 16   # a max_len that makes every call one whose spans are dealt over the card's blocks, whatever the lengths


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D", [16, 64, 80, 128, 144, 192, 208, 256])
@pytest.mark.parametrize("window", [0, 300])
def test_attention_dealt(gpu, bits, D, window):
    """Heads of every register form, sizes that fill their pieces and that do not; rows without tokens among the others."""
    rng = np.random.default_rng(D + bits)
    lens = rng.integers(0, 900, 20)
    lens[[0, 7, 19]] = 0
    a = Attend(rng, lens, 16, 2, D, bits, 6)
    a.check(window=window)
    a.check(window=window, max_len=DEALT if not window else 900)


@pytest.mark.parametrize("rows", [255, 256, 257, 700, 2048, 2049])
def test_attention_dealt_over_many_rows(gpu, rows):
    """Running sums of one and of several rows a thread, up to the most that are dealt and past them."""
    rng = np.random.default_rng(rows)
    lens = np.where(rng.random(rows) < 0.5, 0, rng.integers(0, 300, rows))
    lens[rng.integers(0, rows, 3)] = [1500, 900, 513]
    a = Attend(rng, lens, 64, 1, 16, 8, 1)
    a.check(max_len=DEALT)
    a.check(window=400)


def test_attention_dealt_without_any_tokens(gpu):
    a = Attend(np.random.default_rng(50), np.zeros(300, np.int64), 16, 4, 64, 8, 8)
    a.check(max_len=DEALT)


def test_attention_dealt_over_absent_pages(gpu):
    a = Attend(np.random.default_rng(51), [1000, 800, 600, 300, 20], 16, 2, 64, 8, 4)
    a.table[0, 3], a.table[0, 20], a.table[0, 62] = -1, a.cache.c.pages, -(1 << 31)
    a.table[1, 16:32] = -1
    a.table[2, :38] = 1 << 30
    a.check(max_len=DEALT)


@pytest.mark.parametrize("D", [16, 48, 80, 128, 256])
@pytest.mark.parametrize("rows,Hq", [(5, 2), (130, 2)])
def test_attention_joins(gpu, D, rows, Hq):
    """Heads cut into dimensions where few join many spans, and whole; more spans than a block weighs at a time."""
    rng = np.random.default_rng(D + rows)
    lens = rng.integers(0, 600, rows)
    lens[rows // 2] = 5000 if rows > 5 else 140000 if D == 16 else 20000
    a = Attend(rng, lens, 256, 1, D, 8, Hq)
    a.check(max_len=max(20000, int(lens.max())), pad=4)


@pytest.mark.parametrize("kind", ["random", "equal", "two", "banned", "lane", "last"])
def test_select_of_many_spans(gpu, kind):
    """A wave a span, its best ones by threshold and one after the other."""
    rng = np.random.default_rng(52)
    groups, beams, n, V = 70, 4, 12, 33003
    z = logits(rng, groups * beams, V)
    if kind == "equal":
        z[...] = -5
    if kind == "two":
        z[...] = np.where(rng.random(z.shape) < 0.5, 5, 6)
    if kind == "banned":
        z[rng.random(z.shape) < 0.999] = km.LOW
        z[1] = z[4:8] = km.LOW
    if kind == "lane":
        z[:, 8:12] += 1 << 24
        z[:, 264:268] += 1 << 24
        z[:, 520:524] += 1 << 24
        z[:, 776:780] += 1 << 24
    if kind == "last":
        z[:, -5:] = 1 << 29
    check_select(z, scores(rng, groups * beams, 0.2), groups, beams, n, pad=1)


def test_select_of_scores_far_apart(gpu):
    """The best beams have fewer tokens than are asked for, the next lies 2^40 and more below: no key tells them apart."""
    rng = np.random.default_rng(53)
    for V in (3, 20):
        s = np.array([0, -(1 << 41), -(1 << 50), (1 << 61) - 1, 5, 5, 5, -(1 << 61) + 1], np.int64)
        check_select(logits(rng, 8, V), s, 2, 4, 4 * V if 4 * V <= 64 else 64)
        check_select(logits(rng, 8, V), np.array([0, -(1 << 40), -(1 << 40) + 1, -(1 << 40) - 1] * 2, np.int64), 2, 4, min(4 * V, 64))


def test_select_of_more_ties_than_are_kept(gpu):
    rng = np.random.default_rng(54)
    z = np.full((64, 9001), 4, np.int32)
    check_select(z, np.zeros(64, np.int64), 2, 32, 64)
    z[:, 7::50] = 5
    check_select(z, np.repeat([0, 1], 32).astype(np.int64), 2, 32, 64)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D", [16, 80, 128, 256])
@pytest.mark.parametrize("M", [2047, 4100])
def test_rows_of_prompts(gpu, bits, D, M):
    """Runs of tokens that begin at every place of a group, with rows left out, and tokens in any order: words and single bytes."""
    rng = np.random.default_rng(D + M)
    page, heads = 32, 2
    pages = M // page + 20
    order = rng.permutation(pages)
    slot, t = [], 0
    while len(slot) < M:
        run = int(rng.integers(1, 70))
        at = int(rng.integers(0, 4)) + t
        slot += [int(order[p // page]) * page + p % page for p in range(at, at + run) if p < pages * page]
        t = at + run
        if t >= pages * page - 80:
            break
    rest = rng.permutation(np.setdiff1d(np.arange(pages * page), slot))
    slot = np.concatenate([np.array(slot[:M]), rest[:max(0, M - len(slot))]]).astype(np.int32)
    M = len(slot)
    slot[rng.random(M) < 0.05] = -1
    k, v = (rows_of(rng, M, heads, D, True).reshape(M, -1) for _ in range(2))
    C, ds = Cache(pages, page, heads, D, bits), dev(slot)
    before = C.values()
    vk.k_kv_write(C.c, dev(k), dev(v), heads * D, ds, M)
    after = C.values()
    there = slot >= 0
    ko, vo = full((M, heads * D)), full((M, heads * D))
    vk.k_kv_read(C.c, ds, M, ko, vo, heads * D)
    for x, o, i in ((k, ko, 0), (v, vo, 2)):
        q, e = km.quant(x.reshape(M, heads, D), bits)
        before[i][slot[there]], before[i + 1][slot[there]] = q[there], e[there]
        assert_equal(after[i], before[i])
        assert_equal(after[i + 1], before[i + 1])
        assert_equal(to_np(o), np.where(there[:, None], lm.sat32(q << e[..., None]).reshape(M, -1), 0))


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("M", [70, 4200])
def test_rows_read_alone(gpu, bits, M):
    """Keys without values and values without keys, of few and of many tokens; the other output and what lies between the rows stay."""
    rng = np.random.default_rng(M)
    page, heads, D, pad = 64, 3, 80, 12
    pages = M // page + 2
    slot = rng.permutation(pages * page)[:M].astype(np.int32)
    slot[50:] = np.sort(slot[50:])
    slot[::17] = -1
    k, v = (rows_of(rng, M, heads, D).reshape(M, -1) for _ in range(2))
    C, ds = Cache(pages, page, heads, D, bits), dev(slot)
    vk.k_kv_write(C.c, dev(k), dev(v), heads * D, ds, M)
    for x, i in ((k, 0), (v, 1)):
        o = full((M, heads * D + pad))
        vk.k_kv_read(C.c, ds, M, o if i == 0 else None, None if i == 0 else o, heads * D + pad)
        q, e = km.quant(x.reshape(M, heads, D), bits)
        want = np.full((M, heads * D + pad), JUNK, np.int64)
        want[:, :heads * D] = np.where((slot >= 0)[:, None], lm.sat32(q << e[..., None]).reshape(M, -1), 0)
        assert_equal(to_np(o), want)


def test_shared_pages(gpu):
    """The same pages in the tables of several sequences, twice in one table, and the same slot read many times."""
    a = Attend(np.random.default_rng(55), [300, 300, 64, 300], 16, 2, 64, 8, 4)
    a.table[1] = a.table[0]
    a.table[3, :19] = np.repeat(a.table[0, :1], 19)
    a.table[2, 1] = a.table[2, 0]
    a.check()
    M = 40
    ds, ko, vo = dev(np.full(M, int(a.table[0, 0]) * 16 + 5, np.int32)), full((M, 128)), full((M, 128))
    vk.k_kv_read(a.cache.c, ds, M, ko, vo, 128)
    kq, ek, vq, ev = a.cache.values()
    s = int(a.table[0, 0]) * 16 + 5
    assert_equal(to_np(ko), np.repeat((kq[s] << ek[s][:, None]).reshape(1, -1), M, 0))
    assert_equal(to_np(vo), np.repeat((vq[s] << ev[s][:, None]).reshape(1, -1), M, 0))


def test_attention_over_two_million_tokens(gpu):
    """A table that names the same pages again and again: 8192 spans."""
    rng = np.random.default_rng(56)
    a = Attend(rng, [700, 300], 256, 1, 16, 8, 2)
    n = (1 << 21) - 100
    pages = a.table[0, :2].copy()      # the filled ones: a slot that no call has written has no value
    a.table = np.full((2, n // 256 + 1), -1, np.int32)
    a.table[0] = rng.choice(pages, a.table.shape[1])
    a.table[1, :2] = pages[:2]
    a.lens, a.width = np.array([n, 300]), a.table.shape[1]
    a.check()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D", [16, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("Hq", [2, 10, 24, 40])
def test_attention_of_few_spans(gpu, bits, D, Hq):
    """Sequences whose spans one block takes two at a time and joins: every number of them up to four, some without tokens, a team without a span."""
    rng = np.random.default_rng(D + Hq)
    a = Attend(rng, [0, 1, 256, 257, 512, 513, 768, 769, 1024, 300], 32, 2, D, bits, Hq, extreme=Hq == 10)
    a.check(pad=4)
    a.check(window=300)
    a.check(window=1)
    a.check(max_len=400)


def test_attention_of_few_spans_that_are_absent(gpu):
    a = Attend(np.random.default_rng(57), [1000, 1000, 600, 300, 20], 16, 2, 64, 8, 4)
    a.table[0, 16:32] = -1                      # spans between, first, last and all
    a.table[1, :16] = a.table[1, 48:] = -1
    a.table[2, :38] = 1 << 30
    a.table[3, 16:] = a.cache.c.pages
    a.check()
    a.lexp = np.zeros(1025, np.int64)
    a.check()
    a.lexp = (np.arange(1025) % 2 * (2**31 - 1)).astype(np.int64)
    a.check()


class Turns(Attend):
    """Sequences of any length over a few filled pages, whose tables name them in turn."""

    def __init__(self, rng, lens, D, bits, Hq, filled=80):
        super().__init__(rng, [16 * filled], 16, 1, D, bits, Hq)
        self.lens = np.asarray(lens)
        pages = self.table[0, :filled].copy()
        self.width = -(-int(self.lens.max()) // 16)
        self.table = rng.choice(pages, (len(lens), self.width)).astype(np.int32)
        self.q = rows_of(rng, len(lens), Hq, D)


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 128, 144, 256])
@pytest.mark.parametrize("window", [0, 4400])
def test_attention_joins_every_number_of_spans(gpu, D, window):
    """From two spans a sequence up to the 64 that a wave joins, each with a ragged last one: the weight of every span reaches every lane."""
    rng = np.random.default_rng(D + window)
    lens = 256 * np.arange(1, 64) + rng.integers(1, 257, 63)
    a = Turns(rng, lens, D, 8 if D % 32 else 16, 2)
    a.check(window=window, max_len=16384)
    if window:
        a.check(window=window, max_len=40000)   # a workspace of more spans than the window has


@pytest.mark.parametrize("D", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("n", [2049, 2400, 4097, 4352, 4353, 7200, 7425, 9000, 16384])
def test_attention_joins_one_sequence(gpu, D, n):
    Turns(np.random.default_rng(n), [n], D, 8, 6).check(max_len=16384)


@pytest.mark.parametrize("below", [1, 2, 100, 254, 255, 256, 257, 258, 1000])
@pytest.mark.parametrize("beams,n", [(2, 2), (2, 1), (5, 5), (32, 40), (3, 64)])
def test_select_of_scores_at_the_end_of_the_keys(gpu, below, beams, n):
    """One token a beam, the first beam's score 2^40 - below above the others', and below their neighbours': those that a key can hold and those that it cannot."""
    z = np.zeros((2 * beams, 1), np.int32)
    s = np.zeros((2, beams), np.int64)
    s[0, 1:] = below - (1 << 40)
    s[1, 1:] = below - (1 << 40) + np.arange(beams - 1) * 100 - 200
    check_select(z, s.reshape(-1), 2, beams, n)


@pytest.mark.parametrize("V,n", [(3, 6), (4, 8), (40, 64), (9000, 64)])
def test_select_of_lists_across_the_end_of_the_keys(gpu, V, n):
    """Lists whose entries lie on both sides of what a key holds, behind ones that no key holds, with banned tokens so that all of them are asked for."""
    rng = np.random.default_rng(V)
    z = np.full((4, V), km.LOW, np.int32)
    for r in range(4):
        at = rng.permutation(V)[:min(V, 20)]
        z[r, at] = -20 * rng.integers(0, 20, at.size)
    for below in (100, 300, 500):
        check_select(z, np.array([0, below - (1 << 40), 0, below - (1 << 40) - 7], np.int64), 2, 2, n)


@pytest.mark.parametrize("page", [16, 64])
def test_tables_by_parent_of_absent_pages(gpu, page):
    """A partly filled last page that is none (a plan's list had ended) stays none: a fresh page in its place would hold nothing that was written."""
    rng = np.random.default_rng(page)
    rows, width = 60, 6
    length = rng.integers(0, width * page + 1, rows)
    parent = rng.integers(0, rows, rows)
    table, fresh = rng.integers(0, 999, (rows, width)), rng.integers(0, 999, rows)
    table[rng.random(table.shape) < 0.4] = -1
    table[length == 0] = -1
    table[7] = -(1 << 31)
    parent[:4] = 7
    length[7] = 3 * page + 5
    d = {k: dev(np.asarray(v, np.int32)) for k, v in dict(parent=parent, len=length, table=table, fresh=fresh).items()}
    o = dict(out_len=full(rows), out_table=full((rows, width)), src=full(rows), dst=full(rows))
    vb.k_beam_tables(vb.BeamTables(rows=rows, page=page, width=width, ldt=width, **{k: vg.ptr(v) for k, v in {**d, **o}.items()}))
    out, new, src, dst = km.beam_tables(parent, length, table, fresh, page, width)
    absent = (new % page > 0) & (src < 0)
    assert absent[:4].all() and absent.sum() > 10 and (dst >= 0).sum() > 10
    out[absent, new[absent] // page] = src[absent] = dst[absent] = -1
    for name, w in (("out_table", out), ("out_len", new), ("src", src), ("dst", dst)):
        assert_equal(to_np(o[name]), w, name)


def test_attention_after_tables_of_absent_pages(gpu):
    """Tokens that found no page do not count before their beams are reordered, and do not after it."""
    a = Attend(np.random.default_rng(60), [40, 40, 300, 300], 16, 2, 64, 8, 4)
    a.table[1, 2] = a.table[3, 18] = -1
    a.check()
    spare = np.setdiff1d(np.arange(a.cache.c.pages), a.table[a.table >= 0])   # pages that hold anything
    parent = np.array([1, 1, 3, 2], np.int32)
    d = dict(parent=dev(parent), len=dev(a.lens.astype(np.int32)), table=dev(a.table), fresh=dev(np.resize(spare, 4).astype(np.int32)))
    o = dict(out_len=full(4), out_table=full(a.table.shape), src=full(4), dst=full(4))
    vb.k_beam_tables(vb.BeamTables(rows=4, page=16, width=a.width, ldt=a.table.shape[1], **{k: vg.ptr(v) for k, v in {**d, **o}.items()}))
    vk.k_kv_copy(a.cache.c, o["src"], o["dst"], 4)
    want = a.want()[[1, 1, 3, 2]]            # of the parents' queries
    a.q, a.lens = a.q[parent], to_np(o["out_len"])
    a.table[:, :a.width] = to_np(o["out_table"])[:, :a.width]
    out = a.want()
    assert_equal(out, want, "tables")
    a.check()

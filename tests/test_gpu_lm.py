"""The language-model operators on the GPU against their formulas in 64-bit integers (tests/lm_math.py). Every result is a
whole number: the comparison is equality."""
import numpy as np
import pytest
import torch

from tests import lm_math as lm
from tests.conftest import assert_equal, to_np
from vela_amd import gemm as vg
from vela_amd import moe as vm
from vela_amd import norms as vn
from vela_amd import w4 as vw

pytestmark = pytest.mark.gpu

DEN = 100000
GUARD = -123456789   # what the cells behind an output hold before and after


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def out32(shape, extra=64):
    """An int32 output [shape] inside a larger buffer whose remainder must keep its value."""
    n = int(np.prod(shape))
    buf = torch.full((n + extra,), GUARD, dtype=torch.int32, device="cuda")
    return buf, buf[:n].view(*shape)


def check_guard(buf, n, what):
    assert bool((buf[n:] == GUARD).all()), f"{what}: cells behind the output were written"


# ---------------------------------------------------------------- norm

def run_norm(x, r, g, Kp, view, alias=None, den=DEN):
    M, C = x.shape
    dx, dr, dg = dev(x), (dev(r) if r is not None else None), dev(g)
    H = {None: torch.empty_like(dx), "x": dx, "r": dr, "none": None}[alias]
    hi = torch.full((M, Kp), 77, dtype=torch.int8, device="cuda")
    lo = torch.full((M, Kp), 77, dtype=torch.int8, device="cuda") if view else None
    e = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    vn.k_rmsnorm_q(dx, dr, M, C, dg, den, H, hi, lo, e, Kp)
    torch.cuda.synchronize()
    return (to_np(H) if H is not None else None), to_np(hi), (to_np(lo) if view else None), to_np(e)


def check_norm(x, r, g, Kp, view, alias=None, den=DEN, what=""):
    C = x.shape[1]
    h, y = lm.rmsnorm(x, r, g, den)
    H, hi, lo, e = run_norm(x, r, g, Kp, view, alias, den)
    q, we = lm.quant(y, 15 if view else 7)
    if H is not None:
        assert_equal(H, h, what + " h")
    assert_equal(e, we, what + " e")
    got = 256 * hi.astype(np.int64) + lo + 128 if view else hi.astype(np.int64)
    assert_equal(got[:, :C], q, what + " q")
    assert not got[:, C:].any(), what + " pads"


@pytest.mark.parametrize("view", [False, True])
@pytest.mark.parametrize("M,C,Kp", [(1, 4, 4), (1, 2048, 2048), (3, 252, 256), (5, 256, 272), (2, 260, 260), (7, 512, 512), (4, 516, 528), (9, 1024, 1024),
                                    (2, 1028, 1040), (3, 2052, 2064), (2, 4096, 4096), (3, 4100, 4112), (2, 8188, 8192), (2, 8192, 8192)])
def test_norm_sizes(gpu, M, C, Kp, view):
    rng = np.random.default_rng(M * 10000 + C)
    x = np.round(rng.normal(size=(M, C)) * 150000).astype(np.int32)
    r = np.round(rng.normal(size=(M, C)) * 70000).astype(np.int32)
    g = rng.integers(-90000, 90000, C, dtype=np.int32)
    check_norm(x, r, g, Kp, view, what=f"{M}x{C}")


@pytest.mark.parametrize("kind", ["zero", "one", "small", "spike", "huge", "saturating", "minint", "constant", "big_gain"])
@pytest.mark.parametrize("C", [64, 1500, 4096])
def test_norm_values(gpu, kind, C):
    """Rows of nothing, of single values, of the widest values and saturating sums, and gains that saturate the output."""
    rng = np.random.default_rng(C)
    x, r = np.zeros((4, C), np.int32), np.zeros((4, C), np.int32)
    g = rng.integers(30000, 100000, C, dtype=np.int32)
    if kind == "one":
        x[:, 5] = [1, -1, 3, 100]
    elif kind == "small":
        x[...] = rng.integers(-3, 4, x.shape)
    elif kind == "spike":
        x[...] = rng.integers(-50, 51, x.shape)
        x[:, 7] = [2**31 - 1, -(2**31), 2**30, -(2**20)]
    elif kind == "huge":
        x[...] = rng.integers(-(2**31), 2**31, x.shape)
    elif kind == "saturating":
        x[...] = np.where(rng.random(x.shape) < 0.5, 2**31 - 1, -(2**31))
        r[...] = np.where(rng.random(x.shape) < 0.5, 2**31 - 1, -(2**31))
    elif kind == "minint":
        x[...] = -(2**31)
    elif kind == "constant":
        x[...] = np.array([[12345], [-7], [2**25], [-(2**31) + 1]])
    elif kind == "big_gain":
        x[...] = rng.integers(-90000, 90000, x.shape)
        g = np.where(rng.random(C) < 0.5, 2**31 - 1, -(2**31)).astype(np.int32)
    for view in (False, True):
        check_norm(x, r, g, C, view, what=kind)
    check_norm(x, None, g, C, False, alias="none", what=kind + " without residual")
    check_norm(x, r, g, C, False, den=1 << 40, what=kind + " epsilon 0")


@pytest.mark.parametrize("alias", ["x", "r", "none"])
@pytest.mark.parametrize("M,C", [(6, 320), (3, 5120)])
def test_norm_aliases(gpu, alias, M, C):
    rng = np.random.default_rng(11)
    x, r = (np.round(rng.normal(size=(M, C)) * 100000).astype(np.int32) for _ in range(2))
    check_norm(x, r, rng.integers(1, 90000, C, dtype=np.int32), C, False, alias=alias, what=alias)


def test_norm_many_rows(gpu):
    rng = np.random.default_rng(12)
    for M, C in ((1031, 128), (515, 640), (700, 1280)):
        x = (rng.normal(size=(M, C)) * np.exp(rng.normal(size=(M, 1)) * 3) * 60000).round().clip(-2**31, 2**31 - 1).astype(np.int32)
        check_norm(x, None, rng.integers(1, 90000, C, dtype=np.int32), C, False, what=f"{M}x{C}")


# ---------------------------------------------------------------- 4-bit products

def packed(w: lm.Weights):
    W = vw.W4Weights(w.N, w.K, w.group, count=w.count or 1)
    W.pack(dev(w.nib), dev(w.sc), dev(w.z) if w.z is not None else None, dev(w.msb))
    return W


class Rows:
    """Rows of one of the three kinds on the device, with the values they stand for."""

    def __init__(self, rng, kind, M, K, pad=0, full=False, shifts=True):
        ld = lm.up(K, 16) + pad
        self.keep = []
        if kind == "x32":
            x = np.round(rng.normal(size=(M, K + pad)) * np.exp(rng.normal(size=(M, 1)) * 3) * 3000).clip(-2**31, 2**31 - 1).astype(np.int32)
            if full:
                x = rng.integers(-(2**31), 2**31, x.shape).astype(np.int32)
            self.q, self.e = lm.quant(x[:, :K].astype(np.int64), 15)
            rm = np.abs(x[:, :K].astype(np.int64)).max(1).astype(np.uint32).view(np.int32)
            self.keep = [dev(x), dev(rm)]
            self.A = vg.ASrc(src=vg.SRC_X32, x=vg.ptr(self.keep[0]), ldx=K + pad, rowmax=vg.ptr(self.keep[1]), K=K)
            return
        if kind == "q8":
            hi, e = lm.rows8(rng, M, K, ld, full)
            self.q, planes = hi[:, :K].astype(np.int64), [hi]
        else:
            hi, lo, self.q, e = lm.rows16(rng, M, K, ld, full)
            planes = [hi, lo]
        self.e = e.astype(np.int64) if shifts else np.zeros(M, np.int64)
        self.keep = [dev(p) for p in planes] + [dev(e)]
        self.A = vg.ASrc(src=vg.SRC_I8, hi=vg.ptr(self.keep[0]), lo=vg.ptr(self.keep[1]) if kind == "q16" else None, ld8=ld, K=K,
                         e=vg.ptr(self.keep[-1]) if shifts else None)


def check_w4(rng, kind, M, N, K, group, epi="plain", residual=False, rowmax=True, pad=0, full=False, shifts=True, ldpad=0, **kw):
    w = lm.Weights(rng, N, K, group, pad=pad, **kw)
    rows = Rows(rng, kind, M, K, pad=16 * pad, full=full, shifts=shifts)
    W = packed(w)
    out = N // 2 if epi == "geglu" else N
    ldy = out + ldpad
    want = lm.product(rows.q, rows.e, w.dense(), w.msb)
    lut = lm.sigmoid_table()
    dlut = dev(lut)
    if epi == "geglu":
        want = lm.geglu(want, lut)
    buf, Y = out32((M, ldy))
    if residual:
        res = rng.integers(-(2**31), 2**31, (M, ldy)).astype(np.int32)
        Y.copy_(dev(res))
        want = lm.sat32(want + res[:, :N])
    rm0 = rng.integers(0, 1 << 17, M, dtype=np.int32)
    rm = dev(rm0) if rowmax else None
    E = vg.AEpi(epi=vg.EPI_GEGLU if epi == "geglu" else vg.EPI_PLAIN, Y=vg.ptr(Y), ldy=ldy, residual=vg.ptr(Y) if residual else None,
                Lphi=vg.ptr(dlut), rowmax=vg.ptr(rm))
    vw.k_gemm_w4(rows.A, M, W, E)
    torch.cuda.synchronize()
    got = to_np(Y)
    what = f"{kind} {M}x{K}x{N} group {group} {epi}"
    assert_equal(got[:, :out], want, what)
    if ldpad:
        assert_equal(got[:, out:], res[:, out:] if residual else np.full((M, ldpad), GUARD), what + " columns past N")
    check_guard(buf, M * ldy, what)
    if rowmax:
        assert_equal(to_np(rm).view(np.uint32), np.maximum(rm0, np.abs(want).max(1)).astype(np.uint32), what + " rowmax")


KINDS = ["q8", "q16", "x32"]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_w4_types(gpu, kind, group):
    rng = np.random.default_rng(group)
    for M, K, N in ((1, 256, 64), (5, 640, 100), (16, 384, 33), (1, 2048, 256)):
        check_w4(rng, kind, M, N, K, group)
        check_w4(rng, kind, M, N // 2 * 2, K, group, epi="geglu")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 48, 49, 63, 64, 65, 130])
def test_w4_rows(gpu, kind, M):
    rng = np.random.default_rng(M)
    check_w4(rng, kind, M, 72, 512, 32 << (M % 3), residual=M % 2 == 0, ldpad=3)


@pytest.mark.parametrize("kind,K", [("q8", 1), ("q8", 31), ("q16", 33), ("x32", 4), ("x32", 100), ("q8", 127), ("q16", 129), ("x32", 132), ("q8", 255),
                                    ("q16", 1000), ("x32", 1996), ("q8", 4095)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_depths(gpu, kind, K, group):
    """Depths that end inside a group, a tile or a byte; junk in the padding columns of rows and weights."""
    rng = np.random.default_rng(K)
    check_w4(rng, kind, 3, 40, K, group, pad=2)


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 50, 1000, 5001])
def test_w4_columns(gpu, N):
    rng = np.random.default_rng(N)
    check_w4(rng, "q8", 4, N, 256, 64, ldpad=1, residual=True)
    if N % 2 == 0:
        check_w4(rng, "q16", 4, N, 256, 64, epi="geglu", ldpad=1)


@pytest.mark.parametrize("kind,M,K,N", [("q16", 48, 5000, 40), ("q8", 64, 9000, 24), ("x32", 16, 12000, 24), ("q16", 16, 9999, 24), ("q8", 33, 20000, 16),
                                        ("x32", 64, 4100, 40), ("q8", 7, 64, 40000), ("q16", 30, 128, 35001), ("x32", 3, 192, 33000)])
def test_w4_chunks_and_segments(gpu, kind, M, K, N):
    """Rows that pass the staging area in several chunks of K; blocks of several column tiles, the last ones short."""
    check_w4(np.random.default_rng(K + N), kind, M, N, K, 64, residual=True)


@pytest.mark.parametrize("kind,M,K,N", [("q8", 3, 33, 70001), ("x32", 1, 64, 150000), ("q16", 40, 32, 20002), ("x32", 100, 16, 9000), ("q8", 17, 64, 34000), ("q16", 33, 200, 4096),
                                        ("q8", 1000, 20, 70), ("q16", 700, 40, 33), ("x32", 4100, 8, 20)])
def test_w4_many_columns_or_rows(gpu, kind, M, K, N):
    """Segments of many column tiles, more blocks than CUs, more row tiles than CUs."""
    check_w4(np.random.default_rng(M + N), kind, M, N, K, 64, residual=True)


def test_w4_most_rows(gpu):
    """As many rows as a call takes, eight and sixteen a block: every row as the first ones repeat."""
    M, n = 1 << 18, 64
    for kind in ("x32", "q8"):
        rng = np.random.default_rng(18)
        few, w = Rows(rng, kind, n, 16), lm.Weights(rng, 5, 16, 32)
        W, times = packed(w), lambda t: t.repeat(M // n, *([1] * (t.dim() - 1)))  # noqa: E731
        keep = [times(t) for t in few.keep]
        if kind == "x32":
            A = vg.ASrc(src=vg.SRC_X32, x=vg.ptr(keep[0]), ldx=keep[0].shape[1], rowmax=vg.ptr(keep[1]), K=16)
        else:
            A = vg.ASrc(src=vg.SRC_I8, hi=vg.ptr(keep[0]), ld8=keep[0].shape[1], e=vg.ptr(keep[-1]), K=16)
        y = torch.empty((M, 5), dtype=torch.int32, device="cuda")
        vw.k_gemm_w4(A, M, W, vg.AEpi(Y=vg.ptr(y), ldy=5))
        want = dev(lm.product(few.q, few.e, w.dense(), w.msb).astype(np.int32))
        assert torch.equal(y.view(M // n, n, 5), want.expand(M // n, n, 5))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_extremes(gpu, kind, group):
    """The widest rows, codes, scales and constants at the deepest K: sums near 2^46, products that wrap in 64 bits, shifts
    from saturating left ones to ones past 62."""
    rng = np.random.default_rng(7)
    check_w4(rng, kind, 2, 20, 32768, group, full=True, scale=(4095, 4096), m=(1 << 30, (1 << 31) - 1), s=30, b=2**31 - 1)
    check_w4(rng, kind, 2, 20, 512, group, full=True, scale=(-32768, 32767), m=(-(1 << 31), 1 << 31), s=0)
    check_w4(rng, kind, 2, 20, 512, group, full=True, m=(1, 1 << 20), s=64, shifts=False)


def test_w4_symmetric_and_no_rowmax(gpu):
    rng = np.random.default_rng(8)
    for kind in KINDS:
        check_w4(rng, kind, 3, 48, 320, 64, zeros=False, rowmax=False)


def test_w4_zero_weights_and_rows(gpu):
    """Scales of 0 and rows of 0: only the columns' b remains; int32 rows of zeros with row maximum 0."""
    rng = np.random.default_rng(9)
    check_w4(rng, "q16", 3, 48, 320, 64, scale=(0, 1))
    w = lm.Weights(rng, 32, 128, 128)
    W = packed(w)
    x, rm = torch.zeros((2, 128), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    y = torch.empty((2, 32), dtype=torch.int32, device="cuda")
    vw.k_gemm_w4(vg.ASrc(src=vg.SRC_X32, x=vg.ptr(x), ldx=128, rowmax=vg.ptr(rm), K=128), 2, W, vg.AEpi(Y=vg.ptr(y), ldy=32))
    assert_equal(to_np(y), np.broadcast_to(w.msb[:, 2], (2, 32)))


def test_w4_pack_parts_of_a_stack(gpu):
    """Matrices laid out one by one, in any order, equal the stack laid out at once."""
    rng = np.random.default_rng(10)
    w = lm.Weights(rng, 40, 200, 64, count=5)
    whole, parts = packed(w), vw.W4Weights(40, 200, 64, count=5)
    for i in (3, 0, 4, 1, 2):
        parts.pack(dev(w.nib[i]), dev(w.sc[i]), dev(w.z[i]), dev(w.msb[i]), first=i)
    assert torch.equal(whole.q, parts.q) and torch.equal(whole.cst, parts.cst)


@pytest.mark.parametrize("N,count", [(1, 4), (1, 1), (5, 3), (5, 1)])
def test_w4_pack_strided_sources(gpu, N, count):
    """Slices of wider tensors, scale and zero points of different pitch, every second matrix of a stack, rows broadcast over
    the columns, on a stream of its own: as from dense rows."""
    rng = np.random.default_rng(17 + N)
    w = lm.Weights(rng, N, 200, 64, count=count)
    dense = packed(w)
    wide = lambda a, extra: torch.nn.functional.pad(dev(a), (3, extra))[..., 3:3 + a.shape[-1]]  # noqa: E731
    second = lambda a: torch.stack([dev(a), torch.zeros_like(dev(a))], 1).flatten(0, 1)[::2]  # noqa: E731
    same = lambda W: torch.equal(W.q, dense.q) and torch.equal(W.cst, dense.cst)  # noqa: E731
    st = torch.cuda.Stream()
    for nib, sc, z, msb in ((wide(w.nib, 7), wide(w.sc, 2), wide(w.z, 5), wide(w.msb, 1)), (second(w.nib), second(w.sc), second(w.z), second(w.msb)),
                            (wide(w.nib, 0), dev(w.sc), wide(w.z, 0), dev(w.msb))):
        for stream in (None, st, st.cuda_stream):
            W = vw.W4Weights(N, 200, 64, count=count)
            W.q.zero_(), W.cst.zero_()
            torch.cuda.synchronize()
            W.pack(nib, sc, z, msb, stream=stream)
            torch.cuda.synchronize()
            assert same(W)
    one = vw.W4Weights(N, 200, 64, count=count)
    one.pack(dev(w.nib), dev(w.sc[..., :1, :]).expand(*w.sc.shape), None, dev(w.msb))
    dense.pack(dev(w.nib), dev(np.broadcast_to(w.sc[..., :1, :], w.sc.shape).copy()), dev(np.full_like(w.z, 8)), dev(w.msb))
    assert same(one)


# ---------------------------------------------------------------- mixture of experts

class Layer:
    def __init__(self, rng, M, E, topk, D, F, group=64, group2=None, renorm=True, kind="q8", equal=False):
        self.M, self.E, self.topk, self.D, self.F, self.renorm, self.kind = M, E, topk, D, F, renorm, kind
        self.rows = Rows(rng, kind, M, D)
        self.rw = rng.integers(-127, 128, (E, D + 16)).astype(np.int8)
        if equal:
            self.rw[...] = self.rw[:1]
        self.cst = np.zeros((E, 4), np.int32)
        self.cst[:, 0] = rng.integers(1 << 14, 1 << 15, E) if not equal else 1 << 14
        self.cst[:, 1] = 22 + (8 if kind == "q16" else 0)
        self.cst[:, 2] = rng.integers(-9000, 9000, E) if not equal else 5
        self.cst[:, 3] = self.rw[:, :D].sum(1, dtype=np.int64)
        self.up = lm.Weights(rng, 2 * F, D, group, count=E, s=28 + (8 if kind == "q16" else 0))
        self.down = lm.Weights(rng, D, F, group2 or group, count=E)
        self.res = rng.integers(-(10**6), 10**6, (M, D)).astype(np.int32)
        self.lut, self.lexp = lm.sigmoid_table(), lm.exp_table()
        self.d = {n: dev(getattr(self, n)) for n in ("rw", "cst", "lut", "lexp", "res")}
        self.U, self.V = packed(self.up), packed(self.down)
        self.idx = torch.full((M, topk), -7, dtype=torch.int32, device="cuda")
        self.p = torch.full((M, topk), -7, dtype=torch.int32, device="cuda")
        self.logits = torch.full((M, E), -7, dtype=torch.int32, device="cuda")
        self.ybuf, self.y = out32((M, D))
        self.ws = torch.empty(vm.moe_workspace_bytes(M, topk, F) // 4, dtype=torch.int32, device="cuda")

    def route_args(self, logits=True):
        return vm.MoeRoute(W=vg.ptr(self.d["rw"]), ldw=self.D + 16, cst=vg.ptr(self.d["cst"]), experts=self.E, topk=self.topk, renorm=int(self.renorm),
                           Lexp=vg.ptr(self.d["lexp"]), idx=vg.ptr(self.idx), p=vg.ptr(self.p), logits=vg.ptr(self.logits) if logits else None)

    def moe_args(self, residual=True, idx=None, p=None):
        return vm.MoeArgs(up=self.U.desc, down=self.V.desc, topk=self.topk, idx=vg.ptr(self.idx if idx is None else idx), p=vg.ptr(self.p if p is None else p),
                          Lphi=vg.ptr(self.d["lut"]), Y=vg.ptr(self.y), ldy=self.D, residual=vg.ptr(self.d["res"]) if residual else None,
                          ws=vg.ptr(self.ws), ws_bytes=self.ws.numel() * 4)

    def run(self, stream=None):
        vm.k_moe_route(self.rows.A, self.M, self.route_args(), stream=stream)
        vm.k_moe(self.rows.A, self.M, self.moe_args(), stream=stream)

    def want_route(self):
        return lm.route(self.rows.q, self.rows.e, self.rw[:, :self.D], self.cst, self.topk, self.renorm, self.lexp)

    def check(self, what=""):
        idx, p, z = self.want_route()
        assert_equal(to_np(self.logits), z, what + " logits")
        assert_equal(to_np(self.idx), idx, what + " idx")
        assert_equal(to_np(self.p), p, what + " p")
        assert_equal(to_np(self.y), lm.moe(self.rows.q, self.rows.e, idx, p, self.up, self.down, self.lut, self.res), what + " y")
        check_guard(self.ybuf, self.M * self.D, what)


@pytest.mark.parametrize("M,E,topk,D,F,group", [
    (1, 1, 1, 16, 4, 32), (1, 2, 2, 64, 20, 64), (1, 8, 2, 128, 256, 128), (2, 4, 1, 96, 100, 32), (3, 64, 6, 64, 36, 64), (5, 5, 5, 48, 68, 128),
    (16, 128, 8, 64, 32, 32), (17, 3, 2, 112, 132, 64), (40, 2, 2, 64, 64, 64), (33, 200, 3, 32, 24, 128), (7, 512, 16, 32, 12, 32)])
@pytest.mark.parametrize("renorm", [True, False])
def test_moe_layer(gpu, M, E, topk, D, F, group, renorm):
    rng = np.random.default_rng(M * 1000 + E)
    L = Layer(rng, M, E, topk, D, F, group, renorm=renorm, kind="q16" if (M + E) % 2 else "q8")
    L.run()
    torch.cuda.synchronize()
    L.check(f"{M} tokens {E} experts")


@pytest.mark.parametrize("kind", ["q8", "q16"])
@pytest.mark.parametrize("M,E,topk,K", [(1, 1, 1, 16), (2, 16, 16, 48), (1, 65, 3, 4048), (3, 128, 16, 32), (2, 129, 16, 32), (1, 130, 1, 2032), (5, 256, 8, 1040),
                                        (9, 257, 7, 1024), (1, 384, 16, 5008), (2, 512, 16, 64), (4, 512, 10, 16384), (6, 511, 2, 528)])
def test_route(gpu, M, E, topk, K, kind):
    """With the logits and without, ordinary ones, and ones that saturate at either end or are few different values: the lowest
    indices first."""
    rng = np.random.default_rng(E * 17 + M)
    rows = Rows(rng, kind, M, K, pad=16)
    w = rng.integers(-127, 128, (E, K + 32)).astype(np.int8)
    lexp = lm.exp_table()
    for what in ("plain", "saturated", "steps"):
        cst = np.zeros((E, 4), np.int32)
        cst[:, 0], cst[:, 1] = rng.integers(1 << 14, 1 << 15, E), 22 + (8 if kind == "q16" else 0)
        cst[:, 2] = rng.integers(-9000, 9000, E)
        if what == "saturated":
            cst[:, 2] = rng.choice(np.array([-(2**31), 2**31 - 1], np.int64), E, p=[0.9, 0.1] if M % 2 else [1.0, 0.0])
            cst[:, 0] = 0
        elif what == "steps":
            cst[:, 0], cst[:, 2] = 0, rng.integers(-2, 3, E) * 30000
        cst[:, 3] = w[:, :K].sum(1, dtype=np.int64)
        dw, dc, dl = dev(w), dev(cst), dev(lexp)
        for renorm in (0, 1):
            idx, p, z = lm.route(rows.q, rows.e, w[:, :K], cst, topk, bool(renorm), lexp)
            for logits in (False, True):
                di, dp = (torch.full((M, topk), -7, dtype=torch.int32, device="cuda") for _ in range(2))
                buf, dz = out32((M, E))
                R = vm.MoeRoute(W=vg.ptr(dw), ldw=K + 32, cst=vg.ptr(dc), experts=E, topk=topk, renorm=renorm, Lexp=vg.ptr(dl), idx=vg.ptr(di), p=vg.ptr(dp),
                                logits=vg.ptr(dz) if logits else None)
                vm.k_moe_route(rows.A, M, R)
                assert_equal(to_np(di), idx, what + " idx")
                assert_equal(to_np(dp), p, what + " p")
                if logits:
                    assert_equal(to_np(dz), z, what + " logits")
                check_guard(buf, M * E, what)


@pytest.mark.parametrize("M,E,topk,D,F,kind", [
    (1, 20, 16, 32, 64, "q8"), (1, 20, 16, 32, 5200, "q16"), (1, 6, 3, 5008, 36, "q8"), (1, 40, 6, 96, 1500, "q8"), (40, 2, 2, 32, 3000, "q8"),
    (20, 2, 1, 2512, 20, "q16"), (3, 4, 2, 8208, 24, "q8"), (33, 2, 1, 6000, 16, "q8"), (300, 3, 1, 16, 8, "q8")])
def test_moe_shapes(gpu, M, E, topk, D, F, kind):
    """One token with many choices, rows that fit in LDS or do not; rows in several chunks; more columns than a pass of the down
    product; row tiles of sixteen and what is left of them."""
    L = Layer(np.random.default_rng(D + F), M, E, topk, D, F, 64, kind=kind)
    L.run()
    torch.cuda.synchronize()
    L.check()


def test_moe_one_token_given_choices(gpu):
    rng = np.random.default_rng(15)
    L = Layer(rng, 1, 6, 5, 48, 40, 32)
    for idx in ([-1, -1, -1, -1, -1], [3, 3, 0, 3, 5], [7, 2, -5, 2**31 - 1, 1]):
        di, dp = dev(np.array([idx], np.int32)), dev(np.array([[32767, -32768, 1, 0, 12345]], np.int32))
        for residual in (True, False):
            vm.k_moe(L.rows.A, 1, L.moe_args(residual=residual, idx=di, p=dp))
            want = lm.moe(L.rows.q, L.rows.e, [idx], to_np(dp), L.up, L.down, L.lut, L.res if residual else None)
            assert_equal(to_np(L.y), want, f"{idx}")
    check_guard(L.ybuf, 48, "one token")


@pytest.mark.parametrize("E,topk,F", [(1, 2, 40), (2, 16, 40), (1, 3, 8208), (3, 16, 5200)])
@pytest.mark.parametrize("M", [1, 2])
def test_moe_more_choices_than_experts(gpu, M, E, topk, F):
    """A caller's choices may name every expert several times."""
    rng = np.random.default_rng(E + topk)
    L = Layer(rng, M, E, 1, 48, F, 64)
    idx, p = rng.integers(0, E, (M, topk)).astype(np.int32), rng.integers(-32768, 32768, (M, topk)).astype(np.int32)
    L.topk, L.ws = topk, torch.full((vm.moe_workspace_bytes(M, topk, F) // 4,), GUARD, dtype=torch.int32, device="cuda")
    di, dp = dev(idx), dev(p)
    vm.k_moe(L.rows.A, M, L.moe_args(idx=di, p=dp))
    assert_equal(to_np(L.y), lm.moe(L.rows.q, L.rows.e, idx, p, L.up, L.down, L.lut, L.res))


@pytest.mark.parametrize("M,E,topk,D,F,group", [
    (2, 4, 2, 4112, 36, 32), (3, 7, 5, 64, 132, 64), (16, 9, 1, 80, 100, 128), (8, 3, 2, 8208, 20, 64), (5, 64, 3, 96, 2052, 128), (2, 20, 8, 64, 5200, 32)])
@pytest.mark.parametrize("inplace", [False, True])
def test_moe_few_pairs(gpu, M, E, topk, D, F, group, inplace):
    """Up to sixteen pairs: column tiles alone or several a block, waves left over, rows of Y further apart than D and Y on top of the
    residual; rows that do not fit in LDS."""
    rng = np.random.default_rng(M + D + F)
    L = Layer(rng, M, E, topk, D, F, group)
    idx, p = rng.integers(-1, E + 1, (M, topk)).astype(np.int32), rng.integers(-(2**31), 2**31, (M, topk)).astype(np.int32)
    di, dp, ld = dev(idx), dev(p >> 14), D + 24
    res = rng.integers(-(10**6), 10**6, (M, ld)).astype(np.int32)
    buf, y = out32((M, ld))
    y.copy_(dev(res))
    apart = dev(res)
    args = L.moe_args(idx=di, p=dp)
    args.Y, args.ldy, args.residual = vg.ptr(y), ld, vg.ptr(y if inplace else apart)
    vm.k_moe(L.rows.A, M, args)
    got = to_np(y)
    assert_equal(got[:, :D], lm.moe(L.rows.q, L.rows.e, idx, p >> 14, L.up, L.down, L.lut, res[:, :D]))
    assert_equal(got[:, D:], res[:, D:], "cells between the rows")
    check_guard(buf, M * ld, "few pairs")


@pytest.mark.parametrize("group,group2", [(32, 128), (128, 64), (64, 32)])
def test_moe_groups_differ(gpu, group, group2):
    L = Layer(np.random.default_rng(3), 6, 9, 3, 160, 200, group, group2)
    L.run()
    torch.cuda.synchronize()
    L.check()


def test_moe_equal_logits(gpu):
    """Equal logits: the lowest indices in order, equal shares."""
    L = Layer(np.random.default_rng(4), 3, 70, 4, 64, 32, equal=True)
    L.run()
    torch.cuda.synchronize()
    L.check()
    assert_equal(to_np(L.idx), np.broadcast_to(np.arange(4), (3, 4)))


def test_moe_given_choices(gpu):
    """Choices a caller gives: an expert twice in a token, indices outside the layer, tokens without any, negative shares."""
    rng = np.random.default_rng(5)
    L = Layer(rng, 20, 6, 4, 64, 48, 32)
    idx = rng.integers(-2, 8, (20, 4)).astype(np.int32)
    idx[3] = -1
    idx[4] = [2, 2, 2, 2]
    idx[5] = [2**31 - 1, -(2**31), 6, 5]
    p = rng.integers(-32768, 32768, (20, 4)).astype(np.int32)
    di, dp = dev(idx), dev(p)
    vm.k_moe(L.rows.A, 20, L.moe_args(idx=di, p=dp))
    assert_equal(to_np(L.y), lm.moe(L.rows.q, L.rows.e, idx, p, L.up, L.down, L.lut, L.res))
    vm.k_moe(L.rows.A, 20, L.moe_args(residual=False, idx=di, p=dp))
    assert_equal(to_np(L.y), lm.moe(L.rows.q, L.rows.e, idx, p, L.up, L.down, L.lut, None))
    none = dev(np.full((20, 4), -1, np.int32))
    vm.k_moe(L.rows.A, 20, L.moe_args(idx=none, p=dp))
    assert_equal(to_np(L.y), L.res)
    check_guard(L.ybuf, 20 * 64, "given choices")


def test_moe_more_tokens_than_a_pass(gpu):
    """Tokens beyond one pass over the experts (512 pairs), the last pass a short one."""
    L = Layer(np.random.default_rng(6), 150, 4, 4, 32, 16, 32)
    L.run()
    torch.cuda.synchronize()
    L.check()


# ---------------------------------------------------------------- together, streams, graphs

def test_decode_step_graph(gpu):
    """Norm, 4-bit projection, second norm, router and experts as one captured graph on a stream of its own: every replay, with
    eager work between, gives the eager bytes."""
    rng = np.random.default_rng(20)
    M, D = 3, 256
    L = Layer(rng, M, 12, 3, D, 96, 64)
    proj = lm.Weights(rng, D, D, 128, s=14 + 11 + 13 + 4)
    W = packed(proj)
    x0 = np.round(rng.normal(size=(M, D)) * 70000).astype(np.int32)
    r0 = np.round(rng.normal(size=(M, D)) * 70000).astype(np.int32)
    g = rng.integers(30000, 90000, D, dtype=np.int32)
    x, r, dg = dev(x0), dev(r0), dev(g)
    new = lambda *s, dt=torch.int32: torch.empty(s, dtype=dt, device="cuda")  # noqa: E731
    h, q, e, y, h2, q2, e2 = new(M, D), new(M, D, dt=torch.int8), new(M), new(M, D), new(M, D), new(M, D, dt=torch.int8), new(M)
    A1 = vg.ASrc(src=vg.SRC_I8, hi=vg.ptr(q), ld8=D, e=vg.ptr(e), K=D)
    A2 = vg.ASrc(src=vg.SRC_I8, hi=vg.ptr(q2), ld8=D, e=vg.ptr(e2), K=D)
    E1 = vg.AEpi(Y=vg.ptr(y), ldy=D)
    args = L.moe_args()
    args.residual = vg.ptr(h2)
    st = torch.cuda.Stream()

    def step(stream):
        vn.k_rmsnorm_q(x, r, M, D, dg, DEN, h, q, None, e, D, stream=stream)
        vw.k_gemm_w4(A1, M, W, E1, stream=stream)
        vn.k_rmsnorm_q(y, h, M, D, dg, DEN, h2, q2, None, e2, D, stream=stream)
        vm.k_moe_route(A2, M, L.route_args(), stream=stream)
        vm.k_moe(A2, M, args, stream=stream)

    hh, yy = lm.rmsnorm(x0, r0, g, DEN)
    qq, ee = lm.quant(yy, 7)
    yp = lm.product(qq, ee, proj.dense(), proj.msb)
    hh2, yy2 = lm.rmsnorm(yp.astype(np.int32), hh.astype(np.int32), g, DEN)
    qq2, ee2 = lm.quant(yy2, 7)
    idx, p, _ = lm.route(qq2, ee2, L.rw[:, :D], L.cst, 3, True, L.lexp)
    want = lm.moe(qq2, ee2, idx, p, L.up, L.down, L.lut, hh2)
    st.wait_stream(torch.cuda.current_stream())
    step(st)
    st.synchronize()
    assert_equal(to_np(L.y), want, "eager")
    graph = vg.Graph(st)
    graph.begin()
    step(st)
    graph.end()
    for i in range(4):
        L.y.fill_(-1)
        torch.cuda.synchronize()
        graph.replay()
        st.synchronize()
        assert_equal(to_np(L.y), want, f"replay {i}")
        assert_equal(to_np(L.idx), idx, f"replay {i} idx")
        vn.k_rmsnorm_q(x, None, M, D, dg, DEN, None, q, None, e, D)   # eager work between the replays
        torch.cuda.synchronize()
    graph.destroy()


def test_moe_two_streams(gpu):
    """Two layers at once on two streams, each with its own workspace."""
    a, b = (Layer(np.random.default_rng(30 + i), 4, 16, 4, 128, 96, 64) for i in range(2))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        a.run(stream=s1)
        b.run(stream=s2)
    torch.cuda.synchronize()
    a.check("first stream")
    b.check("second stream")


def test_gated_feed_forward(gpu):
    """Up with GEGLU and row maxima, then down on the int32 rows: the 4-bit form of the engine's feed-forward."""
    rng = np.random.default_rng(40)
    M, D, F = 5, 192, 260
    up_w, down_w = lm.Weights(rng, 2 * F, D, 64, s=30), lm.Weights(rng, D, F, 32)
    rows = Rows(rng, "q8", M, D)
    lut = lm.sigmoid_table()
    dlut, v, rm, y = dev(lut), torch.empty((M, F), dtype=torch.int32, device="cuda"), torch.zeros(M, dtype=torch.int32, device="cuda"), torch.empty((M, D), dtype=torch.int32, device="cuda")
    U, V = packed(up_w), packed(down_w)
    vw.k_gemm_w4(rows.A, M, U, vg.AEpi(epi=vg.EPI_GEGLU, Y=vg.ptr(v), ldy=F, Lphi=vg.ptr(dlut), rowmax=vg.ptr(rm)))
    vw.k_gemm_w4(vg.ASrc(src=vg.SRC_X32, x=vg.ptr(v), ldx=F, rowmax=vg.ptr(rm), K=F), M, V, vg.AEpi(Y=vg.ptr(y), ldy=D))
    wv = lm.geglu(lm.product(rows.q, rows.e, up_w.dense(), up_w.msb), lut)
    q2, e2 = lm.quant(wv, 15)
    assert_equal(to_np(v), wv)
    assert_equal(to_np(y), lm.product(q2, e2, down_w.dense(), down_w.msb))

"""The language-model operators on the GPU where their other tests do not go: every result is a whole number and has to be equal
to the formulas in 64-bit integers (tests/lm_math.py)."""
import numpy as np
import pytest
import torch

from tests import lm_math as lm
from tests.conftest import assert_equal, to_np
from tests.test_gpu_lm import KINDS, Layer, Rows, check_w4, dev, packed
from vela_amd import gemm as vg
from vela_amd import moe as vm
from vela_amd import w4 as vw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E", [16, 128, 129, 512])
@pytest.mark.parametrize("topk", [1, 2, 8, 15, 16])
def test_route_shares_of_many_tokens(gpu, E, topk):
    """Shares over the chosen and over all experts, whose sums go through different lanes, for more tokens than CUs."""
    rng = np.random.default_rng(E + topk)
    M, K = 300, 32
    rows, lexp = Rows(rng, "q8", M, K), lm.exp_table()
    w = rng.integers(-127, 128, (E, K)).astype(np.int8)
    cst = np.zeros((E, 4), np.int32)
    cst[:, 0], cst[:, 1], cst[:, 2] = rng.integers(1 << 14, 1 << 15, E), 24, rng.integers(-60000, 60000, E)
    cst[:, 3] = w.sum(1, dtype=np.int64)
    dw, dc, dl = dev(w), dev(cst), dev(lexp)
    for renorm in (0, 1):
        idx, p, _ = lm.route(rows.q, rows.e, w, cst, topk, bool(renorm), lexp)
        di, dp = (torch.full((M, topk), -7, dtype=torch.int32, device="cuda") for _ in range(2))
        vm.k_moe_route(rows.A, M, vm.MoeRoute(W=vg.ptr(dw), ldw=K, cst=vg.ptr(dc), experts=E, topk=topk, renorm=renorm, Lexp=vg.ptr(dl), idx=vg.ptr(di), p=vg.ptr(dp)))
        assert_equal(to_np(di), idx, f"renorm {renorm} idx")
        assert_equal(to_np(dp), p, f"renorm {renorm} p")


@pytest.mark.parametrize("strided", [False, True])
def test_pack_of_sources_freed_at_once_on_a_busy_stream(gpu, strided):
    """Sources that nobody holds after the call, whose memory the next tensors of their own stream ask for while the packing
    waits behind other work, or first the copies of rows that are laid out otherwise: as from sources that are kept."""
    rng = np.random.default_rng(50)
    w = lm.Weights(rng, 256, 2048, 64)
    dense = packed(w)
    a, b = torch.randn((4096, 4096), device="cuda"), torch.empty((4096, 4096), device="cuda")
    W, st = vw.W4Weights(256, 2048, 64), torch.cuda.Stream()
    parts = [dev(t) for t in (w.nib, w.sc, w.z, w.msb)]
    if strided:
        parts = [t.t().contiguous().t() for t in parts]
    shapes = [(t.shape, t.dtype) for t in parts]
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(20):
            torch.mm(a, a, out=b)
    W.pack(*parts, stream=st)
    del parts
    junk = [torch.full(s, 85, dtype=dt, device="cuda") for s, dt in shapes for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(W.q, dense.q) and torch.equal(W.cst, dense.cst)
    assert all(bool((t == 85).all()) for t in junk)


# ---------------------------------------------------------------- gated products

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [17, 20, 33, 64, 130])
def test_gated_rows(gpu, kind, M):
    """One and two row tiles a block, the last ones short."""
    check_w4(np.random.default_rng(M), kind, M, 72, 512, 32 << (M % 3), epi="geglu", ldpad=3)


@pytest.mark.parametrize("kind,M,N", [("q8", 4, 5002), ("q8", 1, 22016), ("q8", 16, 22016), ("q16", 7, 9998), ("x32", 3, 12288), ("x32", 12, 9002), ("q8", 40, 20002),
                                      ("q16", 33, 13000), ("x32", 64, 22016), ("q8", 64, 5002), ("q8", 17, 34000), ("q16", 2, 70002)])
def test_gated_columns(gpu, kind, M, N):
    """Several column tiles a block, with the gate's table behind their sums, for one and two row tiles."""
    check_w4(np.random.default_rng(M + N), kind, M, N, 192, 64, epi="geglu", ldpad=1)


@pytest.mark.parametrize("kind,M,K,N", [("q16", 48, 5000, 40), ("q8", 64, 9000, 24), ("x32", 16, 12000, 24), ("q16", 16, 9999, 26), ("q8", 33, 20000, 16), ("x32", 64, 4100, 40),
                                        ("q16", 64, 3000, 9000), ("q8", 16, 9000, 8194), ("x32", 40, 2600, 9998)])
def test_gated_chunks(gpu, kind, M, K, N):
    """Rows that pass the staging area in several chunks of K, with few and with many column tiles a block."""
    check_w4(np.random.default_rng(K + N), kind, M, N, K, 128, epi="geglu")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [3, 20, 33])
def test_rows_far_apart(gpu, kind, M):
    """Rows at the widest stride a call takes: 2^21 bytes, 2^23 values."""
    rng = np.random.default_rng(60 + M)
    K, N = 160, 48
    w, few = lm.Weights(rng, N, K, 32), Rows(rng, kind, M, K)
    W, ld = packed(w), 1 << (23 if kind == "x32" else 21)
    far = [torch.full((M, ld), 99, dtype=t.dtype, device="cuda") if t.dim() == 2 else t for t in few.keep]
    for f, t in zip(far, few.keep):
        if t.dim() == 2:
            f[:, :t.shape[1]] = t
    y = torch.empty((M, N), dtype=torch.int32, device="cuda")
    if kind == "x32":
        A = vg.ASrc(src=vg.SRC_X32, x=vg.ptr(far[0]), ldx=ld, rowmax=vg.ptr(far[1]), K=K)
    else:
        A = vg.ASrc(src=vg.SRC_I8, hi=vg.ptr(far[0]), lo=vg.ptr(far[1]) if kind == "q16" else None, ld8=ld, e=vg.ptr(far[-1]), K=K)
    vw.k_gemm_w4(A, M, W, vg.AEpi(Y=vg.ptr(y), ldy=N))
    assert_equal(to_np(y), lm.product(few.q, few.e, w.dense(), w.msb))


# ---------------------------------------------------------------- experts

@pytest.mark.parametrize("M,topk", [(17, 1), (6, 3), (7, 3), (23, 1), (24, 1), (12, 2), (4, 6), (3, 8), (25, 1), (5, 5), (13, 2)])
@pytest.mark.parametrize("D", [64, 4112, 8208])
def test_moe_pairs_about_the_few(gpu, M, topk, D):
    """Up to 24 pairs and just above, with one and with several column tiles a block; more experts than pairs and fewer."""
    rng = np.random.default_rng(M * topk + D)
    for E in (30, 3):
        L = Layer(rng, M, E, min(topk, E), D, 36, 64, kind="q16" if M % 2 else "q8")
        L.run()
        torch.cuda.synchronize()
        L.check(f"{E} experts")


@pytest.mark.parametrize("M,topk", [(129, 4), (33, 16), (513, 1), (135, 4), (100, 16)])
def test_moe_last_pass(gpu, M, topk):
    """A last pass of one token, of few pairs and of many."""
    L = Layer(np.random.default_rng(M), M, 20, topk, 32, 20, 32)
    L.run()
    torch.cuda.synchronize()
    L.check()


def test_moe_rows_far_apart(gpu):
    """The tokens' rows at the widest stride, more tokens than a pass."""
    rng = np.random.default_rng(61)
    L = Layer(rng, 150, 6, 4, 64, 32, 32)
    far = torch.full((150, 1 << 21), 99, dtype=torch.int8, device="cuda")
    far[:, :64] = L.rows.keep[0]
    L.rows.A = vg.ASrc(src=vg.SRC_I8, hi=vg.ptr(far), ld8=1 << 21, e=vg.ptr(L.rows.keep[-1]), K=64)
    L.run()
    torch.cuda.synchronize()
    L.check()


def new_rows(L, rng):
    """Other rows for a layer of 8-bit rows: their values and shifts, and both on the device."""
    q, e = lm.rows8(rng, L.M, L.D)
    return q.astype(np.int64), e.astype(np.int64), dev(q), dev(e)


def want_layer(L, q, e):
    idx, p, _ = lm.route(q, e, L.rw[:, :L.D], L.cst, L.topk, L.renorm, L.lexp)
    return idx, lm.moe(q, e, idx, p, L.up, L.down, L.lut, L.res)


def test_moe_two_streams_other_rows_each_time(gpu):
    """Two layers at once on two streams, each with its own workspace; every run has rows of its own and its outputs are kept."""
    rng = np.random.default_rng(62)
    layers = [Layer(rng, M, 16, 4, 128, 96, 64) for M in (4, 9)]
    rows = [[new_rows(L, rng) for _ in range(5)] for L in layers]
    got = [[torch.empty_like(L.y) for _ in range(5)] for L in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for i in range(5):
        for L, st, r, g in zip(layers, streams, rows, got):
            with torch.cuda.stream(st):
                L.rows.keep[0].copy_(r[i][2])
                L.rows.keep[-1].copy_(r[i][3])
                L.y.fill_(-1)
                L.run(stream=st)
                g[i].copy_(L.y)
    torch.cuda.synchronize()
    for L, r, g in zip(layers, rows, got):
        for i in range(5):
            assert_equal(to_np(g[i]), want_layer(L, *r[i][:2])[1], f"{L.M} tokens, run {i}")


@pytest.mark.parametrize("M,E,topk,D,F", [(1, 8, 2, 64, 40), (5, 300, 8, 1024, 20), (40, 12, 3, 64, 40), (140, 6, 4, 32, 16)])
def test_moe_graph_of_other_rows(gpu, M, E, topk, D, F):
    """One captured layer, replayed with rows of its own each time, eager work between: one kernel of down products and sums, logits
    from a kernel of their own, row tiles, several passes."""
    rng = np.random.default_rng(63 + M)
    L, st = Layer(rng, M, E, topk, D, F, 32), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = vg.Graph(st)
    graph.begin()
    L.run(stream=st)
    graph.end()
    for i in range(4):
        q, e, dq, de = new_rows(L, rng)
        L.rows.keep[0].copy_(dq)
        L.rows.keep[-1].copy_(de)
        L.y.fill_(-1)
        L.ws.fill_(-7 * i)
        torch.cuda.synchronize()
        graph.replay()
        st.synchronize()
        idx, y = want_layer(L, q, e)
        assert_equal(to_np(L.idx), idx, f"replay {i} idx")
        assert_equal(to_np(L.y), y, f"replay {i}")
        L.run()   # eager, on the current stream, of the same rows
        torch.cuda.synchronize()
        assert_equal(to_np(L.y), y, f"eager {i}")
    graph.destroy()


def test_pack_on_a_busy_raw_stream(gpu):
    """As above, on a raw handle: what the caller's stream does next, and what reuses the sources' memory, comes after the packing."""
    rng = np.random.default_rng(51)
    w = lm.Weights(rng, 256, 2048, 64)
    dense = packed(w)
    a, b = torch.randn((4096, 4096), device="cuda"), torch.empty((4096, 4096), device="cuda")
    W, st = vw.W4Weights(256, 2048, 64), torch.cuda.Stream()
    parts = [dev(t) for t in (w.nib, w.sc, w.z, w.msb)]
    shapes = [(t.shape, t.dtype) for t in parts]
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(20):
            torch.mm(a, a, out=b)
    W.pack(*parts, stream=st.cuda_stream)
    del parts
    junk = [torch.full(s, 85, dtype=dt, device="cuda") for s, dt in shapes for _ in range(3)]
    assert torch.equal(W.q, dense.q) and torch.equal(W.cst, dense.cst)   # no synchronization before
    assert all(bool((t == 85).all()) for t in junk)

"""The language-model operators on the GPU where their other tests do not go: every result is a whole number and has to be equal
to the formulas in 64-bit integers (tests/lm_math.py)."""
import numpy as np
import pytest
import torch

from tests import lm_math as lm
from tests.conftest import assert_equal, to_np
from tests.test_gpu_lm import Rows, dev, packed
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

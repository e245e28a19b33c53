"""The language-model operators on the GPU where their other tests do not go: every result is a whole number and has to be equal
to the formulas in 64-bit integers (tests/lm_math.py)."""
import numpy as np
import pytest
import torch

from tests import lm_math as lm
from tests.conftest import assert_equal, to_np
from tests.test_gpu_lm import Rows, dev
from vela_amd import gemm as vg
from vela_amd import moe as vm

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

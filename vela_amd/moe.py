"""A mixture-of-experts layer for few tokens over the C ABI of libvgemm.so (include/vgemm_lm.h; no counterpart in the
reference): the router (k_moe_route: int8 logits, the chosen experts and their Q15 shares by the attention's exp table)
and the chosen experts' GEGLU feed-forward on 4-bit weights with its combination (k_moe). A failed check raises
VgemmError.
"""
from __future__ import annotations

import ctypes

from ._lib import ASrc, Moe, MoeRoute, check, load
from .gemm import stream_ptr

__all__ = ["MoeRoute", "MoeArgs", "moe_workspace_bytes", "k_moe_route", "k_moe"]

MoeArgs = Moe


def moe_workspace_bytes(M: int, topk: int, F: int) -> int:
    """Workspace bytes of k_moe for M tokens with topk choices of experts F wide."""
    return int(load().vgemm_moe_workspace_bytes(M, topk, F))


def k_moe_route(A: ASrc, M: int, R: MoeRoute, stream=None) -> None:
    """vgemm_moe_route: R.idx and R.p [M, topk] (and R.logits [M, experts]) from the tokens' SRC_I8 rows; A.K is the depth."""
    check(load().vgemm_moe_route(stream_ptr(stream), ctypes.byref(A), M, ctypes.byref(R)))


def k_moe(A: ASrc, M: int, P: Moe, stream=None) -> None:
    """vgemm_moe: Y[t] = sum over j of p[t, j] * expert idx[t, j] of row t (+ residual)."""
    check(load().vgemm_moe(stream_ptr(stream), ctypes.byref(A), M, ctypes.byref(P)))

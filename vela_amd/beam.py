"""Beam search over a paged cache, over the C ABI of libvgemm.so (include/vgemm_kv.h; no counterpart in the reference): the best
continuations over a group's beams and the vocabulary (k_beam_select) and the beams' block tables by parent (k_beam_tables), whose partly
filled pages kv.k_kv_copy copies. A failed check raises VgemmError.
"""
from __future__ import annotations

import ctypes

from ._lib import BeamSelect, BeamTables, check, load
from .gemm import stream_ptr

__all__ = ["BeamSelect", "BeamTables", "beam_workspace_bytes", "k_beam_select", "k_beam_tables"]


def beam_workspace_bytes(groups: int, beams: int, V: int, n: int) -> int:
    """Workspace bytes of k_beam_select (0: not supported)."""
    return int(load().vgemm_beam_workspace_bytes(groups, beams, V, n))


def k_beam_select(B: BeamSelect, stream=None) -> None:
    """vgemm_beam_select: B.out_score, B.parent and B.token [groups, n] from the logits of groups * beams rows."""
    check(load().vgemm_beam_select(stream_ptr(stream), ctypes.byref(B)))


def k_beam_tables(T: BeamTables, stream=None) -> None:
    """vgemm_beam_tables: tables and lengths of the rows' parents, and the pages to copy."""
    check(load().vgemm_beam_tables(stream_ptr(stream), ctypes.byref(T)))

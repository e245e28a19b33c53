"""A paged key-value cache over the C ABI of libvgemm.so (include/vgemm_kv.h; no counterpart in the reference): block tables and slot
maps from request lengths (k_kv_plan), keys and values into the pages (k_kv_write) and back (k_kv_read), attention of one new
token a sequence (k_kv_attention), copies of pages (k_kv_copy). A failed check raises VgemmError (ValueError for a
cache that is not supported).
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import Kv, KvAttn, KvPlan, check, load
from .gemm import ptr, stream_ptr

__all__ = ["Kv", "KvAttn", "KvCache", "KvPlan", "kv_page_bytes", "kv_attention_workspace_bytes", "k_kv_plan", "k_kv_write", "k_kv_read", "k_kv_copy",
           "k_kv_attention"]


def kv_page_bytes(page: int, heads: int, D: int, bits: int) -> int:
    """Bytes of one page's keys and values over all heads (0: not supported)."""
    return int(load().vgemm_kv_page_bytes(page, heads, D, bits))


def kv_attention_workspace_bytes(rows: int, Hq: int, D: int, max_len: int) -> int:
    """Workspace bytes of k_kv_attention (0 up to 256 tokens)."""
    return int(load().vgemm_kv_attention_workspace_bytes(rows, Hq, D, max_len))


class KvCache:
    """Device memory of `pages` pages of `page` tokens for `heads` heads of D values in 8 or 16 bits; desc is the argument of the calls."""

    def __init__(self, pages: int, page: int, heads: int, D: int, bits: int, device="cuda"):
        nb = kv_page_bytes(page, heads, D, bits)
        if not nb or pages < 1 or pages * page >= 1 << 31:
            raise ValueError(f"KvCache: a page of 16, 32, 64, 128 or 256 tokens, 1 to 1024 heads, D % 16 == 0, 16 <= D <= 256, 8 or 16 bits, pages >= 1 and "
                             f"pages * page < 2^31 expected, got {page}, {heads}, {D}, {bits}, {pages}")
        self.pages, self.page, self.heads, self.D, self.bits = pages, page, heads, D, bits
        self.data = torch.empty(pages * nb, dtype=torch.int8, device=device)
        self.shift = torch.empty(pages * heads * 2 * page, dtype=torch.uint8, device=device)
        self.desc = Kv(pages=pages, page=page, heads=heads, D=D, bits=bits, data=ptr(self.data), shift=ptr(self.shift))


def _desc(cache):
    return ctypes.byref(cache.desc if isinstance(cache, KvCache) else cache)


def k_kv_plan(P: KvPlan, stream=None) -> None:
    """vgemm_kv_plan: the new pages into P.table, and start, slot, pos of the new tokens, new_len and used."""
    check(load().vgemm_kv_plan(stream_ptr(stream), ctypes.byref(P)))


def k_kv_write(cache: KvCache | Kv, K, V, ld: int, slot, M: int, stream=None) -> None:
    """vgemm_kv_write: int32 rows K and V [M, heads * D], ld apart, into slots slot[t] (others than the cache's are left out)."""
    check(load().vgemm_kv_write(stream_ptr(stream), _desc(cache), ptr(K), ptr(V), ld, ptr(slot), M))


def k_kv_read(cache: KvCache | Kv, slot, M: int, K, V, ld: int, stream=None) -> None:
    """vgemm_kv_read: the rows of slots slot[t] as int32 (K or V may be None)."""
    check(load().vgemm_kv_read(stream_ptr(stream), _desc(cache), ptr(slot), M, ptr(K), ptr(V), ld))


def k_kv_copy(cache: KvCache | Kv, src, dst, n: int, stream=None) -> None:
    """vgemm_kv_copy: page dst[i] becomes a copy of page src[i]."""
    check(load().vgemm_kv_copy(stream_ptr(stream), _desc(cache), ptr(src), ptr(dst), n))


def k_kv_attention(cache: KvCache | Kv, A: KvAttn, stream=None) -> None:
    """vgemm_kv_attention: A.out[r] = attention of row r of A.Q over the A.len[r] tokens of its block table, row maxima onto the caller's values."""
    check(load().vgemm_kv_attention(stream_ptr(stream), _desc(cache), ctypes.byref(A)))

"""Products of few rows with 4-bit weights over the C ABI of libvgemm.so (include/vgemm_lm.h; no counterpart in the
reference): w[n, k] = (u[n, k] - z[n, k // group]) * sc[n, k // group] with 4-bit codes u and zero points z and scales
sc in 0..4095, requantised per column as the W8A16 products are. A failed check raises VgemmError (ValueError for a
tensor of another shape, type or device).
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import W4, AEpi, ASrc, check, load
from .gemm import ptr, stream_ptr

__all__ = ["W4", "W4Weights", "w4_bytes", "k_gemm_w4"]


def w4_bytes(N: int, K: int, group: int) -> int:
    """Bytes of one packed N x K matrix (0: not supported)."""
    return int(load().vgemm_w4_bytes(N, K, group))


class W4Weights:
    """Device memory of `count` packed N x K matrices and their column constants; desc is the argument of the calls."""

    def __init__(self, N: int, K: int, group: int, count: int = 1, device="cuda"):
        nb = w4_bytes(N, K, group)
        if not nb or count < 1:
            raise ValueError(f"W4Weights: 1 <= N <= 2^24, 1 <= K <= 32768, group 32, 64 or 128 and count >= 1 expected, got {N}, {K}, {group}, {count}")
        self.N, self.K, self.group, self.count = N, K, group, count
        self.q = torch.empty(count * nb, dtype=torch.uint8, device=device)
        self.cst = torch.empty((count, (N + 15) // 16 * 16, 4), dtype=torch.int32, device=device)
        self.desc = W4(N=N, K=K, group=group, count=count, q=ptr(self.q), cst=ptr(self.cst))

    def pack(self, nib: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None, msb: torch.Tensor, first: int = 0, stream=None) -> None:
        """Lay out matrices first, first + 1, ...: nib uint8 [(n,) N, >= K/2] (column 2i in the low half of byte i), scale
        int16 or uint16 [(n,) N, groups], zero uint8 alike or None (8 throughout), msb int32 [(n,) N, 4] {m, s, b, unused}. Row
        strides may be larger than the rows. The sources need not be kept after the call, which runs on the
        weights' device whichever is current; stream, where given, is one of that device. The current stream waits for the work on a
        stream that is given as a raw handle."""
        N, groups = self.N, (self.K + self.group - 1) // self.group
        n = nib.shape[0] if nib.dim() == 3 else 1
        # from one row to the next, over all matrices
        pitch = lambda t: t.stride(-2) if N > 1 else (t.stride(0) if n > 1 else t.shape[-1])  # noqa: E731

        sources = [("nib", nib, (torch.uint8,), (self.K + 1) // 2), ("scale", scale, (torch.int16, torch.uint16), groups), ("zero", zero, (torch.uint8,), groups),
                   ("msb", msb, (torch.int32,), 4)]
        for name, t, dtypes, width in sources:
            if t is None and name == "zero":
                continue
            shape = (n, N) if nib.dim() == 3 else (N,)
            if t.dtype not in dtypes or t.dim() != nib.dim() or tuple(t.shape[:-1]) != shape or t.shape[-1] < width or t.device != self.q.device:
                raise ValueError(f"W4Weights.pack: {name} of shape {tuple(t.shape)}, {t.dtype} on {t.device}")

        def rows(t):
            return t.contiguous() if t.stride(-1) != 1 or pitch(t) < t.shape[-1] or (n > 1 and t.stride(0) != N * pitch(t)) else t

        dev = self.q.device
        if getattr(stream, "device", dev) != dev:
            raise ValueError(f"W4Weights.pack: a stream of {stream.device} for weights on {dev}")
        raw = isinstance(stream, (int, torch.cuda.ExternalStream))
        with torch.cuda.device(dev):
            callers = torch.cuda.current_stream()
            # copies of rows that are laid out otherwise are made, and freed, on the kernels' stream
            with torch.cuda.stream(torch.cuda.ExternalStream(stream) if isinstance(stream, int) else stream):
                own = torch.cuda.current_stream()
                if not raw:   # nothing that the call uses is handed out again, once freed, before its work is done
                    for t in (nib, scale, zero, msb, self.q, self.cst):
                        if t is not None:
                            t.record_stream(own)
                try:
                    nib, scale, zero = rows(nib), rows(scale), rows(zero) if zero is not None else None
                    if zero is not None and pitch(zero) != pitch(scale):
                        scale, zero = scale[..., :groups].contiguous(), zero[..., :groups].contiguous()
                    msb = msb[..., :4].contiguous()
                    check(load().vgemm_w4_pack(stream_ptr(stream), ctypes.byref(self.desc), first, n, ptr(nib), pitch(nib), ptr(scale), ptr(zero), pitch(scale),
                                               ptr(msb)))
                finally:
                    if raw:   # its owner may end it while the weights live, so the allocator may not hold on to it: the caller's stream waits
                        callers.wait_stream(own)


def k_gemm_w4(A: ASrc, M: int, W: W4Weights | W4, E: AEpi, stream=None) -> None:
    """vgemm_w4: M rows (SRC_I8 with or without the low plane, or SRC_X32) times the packed weights; EPI_PLAIN (with a
    residual) or EPI_GEGLU, row maxima onto the caller's values."""
    desc = W.desc if isinstance(W, W4Weights) else W
    check(load().vgemm_w4(stream_ptr(stream), ctypes.byref(A), M, ctypes.byref(desc), ctypes.byref(E)))

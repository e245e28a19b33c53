"""The language-model operators without a GPU, beyond their argument checks: what the sources and the Python objects promise."""
import contextlib
import ctypes
import re
import types
from pathlib import Path

import pytest
import torch

from vela_amd import _lib, moe, w4

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "vela_amd" / "csrc"


def test_every_device_helper_has_a_caller():
    """A helper that nobody calls is dead, and one written to order an exchange through LDS leaves that exchange unordered."""
    text = {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in CSRC.iterdir() if p.suffix in (".h", ".hip")}
    everything = "\n".join(text.values())
    for name in ("w4_kernel.h", "w4.hip", "moe.hip", "rmsnorm.hip", "norm_math.h"):
        for fn in re.findall(r"^(?:template[^\n]*\n)?__device__ __forceinline__ [\w:& ]+? \*?(\w+)\(", text[name], flags=re.M):
            assert len(re.findall(rf"\b{fn}\b", everything)) > 1, f"{name}: {fn} has no caller"


FAKE = 1 << 40   # a 16-byte aligned address that is never dereferenced: every case fails validation first


@pytest.mark.parametrize("epi,rc", [(0, -1), (2, 0)])
def test_w4_statistics(epi, rc):
    """GroupNorm records, which the W8A16 products' PLAIN epilogue adds to, are refused, not left as they were; GEGLU does not read
    them, as in those products (no rows: nothing else is asked for)."""
    lib = _lib.load()
    W = _lib.W4(N=64, K=64, group=64, count=1, q=FAKE, cst=FAKE)
    A, E = _lib.ASrc(src=0, hi=FAKE, ld8=64), _lib.AEpi(epi=epi, Y=FAKE, ldy=64, Lphi=FAKE, gnstat=FAKE, gnT=64)
    assert lib.vgemm_w4(None, ctypes.byref(A), 0, ctypes.byref(W), ctypes.byref(E)) == rc
    assert ("statistics" in lib.vgemm_last_error().decode()) == (rc != 0)


class External:
    def __init__(self, raw, device=None):
        self.raw = raw


class PackCall:
    """W4Weights.pack on CPU tensors with the library, the CUDA contexts and record_stream replaced by recorders."""

    def __init__(self, monkeypatch, device="cuda:1"):
        self.where, self.calls, self.recorded, self.device = [], [], [], torch.device(device)
        me = self

        class Lib:
            def vgemm_w4_pack(self, stream, *args):
                me.calls.append((stream, tuple(me.where)))
                return 0

        @contextlib.contextmanager
        def enter(kind, what):
            me.where.append((kind, what))
            yield
            me.where.pop()

        monkeypatch.setattr(w4, "load", Lib)
        monkeypatch.setattr(w4, "ptr", lambda t: None if t is None else t.data_ptr())
        monkeypatch.setattr(w4, "stream_ptr", lambda s=None: ("raw", s))
        monkeypatch.setattr(torch.cuda, "device", lambda d: enter("device", d))
        monkeypatch.setattr(torch.cuda, "stream", lambda s: enter("stream", s))
        self.waits = []

        class Current(str):   # the current stream: the caller's, or the one made current for the call
            def wait_stream(self, other):
                me.waits.append((str(self), str(other), len(me.calls)))

        monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: Current("current" if any(k == "stream" for k, _ in me.where) else "caller's"))
        monkeypatch.setattr(torch.cuda, "ExternalStream", External)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: me.recorded.append((t.data_ptr(), s)))
        self.W = w4.W4Weights.__new__(w4.W4Weights)
        self.W.N, self.W.K, self.W.group, self.W.count, self.W.desc = 8, 64, 32, 1, _lib.W4()
        self.W.q, self.W.cst = torch.zeros(2048, dtype=torch.uint8), torch.zeros((1, 16, 4), dtype=torch.int32)
        self.parts = [torch.zeros((8, 32), dtype=torch.uint8), torch.zeros((8, 2), dtype=torch.int16), torch.zeros((8, 2), dtype=torch.uint8),
                      torch.zeros((8, 4), dtype=torch.int32)]


@pytest.mark.parametrize("stream", [None, "side"])
def test_pack_keeps_memory_until_its_stream_is_done(monkeypatch, stream):
    """The sources may be freed right after the call, and so may the weights: the allocator has to know the stream that uses them."""
    c = PackCall(monkeypatch)
    c.W.pack(*c.parts, stream=stream)
    assert len(c.calls) == 1
    used = {t.data_ptr() for t in (*c.parts, c.W.q, c.W.cst)}
    assert {p for p, _ in c.recorded} == used and {s for _, s in c.recorded} == {"current"}   # the one made current for the call


@pytest.mark.parametrize("stream", [1234, External(1234)])
def test_pack_on_a_raw_stream(monkeypatch, stream):
    """The owner of a raw stream may end it before the weights go, so the allocator must not hold on to it: the caller's stream waits
    for the packing instead, once it is launched."""
    c = PackCall(monkeypatch)
    c.W.pack(*c.parts, stream=stream)
    assert len(c.calls) == 1 and not c.recorded
    assert c.waits == [("caller's", "current", 1)]


def test_pack_keeps_sources_that_it_copies(monkeypatch):
    """Rows that are laid out otherwise are copied on the call's stream, which reads the given ones."""
    c = PackCall(monkeypatch)
    strided = [torch.zeros((t.shape[1], t.shape[0]), dtype=t.dtype).t() for t in c.parts]
    c.W.pack(*strided, stream="side")
    assert {t.data_ptr() for t in strided} <= {p for p, _ in c.recorded}


@pytest.mark.parametrize("stream", [None, "side", 1234])
def test_pack_runs_on_the_device_of_the_weights(monkeypatch, stream):
    """Whatever device is current; a raw handle is one of that device."""
    c = PackCall(monkeypatch)
    c.W.pack(*c.parts, stream=stream)
    (given, where), = c.calls
    kinds = [k for k, _ in where]
    assert where[0] == ("device", c.W.q.device) and kinds == ["device", "stream"]
    assert where[1][1] == stream if stream != 1234 else where[1][1].raw == 1234


def test_pack_refuses_a_stream_of_another_device(monkeypatch):
    c = PackCall(monkeypatch)
    with pytest.raises(ValueError, match="stream of cuda:3"):
        c.W.pack(*c.parts, stream=types.SimpleNamespace(device=torch.device("cuda:3"), cuda_stream=5))
    assert not c.calls


def test_most_columns():
    """2^24 columns a matrix, with the limit in the message."""
    lib = _lib.load()
    assert w4.w4_bytes(1 << 24, 64, 64) > 0 and w4.w4_bytes((1 << 24) + 1, 64, 64) == 0
    W = _lib.W4(N=(1 << 24) + 1, K=64, group=64, count=1, q=FAKE, cst=FAKE)
    A, E = _lib.ASrc(src=0, hi=FAKE, ld8=64), _lib.AEpi(Y=FAKE, ldy=1 << 25)
    assert lib.vgemm_w4(None, ctypes.byref(A), 1, ctypes.byref(W), ctypes.byref(E)) == -1
    assert "N <= 2^24" in lib.vgemm_last_error().decode()


@pytest.mark.parametrize("F", [-4, 0, 63, 32772, 1 << 30, (1 << 31) - 4])
def test_no_workspace_for_sizes_a_layer_does_not_take(F):
    assert moe.moe_workspace_bytes(3, 2, F) == 0


def test_workspace_of_the_widest_experts():
    pairs, F = 512, 32768   # the rows of v and of a pass of the down product, the maxima of v's column tiles
    assert moe.moe_workspace_bytes(1 << 30, 16, F) == pairs * (F + 8192 + 2 * F // 16) * 4

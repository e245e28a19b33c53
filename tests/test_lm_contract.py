"""The language-model operators without a GPU, beyond their argument checks: what the sources and the Python objects promise."""
import ctypes
import re
from pathlib import Path

import pytest

from vela_amd import _lib

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

"""The language-model operators without a GPU, beyond their argument checks: what the sources and the Python objects promise."""
import re
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "vela_amd" / "csrc"


def test_every_device_helper_has_a_caller():
    """A helper that nobody calls is dead, and one written to order an exchange through LDS leaves that exchange unordered."""
    text = {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in CSRC.iterdir() if p.suffix in (".h", ".hip")}
    everything = "\n".join(text.values())
    for name in ("w4_kernel.h", "w4.hip", "moe.hip", "rmsnorm.hip", "norm_math.h"):
        for fn in re.findall(r"^(?:template[^\n]*\n)?__device__ __forceinline__ [\w:& ]+? \*?(\w+)\(", text[name], flags=re.M):
            assert len(re.findall(rf"\b{fn}\b", everything)) > 1, f"{name}: {fn} has no caller"

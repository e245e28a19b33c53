"""The paged key-value cache's operators without a GPU: include/vgemm_kv.h against the ctypes mirror and the exported symbols, the
argument checks before any device work, sizes, and the tests' own 64-bit formulas against closed forms."""
import ctypes
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest

from tests import kv_math as km
from tests import lm_math as lm
from vela_amd import _lib, beam, kv

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "vgemm_kv.h"
FAKE = 1 << 40   # a 16-byte aligned address that is never dereferenced: every case fails validation first


def last():
    return _lib.load().vgemm_last_error().decode()


def test_every_declared_symbol_is_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    decl = {m.group(1): m.group(2).count(",") + 1 for m in re.finditer(r"^[A-Za-z_][\w \*]*?\b(vgemm_\w+)\s*\(([^)]*)\)\s*;", text, flags=re.M)}
    sigs = {name: len(args) for name, _, args in _lib.KV_SIGNATURES}
    assert decl == sigs
    for name in decl:
        assert hasattr(_lib.load(), name)


def test_struct_layout_matches_c(tmp_path):
    structs = (("VgemmKv", _lib.Kv), ("VgemmKvPlan", _lib.KvPlan), ("VgemmKvAttn", _lib.KvAttn), ("VgemmBeam", _lib.BeamSelect),
               ("VgemmBeamTables", _lib.BeamTables))
    lines = [f'printf("{T} %zu", sizeof({T}));' + "".join(f'printf(" %zu", offsetof({T}, {f}));' for f, _ in cls._fields_) + 'printf("\\n");' for T, cls in structs]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include "vgemm_kv.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [line.split() for line in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines()]
    for (T, cls), row in zip(structs, got):
        assert row == [T, str(ctypes.sizeof(cls))] + [str(getattr(cls, f).offset) for f, _ in cls._fields_]


# ---------------------------------------------------------------- refusals

def cache(**change):
    return _lib.Kv(**{**dict(pages=8, page=16, heads=2, D=64, bits=8, data=FAKE, shift=FAKE), **change})


BAD_CACHES = [(dict(data=None), "data and shift"), (dict(shift=None), "data and shift"), (dict(data=FAKE + 8), "16-byte"), (dict(shift=FAKE + 1), "16-byte"),
              (dict(page=8), "page of 16"), (dict(page=48), "page of 16"), (dict(page=512), "page of 16"), (dict(page=0), "page of 16"), (dict(heads=0), "heads"),
              (dict(heads=1025), "heads"), (dict(D=8), "D % 16"), (dict(D=0), "D % 16"), (dict(D=272), "D <= 256"), (dict(D=72), "D % 16"), (dict(bits=4), "8 or 16"),
              (dict(bits=32), "8 or 16"), (dict(pages=0), "pages >= 1"), (dict(pages=-3), "pages >= 1"), (dict(pages=1 << 27), "2^31")]


@pytest.mark.parametrize("change,msg", BAD_CACHES)
def test_cache_refusals(change, msg):
    lib, C = _lib.load(), cache(**change)
    A = attn()
    assert lib.vgemm_kv_write(None, ctypes.byref(C), FAKE, FAKE, 128, FAKE, 3) == -1 and msg in last()
    assert lib.vgemm_kv_read(None, ctypes.byref(C), FAKE, 3, FAKE, FAKE, 128) == -1 and msg in last()
    assert lib.vgemm_kv_copy(None, ctypes.byref(C), FAKE, FAKE, 3) == -1 and msg in last()
    assert lib.vgemm_kv_attention(None, ctypes.byref(C), ctypes.byref(A)) == -1 and msg in last()
    assert lib.vgemm_kv_write(None, None, FAKE, FAKE, 128, FAKE, 3) == -1


def plan(**change):
    return _lib.KvPlan(**{**dict(R=3, tokens=5, pages=8, page=16, width=4, ldt=4, len=FAKE, add=FAKE, table=FAKE, free=FAKE, nfree=FAKE, slot=FAKE), **change})


@pytest.mark.parametrize("change,rc,msg", [
    (dict(R=-1), -1, "bad arguments"), (dict(tokens=-1), -1, "bad arguments"), (dict(page=17), -1, "page of 16"), (dict(pages=0), -1, "pages >= 1"),
    (dict(pages=1 << 27), -1, "2^31"), (dict(R=4097), -3, "at most 4096"), (dict(width=-1), -1, "width"), (dict(ldt=3), -1, "width <= ldt"), (dict(len=None), -1, "len, add"),
    (dict(add=None), -1, "len, add"), (dict(table=None), -1, "len, add"), (dict(free=None), -1, "len, add"), (dict(nfree=None), -1, "len, add"), (dict(slot=None), -1, "slot")])
def test_plan_refusals(change, rc, msg):
    assert _lib.load().vgemm_kv_plan(None, ctypes.byref(plan(**change))) == rc
    assert msg in last()


@pytest.mark.parametrize("change,rc,msg", [
    (dict(K=None), -1, "K, V"), (dict(V=None), -1, "K, V"), (dict(slot=None), -1, "slot"), (dict(M=-1), -1, "bad arguments"), (dict(K=FAKE + 4), -1, "16-byte"),
    (dict(V=FAKE + 8), -1, "16-byte"), (dict(ld=124), -1, "ld >= heads"), (dict(ld=130), -1, "ld % 4"), (dict(M=(1 << 24) + 1), -3, "at most 16777216")])
def test_row_refusals(change, rc, msg):
    a = {**dict(K=FAKE, V=FAKE, ld=128, slot=FAKE, M=3), **change}
    lib, C = _lib.load(), cache()
    assert lib.vgemm_kv_write(None, ctypes.byref(C), a["K"], a["V"], a["ld"], a["slot"], a["M"]) == rc
    assert msg in last()
    if a["K"] and a["V"]:
        assert lib.vgemm_kv_read(None, ctypes.byref(C), a["slot"], a["M"], a["K"], a["V"], a["ld"]) == rc
        assert msg in last()


@pytest.mark.parametrize("src,dst,n,rc,msg", [(None, FAKE, 3, -1, "src and dst"), (FAKE, None, 3, -1, "src and dst"), (FAKE, FAKE, -1, -1, "bad arguments"),
                                              (FAKE, FAKE, (1 << 23) + 1, -3, "at most 8388608")])
def test_copy_refusals(src, dst, n, rc, msg):
    assert _lib.load().vgemm_kv_copy(None, ctypes.byref(cache()), src, dst, n) == rc
    assert msg in last()


def attn(**change):
    return _lib.KvAttn(**{**dict(Q=FAKE, ldq=256, rows=3, Hq=4, table=FAKE, ldt=40, width=40, len=FAKE, max_len=600, window=0, m=16384, s=34, Lexp=FAKE, out=FAKE,
                                 ldo=256, ws=FAKE, ws_bytes=1 << 30), **change})


@pytest.mark.parametrize("change,rc,msg", [
    (dict(rows=-1), -1, "bad arguments"), (dict(Hq=0), -1, "multiple of the cache's heads"), (dict(Hq=3), -1, "multiple of the cache's heads"), (dict(Hq=4098, ldq=1 << 20, ldo=1 << 20), -1, "at most 4096"),
    (dict(m=0), -1, "m <= 32768"), (dict(m=32769), -1, "m <= 32768"), (dict(s=-65), -1, "-64 <= s"), (dict(s=129), -1, "s <= 128"), (dict(max_len=-1), -1, "max_len >= 0"),
    (dict(window=-1), -1, "window >= 0"), (dict(width=-1), -1, "width"), (dict(ldt=39), -1, "width <= ldt"), (dict(rows=65536), -3, "at most 65535"),
    (dict(max_len=(1 << 23) + 1), -3, "at most 8388608"), (dict(Q=None), -1, "required"), (dict(len=None), -1, "required"), (dict(table=None), -1, "required"), (dict(Lexp=None), -1, "required"),
    (dict(out=None), -1, "required"), (dict(Q=FAKE + 4), -1, "16-byte"), (dict(out=FAKE + 8), -1, "16-byte"), (dict(ldq=252), -1, "ldq"), (dict(ldo=252), -1, "ldo"), (dict(ldq=258), -1, "multiples of 4"),
    (dict(ldo=258), -1, "multiples of 4"), (dict(ws=None), -1, "workspace"), (dict(ws=FAKE + 4), -1, "workspace"), (dict(ws_bytes=3 * 4 * 3 * (8 + 256) - 1), -1, "workspace")])
def test_attention_refusals(change, rc, msg):
    assert _lib.load().vgemm_kv_attention(None, ctypes.byref(cache()), ctypes.byref(attn(**change))) == rc
    assert msg in last()


def select(**change):
    return _lib.BeamSelect(**{**dict(groups=2, beams=3, V=5000, n=6, logits=FAKE, ldz=5000, score=FAKE, Lexp=FAKE, Lln=FAKE, out_score=FAKE, parent=FAKE, token=FAKE,
                                     ws=FAKE, ws_bytes=1 << 30), **change})


@pytest.mark.parametrize("change,msg", [
    (dict(groups=-1), "bad arguments"), (dict(beams=0), "beams <= 32"), (dict(beams=33), "beams <= 32"), (dict(V=0), "1 <= V"), (dict(V=(1 << 18) + 1, ldz=1 << 19), "1 <= V"), (dict(n=0), "1 <= n"),
    (dict(n=65), "n <= 64"), (dict(groups=21846), "65535"), (dict(logits=None), "required"), (dict(ldz=4999), "ldz >= V"), (dict(score=None), "required"), (dict(Lexp=None), "required"),
    (dict(Lln=None), "required"), (dict(out_score=None), "required"), (dict(parent=None), "required"), (dict(token=None), "required"), (dict(ws=None), "workspace"), (dict(ws=FAKE + 8), "workspace"),
    (dict(ws_bytes=6 * 2 * (16 + 48) - 1), "workspace")])
def test_select_refusals(change, msg):
    assert _lib.load().vgemm_beam_select(None, ctypes.byref(select(**change))) == -1
    assert msg in last()


def tables(**change):
    return _lib.BeamTables(**{**dict(rows=3, page=16, width=4, ldt=4, parent=FAKE, len=FAKE, table=FAKE, fresh=FAKE, out_len=FAKE, out_table=FAKE, src=FAKE, dst=FAKE), **change})


@pytest.mark.parametrize("change,rc,msg", [
    (dict(rows=-1), -1, "bad arguments"), (dict(page=12), -1, "page of 16"), (dict(width=-1), -1, "width"), (dict(ldt=3), -1, "width <= ldt"), (dict(rows=65536), -3, "at most 65535"),
    *((dict([(f, None)]), -1, "required") for f in ("parent", "len", "table", "fresh", "out_len", "out_table", "src", "dst"))])
def test_tables_refusals(change, rc, msg):
    assert _lib.load().vgemm_beam_tables(None, ctypes.byref(tables(**change))) == rc
    assert msg in last()


def test_empty_calls_do_nothing():
    lib, C = _lib.load(), cache()
    assert lib.vgemm_kv_write(None, ctypes.byref(C), None, None, 0, None, 0) == 0
    assert lib.vgemm_kv_read(None, ctypes.byref(C), None, 0, None, None, 0) == 0
    assert lib.vgemm_kv_read(None, ctypes.byref(C), FAKE, 3, None, None, 0) == 0
    assert lib.vgemm_kv_copy(None, ctypes.byref(C), None, None, 0) == 0
    assert lib.vgemm_kv_attention(None, ctypes.byref(C), ctypes.byref(attn(rows=0, Q=None, out=None, ws=None))) == 0
    assert lib.vgemm_beam_select(None, ctypes.byref(select(groups=0, logits=None, ws=None))) == 0
    assert lib.vgemm_beam_tables(None, ctypes.byref(tables(rows=0, parent=None))) == 0


def test_null_arguments():
    lib, C = _lib.load(), cache()
    assert lib.vgemm_kv_plan(None, None) == lib.vgemm_kv_attention(None, ctypes.byref(C), None) == lib.vgemm_beam_select(None, None) == lib.vgemm_beam_tables(None, None) == -1


def test_sizes():
    assert kv.kv_page_bytes(16, 8, 128, 8) == 8 * 2 * 16 * 128 and kv.kv_page_bytes(256, 3, 80, 16) == 3 * 2 * 256 * 80 * 2
    for bad in ((24, 8, 128, 8), (16, 0, 128, 8), (16, 8, 120, 8), (16, 8, 512, 8), (16, 8, 128, 4)):
        assert kv.kv_page_bytes(*bad) == 0
        with pytest.raises(ValueError, match="KvCache"):
            kv.KvCache(4, *bad, device="meta")
    for pages in (0, -1, 1 << 27):
        with pytest.raises(ValueError, match="KvCache"):
            kv.KvCache(pages, 16, 8, 128, 8, device="meta")
    # no workspace up to one span; 64 bits where 32 would not do
    assert kv.kv_attention_workspace_bytes(7, 8, 64, 256) == 0 and kv.kv_attention_workspace_bytes(7, 8, 64, 257) == 7 * 8 * 2 * (8 + 256)
    assert kv.kv_attention_workspace_bytes(65535, 128, 128, 1 << 20) == 65535 * 128 * 4096 * (8 + 512)
    for bad in ((0, 8, 64, 999), (65536, 8, 64, 999), (7, 0, 64, 999), (7, 4097, 64, 999), (7, 8, 60, 999), (7, 8, 512, 999), (7, 8, 64, (1 << 23) + 1)):
        assert kv.kv_attention_workspace_bytes(*bad) == 0
    assert beam.beam_workspace_bytes(3, 4, 4097, 8) == 12 * 2 * (16 + 64)
    assert beam.beam_workspace_bytes(65535, 1, 1 << 18, 64) == 65535 * 64 * (16 + 512)
    for bad in ((0, 4, 99, 8), (3, 33, 99, 8), (3, 4, 0, 8), (3, 4, (1 << 18) + 1, 8), (3, 4, 99, 65), (1 << 30, 4, 99, 8)):
        assert beam.beam_workspace_bytes(*bad) == 0


# ---------------------------------------------------------------- the formulas against closed forms

def test_formula_of_attention():
    """Against a softmax in floating point; one key gives its own row; equal keys give the mean; spans far below the best do not count."""
    rng = np.random.default_rng(1)
    D, n, heads, L = 64, 700, 2, lm.exp_table()
    m, s = km.scale_of(D)
    q = np.round(rng.standard_normal((4, D)) * 65536 * 2).astype(np.int64)
    k, v = (np.round(rng.standard_normal((n, heads, D)) * 65536).astype(np.int64) for _ in range(2))
    (kq, ek), (vq, ev) = km.quant(k, 16), km.quant(v, 16)
    out = km.attend(q, kq, ek, vq, ev, np.ones(n, bool), heads, m, s, L)
    for h in range(4):
        z = (k[:, h // 2] @ q[h]) / 65536.0**2 / 8
        w = np.exp(z - z.max())
        want = (w[:, None] * v[:, h // 2]).sum(0) / w.sum()
        # a score is off by a rounding of Q16, queries of 15 bits and keys of 16: below 2e-3 here, so a weight by 0.2 % and the table's 1/64 steps by
        # 3e-5; a weight below 2^-16 of the best is dropped. Means of 65536-sized values: half a percent of 65536 is ample.
        assert np.abs(out[h] - want).max() < 330
    one = km.attend(q, kq[:1], ek[:1], vq[:1], ev[:1], np.ones(1, bool), heads, m, s, L)
    assert np.array_equal(one, np.repeat(vq[0] << ev[0][:, None], 2, 0))
    same = km.attend(q, np.repeat(kq[:1], 300, 0), np.repeat(ek[:1], 300, 0), vq[:300], ev[:300], np.ones(300, bool), heads, m, s, L)
    mean = (vq[:300].astype(np.int64) << ev[:300][..., None]).mean(0)
    assert np.abs(same - np.repeat(mean, 2, 0)).max() <= 1.5
    assert not km.attend(q, kq, ek, vq, ev, np.zeros(n, bool), heads, m, s, L).any()


def test_formula_of_log_sum():
    rng = np.random.default_rng(2)
    z = np.round(rng.standard_normal(9000) * 3 * 65536).astype(np.int64)
    z[5] = km.LOW
    mx, lz = km.logz(z, lm.exp_table(), km.ln_table())
    x = np.delete(z, 5) / 65536
    # the tables are linear between steps of 1/64 and 1/1024: relative 2^-15 in the sum, so 2^-15 in its logarithm, 2 of Q16
    assert mx == np.delete(z, 5).max() and abs(lz - 65536 * (np.log(np.exp(x - x.max()).sum()))) < 4
    assert km.logz(np.full(10, km.LOW), lm.exp_table(), km.ln_table()) is None


def test_formula_of_plan():
    table = np.array([[3, -1, -1], [7, 2, -1], [-1, -1, -1]])
    t, new, start, slot, pos, used = km.plan([16, 20, 0], [1, 13, 0], table, [5, 9, 1], 10, 16, 3, 16)
    assert t.tolist() == [[3, 5, -1], [7, 2, 9], [-1, -1, -1]] and new.tolist() == [17, 33, 0] and start.tolist() == [0, 1, 14, 14] and used == 2
    assert slot.tolist() == [80, *range(36, 48), 144, -1, -1] and pos.tolist() == [16, *range(20, 33), -1, -1]

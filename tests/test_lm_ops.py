"""The language-model operators without a GPU: include/vgemm_lm.h against the ctypes mirror and the exported symbols, the
argument checks before any device work, sizes, and the tests' own 64-bit formulas against closed forms."""
import ctypes
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from tests import lm_math as lm
from vela_amd import _lib, moe, w4

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "vgemm_lm.h"
FAKE = 1 << 40   # a 16-byte aligned address that is never dereferenced: every case fails validation first


def last():
    return _lib.load().vgemm_last_error().decode()


def test_every_declared_symbol_is_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    decl = {m.group(1): m.group(2).count(",") + 1 for m in re.finditer(r"^[A-Za-z_][\w \*]*?\b(vgemm_\w+)\s*\(([^)]*)\)\s*;", text, flags=re.M)}
    sigs = {name: len(args) for name, _, args in _lib.LM_SIGNATURES}
    assert decl == sigs
    for name in decl:
        assert hasattr(_lib.load(), name)


def test_struct_layout_matches_c(tmp_path):
    structs = (("VgemmW4", _lib.W4), ("VgemmMoeRoute", _lib.MoeRoute), ("VgemmMoe", _lib.Moe))
    lines = [f'printf("{T} %zu", sizeof({T}));' + "".join(f'printf(" %zu", offsetof({T}, {f}));' for f, _ in cls._fields_) + 'printf("\\n");' for T, cls in structs]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include "vgemm_lm.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [line.split() for line in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines()]
    for (T, cls), row in zip(structs, got):
        assert row == [T, str(ctypes.sizeof(cls))] + [str(getattr(cls, f).offset) for f, _ in cls._fields_]


@pytest.mark.parametrize("change,msg", [
    (dict(X=None), "bad arguments"), (dict(M=-1), "bad arguments"), (dict(g=None), "bad arguments"), (dict(hi=None), "bad arguments"),
    (dict(e=None), "bad arguments"), (dict(den=0), "bad arguments"), (dict(C=6), "multiple of 4"), (dict(C=0), "multiple of 4"),
    (dict(C=8196, Kp=8196), "at most 8192"), (dict(X=FAKE + 4), "16-byte"), (dict(R=FAKE + 8), "16-byte"), (dict(H=FAKE + 4), "16-byte"),
    (dict(g=FAKE + 4), "16-byte"), (dict(Kp=60), "Kp >= C"), (dict(Kp=66), "Kp % 4"), (dict(hi=FAKE + 2), "4-byte"), (dict(lo=FAKE + 1), "4-byte")])
def test_norm_refusals(change, msg):
    a = dict(X=FAKE, R=None, M=3, C=64, g=FAKE, den=100000, H=None, hi=FAKE, lo=None, e=FAKE, Kp=64)
    a.update(change)
    assert _lib.load().vgemm_rmsnorm_q(None, *a.values()) == -1
    assert msg in last()


def test_empty_calls_do_nothing():
    lib = _lib.load()
    assert lib.vgemm_rmsnorm_q(None, None, None, 0, 64, None, 1, None, None, None, None, 64) == 0
    W = _lib.W4(N=64, K=64, group=64, count=1, q=FAKE, cst=FAKE)
    A, E = _lib.ASrc(), _lib.AEpi()
    assert lib.vgemm_w4(None, ctypes.byref(A), 0, ctypes.byref(W), ctypes.byref(E)) == 0
    assert lib.vgemm_w4_pack(None, ctypes.byref(W), 1, 0, None, 0, None, None, 0, None) == 0
    R = _lib.MoeRoute(experts=4, topk=2)
    assert lib.vgemm_moe_route(None, ctypes.byref(A), 0, ctypes.byref(R)) == 0
    P = _lib.Moe(up=W, down=_lib.W4(N=64, K=32, group=64, count=1, q=FAKE, cst=FAKE), topk=1)
    assert lib.vgemm_moe(None, ctypes.byref(A), 0, ctypes.byref(P)) == 0


WEIGHTS = [(dict(N=0), "N >= 1"), (dict(K=0), "K <= 32768"), (dict(K=32769), "K <= 32768"), (dict(group=16), "group of 32"), (dict(group=256), "group of 32"),
           (dict(q=None), "q and cst"), (dict(q=FAKE + 8), "16-byte"), (dict(cst=None), "q and cst"), (dict(cst=FAKE + 4), "16-byte"), (dict(count=0), "count >= 1")]


@pytest.mark.parametrize("change,msg", WEIGHTS)
def test_weight_refusals(change, msg):
    lib = _lib.load()
    W = _lib.W4(**{**dict(N=64, K=64, group=64, count=1, q=FAKE, cst=FAKE), **change})
    A, E = _lib.ASrc(src=0, hi=FAKE, ld8=64), _lib.AEpi(Y=FAKE, ldy=64)
    assert lib.vgemm_w4(None, ctypes.byref(A), 2, ctypes.byref(W), ctypes.byref(E)) == -1 and msg in last()
    assert lib.vgemm_w4_pack(None, ctypes.byref(W), 0, 1, FAKE, 32, FAKE, None, 1, FAKE) == -1 and msg in last()


@pytest.mark.parametrize("w,a,e,M,msg", [
    (dict(count=2), {}, {}, 1, "one matrix"), ({}, {}, {}, -1, "bad arguments"), ({}, dict(src=3), {}, 1, "VGEMM_SRC_I8"), ({}, dict(hi=None), {}, 1, "SRC_I8"),
    ({}, dict(ld8=48), {}, 1, "ld8"), ({}, dict(ld8=72), {}, 1, "ld8"), ({}, dict(hi=FAKE + 8), {}, 1, "16-byte"), ({}, dict(lo=FAKE + 4), {}, 1, "16-byte"),
    ({}, dict(src=1, x=FAKE, ldx=64, K=64), {}, 1, "SRC_X32"), ({}, dict(src=1, x=FAKE, ldx=64, K=60, rowmax=FAKE), {}, 1, "SRC_X32"),
    ({}, dict(src=1, x=FAKE, ldx=60, K=64, rowmax=FAKE), {}, 1, "SRC_X32"), (dict(K=62), dict(src=1, x=FAKE, ldx=64, K=62, rowmax=FAKE), {}, 1, "SRC_X32"),
    ({}, {}, dict(Y=None), 1, "null Y"), ({}, {}, dict(ldy=63), 1, "ldy < N"), ({}, {}, dict(epi=3), 1, "EPI_PLAIN or EPI_GEGLU"),
    ({}, {}, dict(epi=2), 1, "Lphi"), (dict(N=63), {}, dict(epi=2, Lphi=FAKE), 1, "even N"), ({}, {}, dict(epi=2, Lphi=FAKE, ldy=31), 1, "ldy >= N / 2")])
def test_w4_refusals(w, a, e, M, msg):
    W = _lib.W4(**{**dict(N=64, K=64, group=64, count=1, q=FAKE, cst=FAKE), **w})
    A = _lib.ASrc(**{**dict(src=0, hi=FAKE, ld8=64), **a})
    E = _lib.AEpi(**{**dict(Y=FAKE, ldy=64), **e})
    assert _lib.load().vgemm_w4(None, ctypes.byref(A), M, ctypes.byref(W), ctypes.byref(E)) == -1
    assert msg in last()


@pytest.mark.parametrize("args,msg", [
    ((0, 3, FAKE, 32, FAKE, None, 1, FAKE), "of 2"), ((-1, 1, FAKE, 32, FAKE, None, 1, FAKE), "of 2"), ((2, 1, FAKE, 32, FAKE, None, 1, FAKE), "of 2"),
    ((0, 1, None, 32, FAKE, None, 1, FAKE), "required"), ((0, 1, FAKE, 31, FAKE, None, 1, FAKE), "ldn"), ((0, 1, FAKE, 32, FAKE, None, 0, FAKE), "lds"),
    ((0, 1, FAKE, 32, FAKE + 1, None, 1, FAKE), "required"), ((0, 1, FAKE, 32, FAKE, None, 1, None), "required")])
def test_pack_refusals(args, msg):
    W = _lib.W4(N=64, K=64, group=64, count=2, q=FAKE, cst=FAKE)
    assert _lib.load().vgemm_w4_pack(None, ctypes.byref(W), *args) == -1
    assert msg in last()


@pytest.mark.parametrize("r,a,msg", [
    (dict(experts=0), {}, "topk <= experts"), (dict(experts=513), {}, "experts <= 512"), (dict(topk=0), {}, "topk"), (dict(topk=17, experts=20), {}, "topk <= 16"),
    (dict(topk=9), {}, "topk <= experts"), (dict(W=None), {}, "required"), (dict(cst=FAKE + 4), {}, "16-byte"), (dict(Lexp=None), {}, "required"),
    (dict(idx=None), {}, "required"), (dict(p=None), {}, "required"), (dict(ldw=48), {}, "ldw >= K"), (dict(ldw=72), {}, "ldw % 16"), ({}, dict(K=40), "K % 16"),
    ({}, dict(K=16400, ld8=16400), "K <= 16384"), ({}, dict(src=1), "VGEMM_SRC_I8"), ({}, dict(hi=None), "SRC_I8"), ({}, dict(ld8=48), "ld8")])
def test_route_refusals(r, a, msg):
    R = _lib.MoeRoute(**{**dict(W=FAKE, ldw=64, cst=FAKE, experts=8, topk=2, Lexp=FAKE, idx=FAKE, p=FAKE), **r})
    if a.get("K", 0) > 16384:
        R.ldw = 16400
    A = _lib.ASrc(**{**dict(src=0, hi=FAKE, ld8=64, K=64), **a})
    assert _lib.load().vgemm_moe_route(None, ctypes.byref(A), 2, ctypes.byref(R)) == -1
    assert msg in last()


@pytest.mark.parametrize("up,down,c,a,msg", [
    (dict(N=100), {}, {}, {}, "up.N == 2 down.K"), ({}, dict(count=3), {}, {}, "equal counts"), (dict(count=513), dict(count=513), {}, {}, "at most 512"),
    (dict(N=60), dict(K=30), {}, {}, "down.K % 4"), (dict(group=8), {}, {}, {}, "group of 32"), ({}, dict(q=None), {}, {}, "q and cst"),
    ({}, {}, dict(topk=0), {}, "topk"), ({}, {}, dict(topk=17), {}, "topk"), ({}, {}, dict(idx=None), {}, "required"), ({}, {}, dict(p=None), {}, "required"),
    ({}, {}, dict(Lphi=None), {}, "required"), ({}, {}, dict(Y=None), {}, "required"), ({}, {}, dict(ldy=63), {}, "ldy"), ({}, {}, dict(ws=None), {}, "workspace"),
    ({}, {}, dict(ws=FAKE + 8), {}, "workspace"), ({}, {}, dict(ws_bytes=100), {}, "workspace"), ({}, {}, {}, dict(src=1), "VGEMM_SRC_I8"), ({}, {}, {}, dict(ld8=32), "ld8")])
def test_moe_refusals(up, down, c, a, msg):
    U = _lib.W4(**{**dict(N=64, K=64, group=64, count=4, q=FAKE, cst=FAKE), **up})
    V = _lib.W4(**{**dict(N=64, K=32, group=64, count=4, q=FAKE, cst=FAKE), **down})
    P = _lib.Moe(**{**dict(up=U, down=V, topk=2, idx=FAKE, p=FAKE, Lphi=FAKE, Y=FAKE, ldy=64, ws=FAKE, ws_bytes=1 << 20), **c})
    A = _lib.ASrc(**{**dict(src=0, hi=FAKE, ld8=64), **a})
    assert _lib.load().vgemm_moe(None, ctypes.byref(A), 2, ctypes.byref(P)) == -1
    assert msg in last()


def test_limits():
    """Row strides and row counts past what a kernel addresses are refused before any launch."""
    lib, W, E = _lib.load(), _lib.W4(N=64, K=64, group=64, count=1, q=FAKE, cst=FAKE), _lib.AEpi(Y=FAKE, ldy=64)
    rows, x32 = _lib.ASrc(src=0, hi=FAKE, ld8=64, K=64), _lib.ASrc(src=1, x=FAKE, rowmax=FAKE, K=64, ldx=(1 << 23) + 4)
    wide = _lib.ASrc(src=0, hi=FAKE, ld8=(1 << 21) + 16, K=64)
    R = _lib.MoeRoute(W=FAKE, ldw=64, cst=FAKE, experts=8, topk=2, Lexp=FAKE, idx=FAKE, p=FAKE)
    P = _lib.Moe(up=W, down=_lib.W4(N=64, K=32, group=64, count=1, q=FAKE, cst=FAKE), topk=1, idx=FAKE, p=FAKE, Lphi=FAKE, Y=FAKE, ldy=64, ws=FAKE, ws_bytes=1 << 20)
    for call, msg in ((lambda: lib.vgemm_w4(None, ctypes.byref(rows), (1 << 18) + 1, ctypes.byref(W), ctypes.byref(E)), "w4: at most"),
                      (lambda: lib.vgemm_w4(None, ctypes.byref(wide), 1, ctypes.byref(W), ctypes.byref(E)), "ld8 above"),
                      (lambda: lib.vgemm_w4(None, ctypes.byref(x32), 1, ctypes.byref(W), ctypes.byref(E)), "ldx above"),
                      (lambda: lib.vgemm_moe_route(None, ctypes.byref(rows), (1 << 18) + 1, ctypes.byref(R)), "moe_route: at most"),
                      (lambda: lib.vgemm_moe_route(None, ctypes.byref(wide), 1, ctypes.byref(R)), "ld8 above"),
                      (lambda: lib.vgemm_moe(None, ctypes.byref(wide), 1, ctypes.byref(P)), "ld8 above"),
                      (lambda: lib.vgemm_rmsnorm_q(None, FAKE, None, (1 << 22) + 1, 64, FAKE, 100000, None, FAKE, None, FAKE, 64), "rmsnorm_q: at most")):
        assert call() == -3 and msg in last()


def test_sizes():
    assert w4.w4_bytes(16, 128, 128) == 1024 + 32
    assert w4.w4_bytes(17, 129, 32) == 4 * (1024 + 128)
    for bad in ((0, 64, 64), (64, 0, 64), (64, 32769, 64), (64, 64, 48)):
        assert w4.w4_bytes(*bad) == 0
    assert moe.moe_workspace_bytes(0, 2, 64) == 0 and moe.moe_workspace_bytes(1, 17, 64) == 0
    assert moe.moe_workspace_bytes(10, 2, 64) >= 20 * 64 * 4
    assert moe.moe_workspace_bytes(10**6, 4, 64) == moe.moe_workspace_bytes(128, 4, 64)       # a pass takes 512 pairs


def test_weights_object_refuses_shapes():
    W = w4.W4Weights.__new__(w4.W4Weights)
    W.N, W.K, W.group, W.count, W.q = 8, 64, 32, 1, torch.empty(1)
    good = (torch.zeros((8, 32), dtype=torch.uint8), torch.zeros((8, 2), dtype=torch.int16), None, torch.zeros((8, 4), dtype=torch.int32))
    for i, bad in ((0, torch.zeros((8, 31), dtype=torch.uint8)), (0, torch.zeros((8, 32), dtype=torch.int8)), (1, torch.zeros((8, 1), dtype=torch.int16)),
                   (1, torch.zeros((7, 2), dtype=torch.int16)), (2, torch.zeros((8, 2), dtype=torch.int32)), (3, torch.zeros((8, 3), dtype=torch.int32))):
        with pytest.raises(ValueError):
            W.pack(*[bad if j == i else t for j, t in enumerate(good)])
    with pytest.raises(ValueError):
        w4.W4Weights(8, 64, 48, device="cpu")


# ---------------------------------------------------------------- the tests' formulas

def test_formula_norm():
    """Against the real-valued norm: y / 65536 = h g / 65536 / rms(h) within the formula's three roundings."""
    rng = np.random.default_rng(1)
    x, g = np.round(rng.normal(size=(4, 512)) * 100000).astype(np.int32), rng.integers(30000, 90000, 512, dtype=np.int32)
    h, y = lm.rmsnorm(x, None, g, 100000)
    real = h / np.sqrt((h.astype(float) ** 2).mean(1, keepdims=True) + 2.0**32 / 100000) * g
    # half a step of the quotient times g / 65536 and half a step of the product, and the root's own step: sd is the floor of
    # 256 rms, so it is off by less than 1 / sd relative to itself
    sd = 256 * np.sqrt((h.astype(float) ** 2).mean(1, keepdims=True))
    assert (np.abs(y - real) <= 0.5 * g / 65536 + 0.5 + np.abs(real) * 2.0 / sd + 1e-6).all()


def test_formula_product_and_codes():
    rng = np.random.default_rng(2)
    w = lm.Weights(rng, 6, 45, 32)
    d = w.dense()
    for n in range(6):
        for k in range(45):
            byte = int(w.nib[n, k // 2])
            u = byte & 15 if k % 2 == 0 else byte >> 4
            assert d[n, k] == (u - int(w.z[n, k // 32])) * min(int(w.sc[n, k // 32]), 4095)
    q = rng.integers(-127, 128, (3, 45))
    y = lm.product(q, np.array([0, 3, 7]), d, w.msb)
    for r in range(3):
        for n in range(6):
            v = sum(int(q[r, k]) * int(d[n, k]) for k in range(45)) * int(w.msb[n, 0])
            s = int(w.msb[n, 1]) - (0, 3, 7)[r]
            assert y[r, n] == max(-2**31, min(2**31 - 1, max(-2**31, min(2**31 - 1, (v + (1 << s >> 1)) >> s)) + int(w.msb[n, 2])))


def test_formula_route_shares():
    """Shares are the softmax in Q15 within a step, and ties take the lowest index."""
    w = np.zeros((5, 16), np.int8)
    cst = np.zeros((5, 4), np.int32)
    cst[:, 2] = [65536, 0, 131072, 131072, -65536]
    idx, p, z = lm.route(np.zeros((1, 16)), [0], w, cst, 3, True, lm.exp_table())
    assert idx.tolist() == [[2, 3, 0]] and z.tolist() == [[65536, 0, 131072, 131072, -65536]]
    soft = np.exp([2.0, 2.0, 1.0]) / np.exp([2.0, 2.0, 1.0]).sum() * 32768
    assert np.abs(p[0] - soft).max() <= 1.0

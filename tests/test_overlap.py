"""Operands that share memory: the exact test of two strided operands against every byte of both, and the entry points that refuse."""
import ctypes as C
import os
import random
import subprocess

import pytest

from helixml_b200 import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    src, so = str(d / "t.cpp"), str(d / "t.so")
    open(src, "w").write('#include "hx_overlap.h"\n'
                         'extern "C" int t(hx::Rows *a, hx::Rows *b) { return hx::overlap(*a, *b); }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "helixml_b200", "csrc"), src,
                    "-o", so], check=True)
    return C.CDLL(so).t


class Rows(C.Structure):
    _fields_ = [("at", C.c_void_p)] + [(n, C.c_int64) for n in ("outer", "outer_stride", "inner", "inner_stride", "bytes")]


def every_byte(r):
    at, no, so, ni, si, n = r
    return {at + i * so + j * si + k for i in range(no) for j in range(ni) for k in range(n)}


def test_against_every_byte(overlap):
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(30000):
        strides = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 24, 30, 48]) for _ in range(2)]
        rows = []
        for _ in range(2):
            if rng.random() < 0.4:
                strides = [rng.choice([0, 1, 2, 5, 7, 16, 20, 40]) for _ in range(2)]
            rows.append((1000 + rng.randrange(0, 120), rng.randrange(0, 5), strides[0], rng.randrange(0, 5), strides[1], rng.randrange(0, 9)))
        want = bool(every_byte(rows[0]) & every_byte(rows[1]))
        assert bool(overlap(*(C.byref(Rows(*r)) for r in rows))) == want, rows
        seen[want] += 1
    assert min(seen) > 3000


def test_large_operands_take_no_time(overlap):
    """Halves of one buffer of 2^31 rows, batch first and time first."""
    n = 1 << 20
    for outer, inner in (((n, 4096 * 2048), (2048, 4096)), ((2048, 4096), (n, 4096 * 2048))):
        a = Rows(1 << 30, *outer, *inner, 2048)
        for shift, want in ((2048, 0), (2047, 1), (0, 1), (4096 * 5 + 2048, 0), (4096 * 5 + 2049, 1)):
            assert overlap(C.byref(a), C.byref(Rows((1 << 30) + shift, *outer, *inner, 2048))) == want
    assert overlap(C.byref(Rows(0, 4, 8, 4, 8, 8)), C.byref(Rows(0, 4, 8, 4, 8, 8))) == 0   # NULL operands


# ------------------------------------------------------------------ the entry points; nothing is launched, so that the addresses are never used
FAR = 1 << 32


def scan_args(kind, **kw):
    a = kind()
    a.batch, a.seq_len, a.d_inner, a.io_dtype, a.gate = 2, 5, 8, L.HX_F32, L.GATE_SIGMOID
    for i, (name, _) in enumerate(kind._fields_):
        if name.endswith("batch_stride"):
            setattr(a, name, 40)
        elif name.endswith("row_stride"):
            setattr(a, name, 8)
        elif name in ("x", "g", "h", "dh", "dx", "dg", "states", "h0", "h_last", "dh0", "dh_last", "lengths"):
            setattr(a, name, FAR * (1 + i))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


SCAN = [("hx_gated_scan_fwd", L.GatedScanArgs, ("h", "h_last", "states"), ("x", "g", "h0", "lengths")),
        ("hx_gated_scan_bwd", L.GatedScanBwdArgs, ("dx", "dg", "dh0"), ("x", "g", "dh", "states", "dh_last", "lengths"))]


@pytest.mark.parametrize("fn,kind,outs,ins", SCAN, ids=["forward", "backward"])
def test_scans_refuse_shared_memory(fn, kind, outs, ins):
    call = getattr(L.lib(), fn)
    for o in outs:
        for i in (*ins, *outs):
            if i == o:
                continue
            for shift in (0, 4):
                a = scan_args(kind)
                setattr(a, o, getattr(a, i) + shift)
                assert call(C.byref(a), None) == 10 and b"share memory" in L.lib().hx_last_error(), (o, i)
    a = scan_args(kind, workspace=FAR, workspace_bytes=1 << 20, batch=1, seq_len=4096)
    setattr(a, outs[0], FAR + 64)
    assert call(C.byref(a), None) == 10 and b"share memory" in L.lib().hx_last_error()


def test_step_refuses_shifted_operands():
    lib = L.lib()
    step = lambda x=FAR, g=2 * FAR, h=3 * FAR, ho=4 * FAR, y=5 * FAR, xs=8, ys=8: lib.hx_gated_scan_step(
        x, xs, g, 8, h, ho, y, ys, 2, 8, L.GATE_SIGMOID, L.HX_F32, None)
    for bad in (dict(ho=3 * FAR + 4), dict(y=FAR + 4), dict(y=2 * FAR + 32), dict(y=3 * FAR), dict(y=4 * FAR), dict(ho=FAR),
                dict(y=FAR, xs=0), dict(y=FAR, xs=16, ys=8)):
        assert step(**bad) == 10 and b"share memory" in lib.hx_last_error(), bad


def test_4_bit_entry_points_refuse_shared_memory():
    lib = L.lib()
    m = L.W4MatrixArgs(16, 256, 64, L.HX_F32, FAR, 2 * FAR, 3 * FAR)
    parts = (FAR, 2 * FAR, 3 * FAR)
    for at in parts:
        assert lib.hx_w4_quantize(at + 32, 256, L.HX_F32, C.byref(m), None) == 10 and b"share memory" in lib.hx_last_error()
        assert lib.hx_w4_dequantize(C.byref(m), at + 32, 256, L.HX_F32, None) == 10 and b"share memory" in lib.hx_last_error()
        assert lib.hx_gemm_w4(4 * FAR, 256, L.HX_F32, C.byref(m), None, at, 16, L.HX_F32, 2, 0, None) == 10
        assert b"share memory" in lib.hx_last_error()
    assert lib.hx_w4_pack(FAR + 16, 256, C.byref(m), None) == 10 and b"share memory" in lib.hx_last_error()
    assert lib.hx_gemm_w4(4 * FAR, 256, L.HX_F32, C.byref(m), None, 4 * FAR + 1000, 16, L.HX_F32, 2, 0, None) == 10
    assert lib.hx_gemm_w4(4 * FAR, 256, L.HX_F32, C.byref(m), 5 * FAR, 5 * FAR, 16, L.HX_F32, 2, 0, None) == 10
    m.scale = FAR + 64
    assert lib.hx_w4_quantize(4 * FAR, 256, L.HX_F32, C.byref(m), None) == 10 and b"share memory" in lib.hx_last_error()

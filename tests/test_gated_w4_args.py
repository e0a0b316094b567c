"""CPU tests of the C boundary of the gated recurrence and the 4-bit products: layout of the structures, argument errors, sizes."""
import ctypes as C
import os
import subprocess
import tempfile

from helixml_b200 import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = C.c_void_p(256)   # never dereferenced: the checks come first


def test_struct_layout_matches_c():
    fields = [("hx_gated_scan_args", L.GatedScanArgs, ("x", "x_batch_stride", "h_row_stride", "h0", "lengths")),
              ("hx_gated_scan_bwd_args", L.GatedScanBwdArgs, ("x", "dg", "x_batch_stride", "dg_row_stride", "states", "lengths")),
              ("hx_w4_matrix", L.W4MatrixArgs, ("group", "codes", "scale", "zero"))]
    lines, want = [], []
    for c, py, names in fields:
        lines.append(f'printf("%zu ", sizeof({c}));')
        want.append(C.sizeof(py))
        for n in names:
            lines.append(f'printf("%zu ", offsetof({c}, {n}));')
            want.append(getattr(py, n).offset)
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "helix_b200.h"\nint main(void) {' + "\n".join(lines) + "return 0; }"
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(src, "w").write(prog)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        got = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in got] == want


def gated(kind, **kw):
    a = kind()
    a.batch, a.seq_len, a.d_inner, a.io_dtype, a.gate = 2, 5, 8, L.HX_F32, L.GATE_SIGMOID
    for name, _ in kind._fields_:
        if name.endswith("batch_stride"):
            setattr(a, name, 40)
        elif name.endswith("row_stride"):
            setattr(a, name, 8)
    for n in ("x", "g", "h", "dh", "dx", "dg", "states"):
        if hasattr(a, n):
            setattr(a, n, 256)
    for k, v in kw.items():
        setattr(a, k, v)
    return C.byref(a)


def test_gated_scan_argument_errors():
    lib = L.lib()
    for fn, kind, nulls, outs in ((lib.hx_gated_scan_fwd, L.GatedScanArgs, ("x", "g", "h"), ("h",)),
                                  (lib.hx_gated_scan_bwd, L.GatedScanBwdArgs, ("x", "g", "dh", "dx", "dg", "states"), ("dx", "dg"))):
        assert fn(None, None) == 10
        for bad in ("batch", "seq_len", "d_inner"):
            assert fn(gated(kind, **{bad: -1}), None) == 2
        assert fn(gated(kind, io_dtype=L.HX_U8), None) == 4
        assert fn(gated(kind, gate=2), None) == 10 and b"gate" in lib.hx_last_error()
        for n in nulls:
            assert fn(gated(kind, **{n: None}), None) == 10, n
        assert fn(gated(kind, x_row_stride=-8), None) == 10
        for o in outs:
            assert fn(gated(kind, **{f"{o}_row_stride": 7}), None) == 1
            assert fn(gated(kind, **{f"{o}_batch_stride": 39}), None) == 1
            assert fn(gated(kind, **{f"{o}_batch_stride": 0}), None) == 1
        for empty in ("batch", "d_inner"):
            assert fn(gated(kind, **{empty: 0}), None) == 0


def test_gated_scan_workspace():
    lib = L.lib()
    n = C.c_size_t(7)
    q = lambda *a: (lib.hx_gated_scan_workspace_bytes(*a, C.byref(n)), n.value)
    assert q(32, 2048, 1536, L.HX_BF16) == (0, 0)          # enough chains: the sequence is not cut
    st, size = q(1, 4096, 257, L.HX_F32)
    assert st == 0 and size > 0 and size % (8 * 258) == 0   # maps of whole pairs of channels
    assert q(0, 4096, 257, L.HX_F32) == (0, 0) and q(1, 32, 257, L.HX_F32) == (0, 0)
    assert q(-1, 5, 5, L.HX_F32)[0] == 2 and q(1, 5, 5, L.HX_U8)[0] == 4
    assert lib.hx_gated_scan_workspace_bytes(1, 5, 5, L.HX_F32, None) == 10
    for fn, kind in ((lib.hx_gated_scan_fwd, L.GatedScanArgs), (lib.hx_gated_scan_bwd, L.GatedScanBwdArgs)):
        big = dict(batch=1, seq_len=4096, d_inner=8, workspace=256)
        need = q(1, 4096, 8, L.HX_F32)[1]
        assert fn(gated(kind, workspace_bytes=need - 1, **big), None) == 10 and b"needed" in lib.hx_last_error()
        assert fn(gated(kind, workspace_bytes=need, **{**big, "workspace": 264}), None) == 10


def test_gated_step_argument_errors():
    lib = L.lib()

    def step(x=P, xs=8, g=P, gs=8, h=P, ho=P, y=P, ys=8, B=2, D=8, gate=0, dt=L.HX_F32):
        return lib.hx_gated_scan_step(x, xs, g, gs, h, ho, y, ys, B, D, gate, dt, None)

    for n in ("x", "g", "h", "ho", "y"):
        assert step(**{n: None}) == 10
    assert step(B=-1) == 2 and step(D=-1) == 2 and step(dt=5) == 4 and step(gate=7) == 10
    assert step(ys=7) == 1 and step(xs=-1) == 10 and step(B=0) == 0 and step(D=0, x=None) == 0


def w4(**kw):
    m = L.W4MatrixArgs()
    m.rows, m.cols, m.group, m.scale_dtype, m.codes, m.scale = 16, 256, 64, L.HX_F32, 256, 256
    for k, v in kw.items():
        setattr(m, k, v)
    return C.byref(m)


def test_w4_argument_errors():
    lib = L.lib()
    calls = {
        "quantize": lambda m, W=P, ld=256, dt=L.HX_F32: lib.hx_w4_quantize(W, ld, dt, m, None),
        "pack": lambda m, W=P, ld=256: lib.hx_w4_pack(W, ld, m, None),
        "dequantize": lambda m, W=P, ld=256, dt=L.HX_F32: lib.hx_w4_dequantize(m, W, ld, dt, None),
        "gemm": lambda m, W=P, ld=256, dt=L.HX_F32: lib.hx_gemm_w4(W, ld, dt, m, None, P, 16, L.HX_F32, 2, 0, None),
    }
    for name, f in calls.items():
        assert f(None) == 10, name
        assert f(w4(rows=2 ** 31 - 1)) == 2 and f(w4(rows=-1)) == 2 and f(w4(cols=-64)) == 2 and f(w4(group=48)) == 2, name
        assert f(w4(cols=96)) == 1 and f(w4(scale_dtype=L.HX_U8)) == 4, name
        assert f(w4(codes=None)) == 10 and f(w4(scale=None)) == 10 and f(w4(codes=264)) == 10, name
        assert f(w4(), W=None) == 10, name
        assert f(w4(rows=0)) == 0, name
        if name != "pack":
            assert f(w4(), dt=L.HX_U8) == 4, name
    assert calls["dequantize"](w4(), ld=255) == 1
    assert calls["quantize"](w4(), ld=-1) == 10 and calls["gemm"](w4(), ld=-1) == 10
    g = lambda M=2, ldc=16, epi=0, cdt=L.HX_F32, C_=P: lib.hx_gemm_w4(P, 256, L.HX_F32, w4(), None, C_, ldc, cdt, M, epi, None)
    assert g(M=-1) == 2 and g(M=0) == 0 and g(ldc=15) == 1 and g(epi=3) == 10 and g(cdt=9) == 4 and g(C_=None) == 10
    assert lib.hx_gemm_w4(P, 256, L.HX_F32, w4(cols=0), None, P, 16, L.HX_F32, 2, 0, None) == 2


def test_w4_row_bytes():
    lib = L.lib()
    assert [lib.hx_w4_row_bytes(k) for k in (-5, 0, 32, 128, 160, 256, 2 ** 31 - 128)] == [0, 0, 64, 64, 128, 128, (2 ** 31 - 128) // 2]

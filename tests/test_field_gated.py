"""The C boundary of the gated projections and of the norm and clipping of gradients
without a GPU: struct layouts, workspace sizes, refusals. A null context is refused last,
so that every other refusal shows here."""
import ctypes
import os
import subprocess
import tempfile

import pytest

from gsplat_tt_amd import _lib as L

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")


def test_struct_layouts():
    fields = {"gs_gated_linear": L.GsGatedLinear, "gs_tensor": L.GsTensor}
    lines = [f'printf("{t} %zu\\n", sizeof({t}));' for t in fields]
    lines += [f'printf("{t}.{f} %zu\\n", offsetof({t}, {f}));'
              for t, c in fields.items() for f, _ in c._fields_]
    prog = ('#include <stddef.h>\n#include <stdio.h>\n#include "gsplat_hip.h"\n'
            "int main(void) {\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        with open(c, "w") as f:
            f.write(prog)
        subprocess.run(["gcc", "-std=c11", "-I", HEADER, c, "-o", exe], check=True)
        out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    for line in out.strip().splitlines():
        key, val = line.rsplit(" ", 1)
        t, _, f = key.partition(".")
        got = getattr(fields[t], f).offset if f else ctypes.sizeof(fields[t])
        assert got == int(val), key


def _gated(**changes):
    d = L.GsGatedLinear(0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 100, 32, 16, 16, 16, 16, 0,
                        2, 0)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


GATED_REFUSED = [dict(n=-1), dict(hidden=0), dict(dim=0), dict(dtype=2), dict(act=4),
                 dict(x=None), dict(w_gate=None), dict(w_up=None), dict(x=0x10002),
                 dict(w_up=0x30001), dict(b_gate=0x40002), dict(b_up=0x50001), dict(x_stride=-1),
                 dict(gate_stride=1 << 40), dict(up_stride=-16)]
GATED_PAST = [dict(n=(1 << 31) - 255), dict(hidden=(1 << 20) + 1), dict(dim=65537)]


def test_gated_linear_workspace():
    lib = L.load_library()
    for grad in (0, 1):
        for dtype in (0, 1):
            for n in (1, 100, 10 ** 7):
                size = lib.gs_gated_linear_workspace(ctypes.byref(_gated(n=n, dtype=dtype)), grad)
                assert 0 <= size < 5 << 30
        for bad in GATED_REFUSED + GATED_PAST:
            assert lib.gs_gated_linear_workspace(ctypes.byref(_gated(**bad)), grad) == -1, bad
        # the longest rows and the widest weights
        big = _gated(n=(1 << 31) - 256, dim=65536, x_stride=65536, gate_stride=65536,
                     up_stride=65536)
        assert lib.gs_gated_linear_workspace(ctypes.byref(big), grad) > 0
        big = _gated(n=(1 << 31) - 256, hidden=1 << 20)
        assert lib.gs_gated_linear_workspace(ctypes.byref(big), grad) > 0
    assert lib.gs_gated_linear_workspace(ctypes.byref(_gated(n=0)), 1) >= 0


def test_gated_linear_refusals():
    lib = L.load_library()

    def call(d, h=0x60000, stride=32, ws=0x100000, size=1 << 40):
        return lib.gs_gated_linear_dev(None, ctypes.byref(d), h, stride, ws, size, None)

    def grad(d, dh=(0x60000, 32), dx=(0x70000, 16), dwg=(0x80000, 16), dwu=(0x90000, 16),
             db=(0xa0000, 0xb0000), ws=0x100000, size=1 << 40):
        return lib.gs_gated_linear_grad_dev(None, ctypes.byref(d), *dh, *dx, *dwg, *dwu, *db, ws,
                                            size, None)

    for f in (call, grad):
        assert f(_gated()) == L.GS_E_INVALID and b"ctx" in lib.gs_last_error()
        for bad in GATED_REFUSED:
            assert f(_gated(**bad)) == L.GS_E_INVALID and b"ctx" not in lib.gs_last_error(), bad
        for bad in GATED_PAST:
            assert f(_gated(**bad)) == L.GS_E_CAPACITY, bad
    assert lib.gs_gated_linear_dev(None, None, 0x60000, 32, 0x100000, 1 << 40, None) == \
        L.GS_E_INVALID and b"null desc" in lib.gs_last_error()
    need = lib.gs_gated_linear_workspace(ctypes.byref(_gated(n=5000)), 1)
    for bad in (dict(h=None), dict(h=0x60002), dict(stride=31)):
        assert call(_gated(), **bad) == L.GS_E_INVALID and b"ctx" not in lib.gs_last_error(), bad
    for bad in (dict(dh=(None, 32)), dict(dh=(0x60001, 32)), dict(dh=(0x60000, -1)),
                dict(dx=(None, 16)), dict(dx=(0x70000, 15)), dict(dwg=(None, 16)),
                dict(dwu=(0x90000, 8)), dict(db=(0xa0002, None)), dict(db=(None, 0xb0001)),
                dict(ws=0x100010), dict(ws=None), dict(size=need - 1), dict(size=-1)):
        assert grad(_gated(n=5000), **bad) == L.GS_E_INVALID, bad
        assert b"ctx" not in lib.gs_last_error(), bad


def _tensors(*rows):
    return (L.GsTensor * max(1, len(rows)))(*(L.GsTensor(*r, 0) for r in rows))


def test_grad_norm_workspace_and_refusals():
    lib = L.load_library()
    good = _tensors((0x10000, 1, 100, 0, 0), (0x20000, 5, 7, 9, 1), (None, 0, 7, 9, 1))
    at = ctypes.addressof(good)
    assert lib.gs_grad_norm_workspace(at, 3) > 0
    assert lib.gs_grad_norm_workspace(None, 0) >= 0
    huge = _tensors(*[(0x10000, 1, 1 << 40, 0, 0)] * 200)
    assert 0 < lib.gs_grad_norm_workspace(ctypes.addressof(huge), 200) < 1 << 20
    assert lib.gs_grad_norm_dev(None, at, 3, 0, 0x1000, 0x100000, 1 << 20, None) == \
        L.GS_E_INVALID and b"ctx" in lib.gs_last_error()
    for bad, code in (((0x10000, -1, 5, 5, 0), L.GS_E_INVALID), ((0x10000, 1, -5, 5, 0), L.GS_E_INVALID),
                      ((0x10000, 2, 5, 5, 2), L.GS_E_INVALID), ((None, 2, 5, 5, 0), L.GS_E_INVALID),
                      ((0x10002, 2, 5, 5, 0), L.GS_E_INVALID), ((0x10001, 2, 5, 5, 1), L.GS_E_INVALID),
                      ((0x10000, 2, 5, -5, 0), L.GS_E_INVALID),
                      ((0x10000, 2, 5, 1 << 40, 0), L.GS_E_INVALID),
                      ((0x10000, 1 << 30, 1 << 30, 1 << 31, 0), L.GS_E_CAPACITY)):
        one = _tensors(bad)
        assert lib.gs_grad_norm_workspace(ctypes.addressof(one), 1) == -1, bad
        rc = lib.gs_grad_norm_dev(None, ctypes.addressof(one), 1, 0, 0x1000, 0x100000, 1 << 20, None)
        assert rc == code and b"ctx" not in lib.gs_last_error(), bad
    for args in ((at, 3, 2, 0x1000, 0x100000, 1 << 20), (at, -3, 0, 0x1000, 0x100000, 1 << 20),
                 (None, 3, 0, 0x1000, 0x100000, 1 << 20), (at, 3, 0, None, 0x100000, 1 << 20),
                 (at, 3, 0, 0x1002, 0x100000, 1 << 20), (at, 3, 0, 0x1000, 0x100000, 0),
                 (at, 3, 0, 0x1000, 0x100001, 1 << 20), (at, 3, 0, 0x1000, None, 1 << 20)):
        assert lib.gs_grad_norm_dev(None, *args, None) == L.GS_E_INVALID, args
        assert b"ctx" not in lib.gs_last_error(), args
    assert lib.gs_grad_norm_dev(None, at, (1 << 20) + 1, 0, 0x1000, 0x100000, 1 << 20, None) == \
        L.GS_E_CAPACITY


def _clip(ins, outs, norm=0x1000, max_norm=1.0, kind=-1, ws=None, size=0):
    """What the clipping of these lists says to a null context: b"" where nothing else
    is wrong."""
    lib = L.load_library()
    i, o = _tensors(*ins), _tensors(*outs)
    assert lib.gs_grad_clip_dev(None, ctypes.addressof(i), ctypes.addressof(o), len(ins), kind,
                                norm, max_norm, ws, size, None) == L.GS_E_INVALID
    text = lib.gs_last_error()
    return b"" if b"null ctx" in text else text


F, B = 0, 1


def test_clip_takes_what_shares_no_memory():
    a, b = (0x10000, 1, 100, 0, F), (0x20000, 1, 100, 0, F)
    assert _clip([a], [a]) == b"" and _clip([a], [b]) == b"" and _clip([], []) == b""
    assert _clip([a, b], [a, b]) == b""
    assert _clip([a, a], [b, (0x30000, 1, 100, 0, B)]) == b""  # inputs may share
    # one run into rows and back, and end to end
    assert _clip([a], [(0x20000, 10, 10, 12, B)]) == b"" and _clip([(0x20000, 10, 10, 12, B)], [a]) == b""
    assert _clip([a, (0x10000 + 400, 1, 5, 0, F)], [a, (0x10000 + 400, 1, 5, 0, F)]) == b""
    # columns of one matrix of 64 columns
    left, mid, right = ((0x10000 + 4 * c, 8, w, 64, F) for c, w in ((0, 10), (10, 30), (40, 24)))
    for order in ([left, mid, right], [right, left, mid]):
        assert _clip(order, order) == b""
    assert _clip([left], [mid[:2] + (10,) + mid[3:]]) == b""
    # a row in the gap between rows
    gap = (0x10000 + 4 * 74, 1, 10, 0, F)
    assert _clip([left, gap], [left, gap]) == b""


@pytest.mark.parametrize("ins,outs", [
    ([(0x10000, 1, 100, 0, F)] * 2, [(0x10000, 1, 100, 0, F)] * 2),
    ([(0x10000, 1, 100, 0, F)], [(0x10004, 1, 100, 0, F)]),
    ([(0x10000, 1, 100, 0, F)], [(0x10000, 1, 100, 0, B)]),
    ([(0x10000, 1, 100, 0, F)], [(0x10000, 10, 10, 12, F)]),
    ([(0x10000, 1, 100, 0, F), (0x20000, 1, 9, 0, F)],
     [(0x20000, 1, 100, 0, F), (0x30000, 1, 9, 0, F)]),
    ([(0x10000, 1, 100, 0, F), (0x40000, 1, 100, 0, F)],
     [(0x20000, 1, 100, 0, F), (0x20000 + 396, 1, 100, 0, F)]),
    # columns that meet, columns of other strides, a row across the rows
    ([(0x10000, 8, 10, 64, F), (0x10000 + 36, 8, 10, 64, F)],) * 2,
    ([(0x10000, 8, 10, 64, F), (0x10000 + 240, 8, 10, 64, F)],) * 2,
    ([(0x10000, 8, 10, 64, F), (0x10000 + 80, 8, 10, 32, F)],) * 2,
    ([(0x10000, 8, 10, 64, F), (0x10000 + 80, 1, 60, 0, F)],) * 2,
    ([(0x10000, 8, 10, 64, F), (0x10000 + 256 * 3 + 20, 1, 5, 0, F)],) * 2,
])
def test_clip_refuses_shared_memory(ins, outs):
    assert b"shares memory" in _clip(ins, outs)


def test_clip_refusals():
    a, b = (0x10000, 1, 100, 0, F), (0x20000, 1, 100, 0, F)
    assert b"rows and cols" in _clip([a], [(0x20000, 1, 99, 0, F)])
    assert b"rows and cols" in _clip([(0x10000, 10, 10, 12, F)], [(0x20000, 20, 5, 6, F)])
    assert b"overlap" in _clip([a], [(0x20000, 10, 10, 9, F)])
    assert b"overlap" in _clip([(0x10000, 10, 10, 0, F)], [(0x10000, 10, 10, 0, F)])
    assert b"max_norm" in _clip([a], [b], max_norm=-0.5)
    assert b"max_norm" in _clip([a], [b], max_norm=float("nan"))
    assert b"norm is null" in _clip([a], [b], norm=None)
    assert b"aligned" in _clip([a], [b], norm=0x1002)
    assert b"shares memory" in _clip([a], [b], norm=0x20010)
    assert _clip([a], [b], norm=0x10010) == b""  # a given norm may lie among the inputs
    for kind in (0, 1):
        assert _clip([a], [b], kind=kind, ws=0x100000, size=1 << 20) == b""
        assert b"shares memory" in _clip([a], [b], norm=0x10010, kind=kind, ws=0x100000, size=1 << 20)
        assert b"workspace" in _clip([a], [b], kind=kind)
        assert b"workspace" in _clip([a], [b], kind=kind, ws=0x100010, size=1 << 20)
    assert b"unknown norm" in _clip([a], [b], kind=2)


# ------------------------------------------------------------------ shared memory
X, WG, WU, BG, BU = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000  # of _gated()
NO_CTX = b"null ctx"


def _forward(d=None, h=0x60000, stride=32, ws=0x100000):
    lib = L.load_library()
    assert lib.gs_gated_linear_dev(None, ctypes.byref(d or _gated()), h, stride, ws, 1 << 20,
                                   None) == L.GS_E_INVALID
    return lib.gs_last_error()


def _backward(d=None, dh=(0x60000, 32), dx=(0x70000, 16), dwg=(0x80000, 16), dwu=(0x90000, 16),
              db=(0xa0000, 0xb0000), ws=0x100000):
    lib = L.load_library()
    assert lib.gs_gated_linear_grad_dev(None, ctypes.byref(d or _gated()), *dh, *dx, *dwg, *dwu, *db,
                                        ws, 1 << 40, None) == L.GS_E_INVALID
    return lib.gs_last_error()


@pytest.mark.parametrize("h", [X, X + 4, X + 4 * 16 * 99, WG, WU + 32 * 16 * 4 - 4, BG, BU + 4 * 31,
                               WG - 4 * 32 * 100 + 4])
def test_gated_linear_output_over_an_input(h):
    assert b"shares memory" in _forward(h=h)


@pytest.mark.parametrize("bad", [
    dict(dx=(X, 16)), dict(dx=(0x60000, 32)), dict(dx=(0x60000, 16)), dict(dx=(WG, 16)),
    dict(dx=(BU, 16)), dict(dwg=(0x90000, 16)), dict(dwu=(0x80000 + 4 * 16 * 31, 16)),
    dict(dwg=(WG, 16)), dict(dwu=(WG, 16)), dict(dwu=(0x70000, 16)), dict(dwg=(0x60000 + 64, 16)),
    dict(db=(0xa0000, 0xa0000)), dict(db=(0xa0000, 0xa0000 + 124)), dict(db=(BG, 0xb0000)),
    dict(db=(0xa0000, 0x80000)), dict(db=(0x60000 + 4, None)),
])
def test_gated_linear_grad_outputs_over_others(bad):
    assert b"shares memory" in _backward(**bad)


def test_gated_linear_workspace_over_others():
    """Calls that have a workspace (forward: of more rows than one launch takes)."""
    d = _gated(n=200, dim=144, x_stride=144, gate_stride=144, up_stride=144, w_gate=0x400000,
               w_up=0x500000, x=0x600000)
    assert NO_CTX in _forward(d)
    for ws in (0x400000, 0x500100, 0x600000, 0x60000, 0x60100):
        assert b"shares memory" in _forward(d, ws=ws), hex(ws)
    for ws in (X, WG, BU, 0x60000, 0x70000, 0x80000, 0x90000, 0xa0000, 0xb0000):
        assert b"shares memory" in _backward(ws=ws), hex(ws)


def test_gated_linear_takes_what_shares_no_memory():
    assert NO_CTX in _forward() and NO_CTX in _backward()
    # inputs may share: one weight for both, rows of x and of dh repeated
    d = _gated(w_up=WG, b_up=BG, x_stride=0)
    assert NO_CTX in _forward(d) and NO_CTX in _backward(d, dh=(0x60000, 0))
    # end to end, and columns of one matrix of 64 columns
    assert NO_CTX in _forward(h=X + 4 * 16 * 100) and NO_CTX in _forward(h=X - 4 * 32 * 100)
    d = _gated(n=100, x_stride=64)
    assert NO_CTX in _forward(d, h=X + 64, stride=64) and NO_CTX in _forward(d, h=X + 128, stride=64)
    assert b"shares memory" in _forward(d, h=X + 60, stride=64)
    assert NO_CTX in _backward(d, dh=(X + 64, 64), dx=(X + 192, 64))
    assert b"shares memory" in _backward(d, dh=(X + 64, 64), dx=(X + 180, 64))
    # both weights' gradients in one matrix, row by row in turn
    assert NO_CTX in _backward(dwg=(0x80000, 32), dwu=(0x80000 + 64, 32))
    # without rows nothing is read, and x, dh and dx need not be there
    d = _gated(n=0, x=None, w_gate=None, w_up=None)
    assert NO_CTX in _forward(d, h=None)
    assert NO_CTX in _backward(d, dh=(None, 32), dx=(None, 16))
    assert NO_CTX in _backward(_gated(n=0), dwg=(WG, 16), dwu=(X, 16))
    assert b"shares memory" in _backward(d, dh=(None, 32), dx=(None, 16), dwu=(0x80000, 16))

"""The feature operators' C boundary without a GPU: struct layouts, workspace
sizes, and refusals that need no device."""
import ctypes
import os
import subprocess
import tempfile

import pytest

from gsplat_tt_amd import _lib as L

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")


def test_struct_layouts():
    prog = r"""
#include <stddef.h>
#include <stdio.h>
#include "gsplat_hip.h"
#define P(T, f) printf(#T "." #f " %zu\n", offsetof(T, f));
int main(void) {
  printf("gs_group_norm %zu\ngs_label_loss %zu\n", sizeof(gs_group_norm), sizeof(gs_label_loss));
  P(gs_group_norm, channels) P(gs_group_norm, act) P(gs_group_norm, eps) P(gs_group_norm, weight)
  P(gs_group_norm, bias) P(gs_label_loss, labels) P(gs_label_loss, feat_stride)
  P(gs_label_loss, dim) P(gs_label_loss, labels64) P(gs_label_loss, scale)
  return 0;
}
"""
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        with open(c, "w") as f:
            f.write(prog)
        subprocess.run(["gcc", "-std=c11", "-I", HEADER, c, "-o", exe], check=True)
        lines = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    classes = {"gs_group_norm": L.GsGroupNorm, "gs_label_loss": L.GsLabelLoss}
    for line in lines.strip().splitlines():
        key, val = line.rsplit(" ", 1)
        t, _, f = key.partition(".")
        got = getattr(classes[t], f).offset if f else ctypes.sizeof(classes[t])
        assert got == int(val), key


def test_workspace_sizes():
    lib = L.load_library()
    assert lib.gs_lookup_grad_workspace(0, 10, 4) >= 0
    a, b = (lib.gs_lookup_grad_workspace(n, 4096, 48) for n in (1000, 1_000_000))
    assert 0 < a < b < 1 << 30
    for bad in ((-1, 4, 4), (4, -1, 4), (4, 4, 0), (2 ** 31, 4, 4), (4, 2 ** 30, 4),
                (4, 4, 65537)):
        assert lib.gs_lookup_grad_workspace(*bad) == -1, bad
    assert lib.gs_group_norm_workspace(1, 720 * 1280, 64) > 0
    for bad in ((-1, 4, 4), (4, -1, 4), (4, 4, 0), (2 ** 21, 4, 4), (4, 4, 65537)):
        assert lib.gs_group_norm_workspace(*bad) == -1, bad
    assert lib.gs_label_loss_workspace(0, 5, 4, 0, 1) == 0
    for dtype in (0, 1):
        grad, alone = (lib.gs_label_loss_workspace(10_000, 8192, 48, dtype, k) for k in (1, 0))
        assert grad > alone > 0
    for bad in ((-1, 4, 4, 0, 0), (4, 0, 4, 0, 0), (4, 2 ** 22 + 1, 4, 0, 0), (4, 4, 0, 0, 0),
                (4, 4, 4, 2, 0)):
        assert lib.gs_label_loss_workspace(*bad) == -1, bad


def test_no_context_is_refused():
    lib = L.load_library()
    assert lib.gs_stream(None, None) == L.GS_E_INVALID
    rc = lib.gs_lookup_dev(None, None, 0, 0, 0, None, 0, 0, 1, 1.0, None, 1, 0, None, None)
    assert rc == L.GS_E_INVALID and b"ctx" in lib.gs_last_error()
    n, d = L.GsGroupNorm(), L.GsLabelLoss()
    for rc in (lib.gs_group_norm_dev(None, ctypes.byref(n), None, 0, 0, None, 0, 0, None, None,
                                     None, 0, None),
               lib.gs_label_loss_dev(None, ctypes.byref(d), None, None, None, 0, None, None)):
        assert rc == L.GS_E_INVALID and b"ctx" in lib.gs_last_error()


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="a GPU is present")
def test_field_ops_need_a_gpu():
    from gsplat_tt_amd.field import FieldOps
    with pytest.raises(RuntimeError):
        FieldOps()

"""Tensors that FieldOps does not take, where their memory alone would say something else
than they do. Without a GPU: a library that only counts its calls."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

from gsplat_tt_amd import field


class _Library:
    """Stands for the library: counts the calls that would launch."""

    def __init__(self):
        self.launched = []

    def __getattr__(self, name):
        def call(*args):
            if not name.endswith("_workspace"):
                self.launched.append(name)
            return 0
        return call


class _Context:
    device_index = -1  # what CPU tensors say

    def __init__(self, lib):
        self._L, self.handle = lib, ctypes.c_void_p(0x1000)


class _Stream:
    cuda_stream = 0

    def synchronize(self):
        pass


@pytest.fixture
def ops(monkeypatch):
    real = torch.device
    monkeypatch.setattr(field.torch, "device", lambda *a: real("cpu"))
    monkeypatch.setattr(field.torch.cuda, "current_stream", lambda *a: _Stream())
    return field.FieldOps(_Context(_Library()))


N, DIM, HIDDEN = 6, 4, 3


def _calls(ops):
    """Each operator as a function of its tensors."""
    ids = torch.zeros(N, dtype=torch.int64)
    x, dh, w = torch.ones(N, DIM), torch.ones(N, HIDDEN), torch.ones(HIDDEN, DIM)
    b, stats, image = torch.ones(HIDDEN), torch.ones(1, 2), torch.ones(1, N, DIM)
    c = torch.ones(DIM)
    return {
        "lookup": (lambda table, out: ops.lookup(table, ids, out=out), [x, x.clone()]),
        "lookup_grad": (lambda dout, out: ops.lookup_grad(dout, ids, N, out=out), [x, x.clone()]),
        "group_norm": (lambda x, weight, bias, out: ops.group_norm(x, 2, weight, bias, out=out),
                       [image, c, c, image.clone()]),
        "group_norm_grad": (lambda dy, x, mean, rstd, weight, bias, out: ops.group_norm_grad(
            dy, x, mean, rstd, 2, weight, bias, out=out), [image, image, stats, stats, c, c, image.clone()]),
        "gated_linear": (lambda x, wg, wu, bg, bu, out: ops.gated_linear(x, wg, wu, bg, bu, out=out),
                         [x, w, w, b, b, dh.clone()]),
        "gated_linear_grad": (lambda dh, x, wg, wu, bg, bu, dx, dwg, dwu: ops.gated_linear_grad(
            dh, x, wg, wu, bg, bu, dx=dx, dw_gate=dwg, dw_up=dwu),
            [dh, x, w, w, b, b, x.clone(), w.clone(), w.clone()]),
        "label_loss": (lambda feat, table: ops.label_loss(feat, table, ids), [x, w]),
        "label_loss_grad": (lambda feat, table, rw, df, dt: ops.label_loss_grad(
            feat, table, ids, rw, dfeat=df, dtable=dt), [x, w, torch.ones(N), x.clone(), w.clone()]),
        "grad_norm": (lambda a, b: ops.grad_norm([a, b]), [x, w]),
        "clip_grads in place": (lambda a, b: ops.clip_grads([a, b], 1.0), [x, w]),
        "clip_grads into": (lambda a, o: ops.clip_grads([a], 1.0, out=[o]), [x, x.clone()]),
        "clip_grads by a norm": (lambda a, n: ops.clip_grads([a], 1.0, norm=n),
                                 [x, torch.ones(())]),
    }


NAMES = tuple(_calls(None))


@pytest.mark.parametrize("name", NAMES)
def test_lazily_negated_tensors_are_refused(ops, name):
    """Their memory holds the values with the other sign: each tensor of each call."""
    call, tensors = _calls(ops)[name]
    call(*tensors)
    assert ops._L.launched
    for k, t in enumerate(tensors):
        lazy = torch._neg_view(t)
        assert lazy.is_neg()
        ops._L.launched.clear()
        with pytest.raises(ValueError, match="resolve_neg"):
            call(*tensors[:k], lazy, *tensors[k + 1:])
        assert not ops._L.launched
        call(*tensors[:k], lazy.resolve_neg(), *tensors[k + 1:])


def test_imaginary_parts_of_conjugates_are_refused(ops):
    """Where such tensors come from: rows at a stride of 2 of the complex numbers."""
    z = torch.complex(torch.zeros(4, 1), torch.arange(1.0, 5.0)[:, None])
    t = z.conj().imag
    assert t.shape == (4, 1) and t.stride() == (2, 2) and float(t[0, 0]) == -1.0
    w = torch.ones(HIDDEN, 1)
    for call in (lambda t: ops.grad_norm([t]), lambda t: ops.clip_grads([t], 1.0, out=[torch.ones(4, 1)]),
                 lambda t: ops.gated_linear(t, w, w)):
        with pytest.raises(ValueError, match="resolve_neg"):
            call(t)
        call(z.imag)


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_tensors_are_refused(ops, name):
    """Their tangents would be dropped: each tensor of each call."""
    call, tensors = _calls(ops)[name]
    with fwd.dual_level():
        call(*tensors)  # no dual tensor among them
        for k, t in enumerate(tensors):
            dual = fwd.make_dual(t, torch.ones_like(t))
            ops._L.launched.clear()
            for mode in (torch.enable_grad, torch.no_grad):  # which is for the reverse mode alone
                with mode(), pytest.raises(ValueError, match="forward mode"):
                    call(*tensors[:k], dual, *tensors[k + 1:])
            assert not ops._L.launched
            call(*tensors[:k], dual.detach(), *tensors[k + 1:])
    call(*tensors[:-1], dual)  # its level has ended, and with it the tangent


def test_functions_with_a_rule_for_tangents(ops):
    """A Function's forward gets its inputs with their tangents, which are its jvp's work:
    torch has the forward mode off there, as it has the reverse mode."""
    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(x):
            ops.grad_norm([x])
            return ops.lookup(x, torch.zeros(2, dtype=torch.int64)) * 0

        @staticmethod
        def setup_context(ctx, inputs, output):
            pass

        @staticmethod
        def jvp(ctx, t):
            return torch.full((2, DIM), 5.0)

    x = torch.ones(N, DIM)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        out = Norm.apply(dual)
        assert (fwd.unpack_dual(out).tangent == 5).all()
        assert ops._L.launched == ["gs_grad_norm_dev", "gs_lookup_dev"]
        with pytest.raises(ValueError, match="forward mode"):
            ops.grad_norm([dual])

"""Learned features on splats: table lookups, group norm and the label loss.

`FieldOps` runs the feature operators of the C ABI (include/gsplat_hip.h) on torch
tensors on the GPU, forward and backward:

lookup / lookup_grad          rows of a feature table by id (codebooks of SH
                              coefficients, appearance rows per view), scaled
group_norm / group_norm_grad  group norm with an activation over channels-last
                              feature images
label_loss / label_loss_grad  softmax cross entropy of features against a table
                              of labels, without the scores in memory

The reference has no counterpart. Work is enqueued on torch's current stream of
the context's device and nothing waits; outputs and workspaces come from torch's
allocator on that stream. A tensor made on another stream must be ordered before
the call by the caller, as for any torch operation. The operators are not part of
torch's graph: in grad mode a tensor that requires a gradient is refused, and the
gradients are calls of their own. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib as L

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_ID_TYPES = (torch.int32, torch.int64)
_PARAM_TYPES = (torch.float32,)
_ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
FLAG_ID_RANGE = 1


def _rows(t, name, dim=None):
    """Pointer, rows, row stride of a (rows, dim) tensor with contiguous rows."""
    if t.dim() != 2:
        raise ValueError(f"{name} must have 2 dimensions, not {t.dim()}")
    rows, cols = t.shape
    if dim is not None and cols != dim:
        raise ValueError(f"{name} must have {dim} columns, not {cols}")
    if t.is_contiguous():
        return t.data_ptr(), rows, cols
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the values of a row must be contiguous")
    return t.data_ptr(), rows, t.stride(0)


def _written(out):
    """Counts a given output as changed in place, for graphs that have saved it."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


class FieldOps:
    """The feature operators on one GPU: `ctx` (a Context) or a new one on `device`.

    Ids and labels are int32 or int64 tensors; those below 0 are masked, and one at
    or past the table's rows is treated as masked and remembered: check() raises
    ValueError for it (and waits for the GPU; nothing else here does)."""

    def __init__(self, ctx: "L.Context | None" = None, device: int = 0):
        self.ctx = ctx if ctx is not None else L.Context(device)
        self._L = self.ctx._L
        self.device = torch.device("cuda", self.ctx.device_index)
        self._index = self.ctx.device_index
        self._flags = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._flags_ptr = self._flags.data_ptr()
        torch.cuda.current_stream(self.device).synchronize()
        self._sizes = {}

    # ---- checks
    def _own(self, t, name, dtypes=_DTYPES):
        if isinstance(t, torch.Tensor) and t.get_device() == self._index and t.dtype in dtypes:
            if t.requires_grad and torch.is_grad_enabled():
                raise ValueError(f"{name} requires a gradient, which these operators do not "
                                 "record: detach() it or call under torch.no_grad()")
            return t
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, not on {self.device}")
        raise TypeError(f"{name} has the type {t.dtype}")

    def _ids(self, t, name, n=None):
        self._own(t, name, _ID_TYPES)
        if t.dim() != 1 or (n is not None and t.shape[0] != n):
            raise ValueError(f"{name} must be one-dimensional" +
                             (f" with {n} values" if n is not None else ""))
        return t.contiguous()

    def _param(self, t, name, n):
        if t is None:
            return None
        self._own(t, name, _PARAM_TYPES)
        if t.dim() != 1 or t.shape[0] != n:
            raise ValueError(f"{name} must be one-dimensional with {n} values")
        return t.contiguous()

    def _out(self, out, shape, dtype, name):
        if out is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        self._own(out, name)
        if out.shape != torch.Size(shape):
            raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(out.shape)}")
        _written(out)
        return out

    def _workspace(self, name, *sizes):
        key = (name, *sizes)
        size = self._sizes.get(key)
        if size is None:
            size = getattr(self._L, name)(*sizes)
            if size < 0:
                raise L.GsError(f"{name[3:-10]}: sizes past the limits: {sizes}")
            if len(self._sizes) > 4096:
                self._sizes.clear()
            self._sizes[key] = size
        return torch.empty(size, dtype=torch.uint8, device=self.device), size

    def _stream(self):
        return torch.cuda.current_stream(self._index).cuda_stream

    def check(self):
        """Waits for the GPU, whatever streams the calls were made on, and raises
        ValueError when one since the last check was given an id or label at or past
        its table's rows."""
        torch.cuda.synchronize(self.device)
        flags = int(self._flags.item())
        if flags:
            self._flags.zero_()
            torch.cuda.current_stream(self.device).synchronize()
        if flags & FLAG_ID_RANGE:
            raise ValueError("an id or a label is at or past the table's rows")

    # ---- lookup
    def lookup(self, table, ids, scale=1.0, out=None, dtype=None):
        """scale * table[ids], zeros for masked ids: (n, dim) of the table's type, or
        of `dtype` or `out`'s."""
        self._own(table, "table")
        p, rows, stride = _rows(table, "table")
        ids = self._ids(ids, "ids")
        n, dim = ids.shape[0], table.shape[1]
        out = self._out(out, (n, dim), dtype or table.dtype, "out")
        po, _, so = _rows(out, "out")
        L._check(self._L.gs_lookup_dev(
            self.ctx.handle, p, rows, stride, _DTYPES[table.dtype], ids.data_ptr(),
            int(ids.dtype == torch.int64), n, dim, float(scale), po, so, _DTYPES[out.dtype],
            self._flags_ptr, self._stream()))
        return out

    def lookup_grad(self, dout, ids, rows, scale=1.0, out=None, accumulate=False, dtype=None):
        """The gradient of lookup() for its table of `rows` rows: scale times the sum
        of dout's rows per id, zeros for rows no id names; with `accumulate` added to
        what `out` holds."""
        self._own(dout, "dout")
        p, n, stride = _rows(dout, "dout")
        ids = self._ids(ids, "ids", n)
        dim = dout.shape[1]
        if accumulate and out is None:
            raise ValueError("accumulate needs out")
        out = self._out(out, (int(rows), dim), dtype or dout.dtype, "out")
        po, _, so = _rows(out, "out")
        ws, size = self._workspace("gs_lookup_grad_workspace", n, int(rows), dim)
        L._check(self._L.gs_lookup_grad_dev(
            self.ctx.handle, p, stride, _DTYPES[dout.dtype], ids.data_ptr(),
            int(ids.dtype == torch.int64), n, dim, float(scale), int(bool(accumulate)), po,
            int(rows), so, _DTYPES[out.dtype], ws.data_ptr(), size, self._flags_ptr,
            self._stream()))
        return out

    # ---- group norm
    def _image(self, t, name, shape=None, dtype=None):
        """Pointer, image stride, pixel stride of a (batch, ..., channels) tensor whose
        pixels lie at one distance."""
        self._own(t, name)
        if t.dim() < 2 or (shape is not None and t.shape != shape):
            raise ValueError(f"{name} must be (batch, pixels..., channels)" +
                             (f" = {tuple(shape)}" if shape is not None else ""))
        if dtype is not None and t.dtype is not dtype:
            raise TypeError(f"{name} must have the type {dtype}")
        if t.is_contiguous():
            return t.data_ptr(), t.stride(0), t.shape[-1]
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name}: the channels of a pixel must be contiguous")
        pixel, step = None, None
        for k in range(t.dim() - 2, 0, -1):
            if t.shape[k] == 1:
                continue
            if pixel is None:
                pixel, step = t.stride(k), t.stride(k) * t.shape[k]
            elif t.stride(k) != step:
                raise ValueError(f"{name}: the pixels of an image must lie at one distance "
                                 "(a crop needs .contiguous())")
            else:
                step *= t.shape[k]
        return t.data_ptr(), t.stride(0), t.shape[-1] if pixel is None else pixel

    def _norm(self, x, groups, weight, bias, act, eps):
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}")
        shape = x.shape
        c = shape[-1]
        weight, bias = self._param(weight, "weight", c), self._param(bias, "bias", c)
        d = L.GsGroupNorm(shape[0], math.prod(shape[1:-1]), c, int(groups), _ACTS[act], _DTYPES[x.dtype],
                          float(eps), 0, None if weight is None else weight.data_ptr(),
                          None if bias is None else bias.data_ptr())
        return d, (weight, bias)

    def group_norm(self, x, groups, weight=None, bias=None, act="none", eps=1e-5, out=None):
        """act((x - mean) rstd weight + bias) over (batch, ..., channels) images, with
        the (batch, groups) statistics: (y, mean, rstd). weight and bias (channels)
        are fp32."""
        px, bx, sx = self._image(x, "x")
        d, keep = self._norm(x, groups, weight, bias, act, eps)
        given = out
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        py, by, sy = self._image(out, "out", x.shape, x.dtype)
        if given is not None:
            _written(out)
        stats = torch.zeros if d.pixels == 0 else torch.empty
        mean, rstd = stats((2, d.batch, d.groups), dtype=torch.float32, device=self.device)
        ws, size = self._workspace("gs_group_norm_workspace", d.batch, d.pixels, d.channels)
        L._check(self._L.gs_group_norm_dev(
            self.ctx.handle, ctypes.byref(d), px, bx, sx, py, by, sy, mean.data_ptr(),
            rstd.data_ptr(), ws.data_ptr(), size, self._stream()))
        del keep
        return out, mean, rstd

    def group_norm_grad(self, dy, x, mean, rstd, groups, weight=None, bias=None, act="none",
                        eps=1e-5, out=None):
        """(dx, dweight, dbias) of group_norm() from its output's gradient, its input
        and its statistics; the parameters' gradients are fp32, summed over the batch."""
        px, bx, sx = self._image(x, "x")
        pd, bd, sd = self._image(dy, "dy", x.shape, x.dtype)
        d, keep = self._norm(x, groups, weight, bias, act, eps)
        given = out
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        po, bo, so = self._image(out, "out", x.shape, x.dtype)
        if given is not None:
            _written(out)
        stats = (d.batch, d.groups)
        for t, name in ((mean, "mean"), (rstd, "rstd")):
            self._own(t, name, _PARAM_TYPES)
            if t.shape != stats or not t.is_contiguous():
                raise ValueError(f"{name} must be group_norm()'s: contiguous {stats}")
        dweight, dbias = torch.empty((2, d.channels), dtype=torch.float32, device=self.device)
        ws, size = self._workspace("gs_group_norm_workspace", d.batch, d.pixels, d.channels)
        L._check(self._L.gs_group_norm_grad_dev(
            self.ctx.handle, ctypes.byref(d), pd, bd, sd, px, bx, sx, mean.data_ptr(),
            rstd.data_ptr(), po, bo, so, dweight.data_ptr(), dbias.data_ptr(),
            ws.data_ptr(), size, self._stream()))
        del keep
        return out, dweight, dbias

    # ---- label loss
    def _loss(self, feat, table, labels, scale):
        self._own(feat, "feat")
        self._own(table, "table")
        if table.dtype != feat.dtype:
            raise TypeError(f"feat is {feat.dtype}, table {table.dtype}")
        pf, n, sf = _rows(feat, "feat")
        pt, rows, stt = _rows(table, "table", feat.shape[1])
        labels = self._ids(labels, "labels", n)
        return L.GsLabelLoss(pf, pt, labels.data_ptr(), n, rows, sf, stt, feat.shape[1],
                             _DTYPES[feat.dtype], int(labels.dtype == torch.int64),
                             float(scale)), labels

    def label_loss(self, feat, table, labels, scale=1.0):
        """(loss, lse), fp32 (n): cross entropy of the scores scale * feat @ table.T
        against `labels`, and the scores' log sum exp; 0 and 0 for masked labels."""
        d, keep = self._loss(feat, table, labels, scale)
        loss, lse = torch.empty((2, d.n), dtype=torch.float32, device=self.device)
        ws, size = self._workspace("gs_label_loss_workspace", d.n, d.rows, d.dim, d.dtype, 0)
        L._check(self._L.gs_label_loss_dev(
            self.ctx.handle, ctypes.byref(d), loss.data_ptr(), lse.data_ptr(), ws.data_ptr(),
            size, self._flags_ptr, self._stream()))
        del keep
        return loss, lse

    def label_loss_grad(self, feat, table, labels, row_weight=None, scale=1.0, dfeat=None,
                        dtable=None):
        """(loss, lse, dfeat, dtable): label_loss() and the gradients of
        sum(row_weight * loss) in the inputs' type; row_weight (n) fp32, None: ones."""
        d, keep = self._loss(feat, table, labels, scale)
        row_weight = self._param(row_weight, "row_weight", d.n)
        loss, lse = torch.empty((2, d.n), dtype=torch.float32, device=self.device)
        dfeat = self._out(dfeat, feat.shape, feat.dtype, "dfeat")
        dtable = self._out(dtable, table.shape, table.dtype, "dtable")
        if dfeat.dtype != feat.dtype or dtable.dtype != feat.dtype:
            raise TypeError(f"dfeat and dtable must have the type {feat.dtype}")
        pf, _, sf = _rows(dfeat, "dfeat")
        pt, _, stt = _rows(dtable, "dtable")
        ws, size = self._workspace("gs_label_loss_workspace", d.n, d.rows, d.dim, d.dtype, 1)
        L._check(self._L.gs_label_loss_grad_dev(
            self.ctx.handle, ctypes.byref(d),
            None if row_weight is None else row_weight.data_ptr(), loss.data_ptr(),
            lse.data_ptr(), pf, sf, pt, stt, ws.data_ptr(), size, self._flags_ptr,
            self._stream()))
        del keep
        return loss, lse, dfeat, dtable

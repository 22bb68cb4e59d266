"""Learned features on splats: table lookups, group norm, gated projections, the label
loss, and the norm and clipping of gradients.

`FieldOps` runs the feature operators of the C ABI (include/gsplat_hip.h) on torch
tensors on the GPU, forward and backward:

lookup / lookup_grad          rows of a feature table by id (codebooks of SH
                              coefficients, appearance rows per view), scaled
group_norm / group_norm_grad  group norm with an activation over channels-last
                              feature images
gated_linear / gated_linear_grad  the gated projections of a feed-forward block
label_loss / label_loss_grad  softmax cross entropy of features against a table
                              of labels, without the scores in memory
grad_norm / clip_grads        the global norm of many tensors, and their scaling
                              down to a limit

The reference has no counterpart. Work is enqueued on torch's current stream of
the context's device and nothing waits; outputs and workspaces come from torch's
allocator on that stream. A tensor made on another stream must be ordered before
the call by the caller, as for any torch operation. The operators are not part of
torch's graph: in grad mode a tensor that requires a gradient is refused, and where the
forward mode is on one with a tangent; the gradients are calls of their own.
Tensors are taken by their memory: one with torch's lazy negation (an imaginary part
of a conjugate) is refused, its resolve_neg() is not. Outputs that are given share no
memory with another tensor of the call, but for group_norm's `out` = x,
group_norm_grad's = x or dy, and clip_grads() in place; the gated projections and
clip_grads() refuse such outputs. There is no CPU fallback.
"""
from __future__ import annotations

import array
import ctypes
import math
import operator

import torch
from torch.autograd import forward_ad

from . import _lib as L

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_ID_TYPES = (torch.int32, torch.int64)
_PARAM_TYPES = (torch.float32,)
_ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
_NORMS, _NORM_GIVEN = {"l2": 0, "max": 1}, -1
FLAG_ID_RANGE = 1
_PLAIN = {torch.Tensor, torch.nn.Parameter}
_get_dtype = torch.Tensor.dtype.__get__
_get_device = torch.Tensor.get_device
_get_requires_grad = torch.Tensor.requires_grad.__get__


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


def _collapse(t):
    """Rows, columns and row stride that visit a tensor's values in order, or None where
    one stride between rows is not enough."""
    rows, cols, stride, inner = 1, 1, 0, True
    step = 1  # of the next dimension if it goes on with the run
    for size, st in zip(reversed(t.shape), reversed(t.stride())):
        if size == 1:
            continue
        if inner and st == step:
            cols *= size
            step *= size
        elif inner:
            inner, rows, stride = False, size, st
            step = st * size
        elif st == step:
            rows *= size
            step *= size
        else:
            return None
    return rows, cols, stride if rows > 1 else cols


def _in_forward_mode():
    """Whether there can be tensors with tangents: unpack_dual() of each takes longer than
    all other checks."""
    return forward_ad._current_level >= 0


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
            if _in_forward_mode() and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has a tangent (torch's forward mode), which these "
                                 "operators do not carry on: detach() it")
            if t.is_neg():  # its memory holds the values with the other sign
                raise ValueError(f"{name} is negated when it is read: give its resolve_neg()")
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

    # ---- gated projections
    def _gated(self, x, w_gate, w_up, b_gate, b_up, act):
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}")
        self._own(x, "x")
        px, n, sx = _rows(x, "x")
        dim = x.shape[1]
        weights = []
        for w, name in ((w_gate, "w_gate"), (w_up, "w_up")):
            self._own(w, name)
            if w.dtype != x.dtype:
                raise TypeError(f"x is {x.dtype}, {name} {w.dtype}")
            weights.append(_rows(w, name, dim))
        (pg, hidden, sg), (pu, rows, su) = weights
        if rows != hidden:
            raise ValueError(f"w_gate has {hidden} rows, w_up {rows}")
        b_gate = self._param(b_gate, "b_gate", hidden)
        b_up = self._param(b_up, "b_up", hidden)
        return L.GsGatedLinear(px, pg, pu, None if b_gate is None else b_gate.data_ptr(),
                               None if b_up is None else b_up.data_ptr(), n, hidden, sx, sg, su,
                               dim, _DTYPES[x.dtype], _ACTS[act], 0), (b_gate, b_up)

    def _gated_workspace(self, d, grad):
        # -1 for what the call itself refuses
        size = max(self._L.gs_gated_linear_workspace(ctypes.byref(d), grad), 0)
        if size == 0:
            return None, None, 0
        ws = torch.empty(size, dtype=torch.uint8, device=self.device)
        return ws, ws.data_ptr(), size

    def gated_linear(self, x, w_gate, w_up, b_gate=None, b_up=None, act="silu", out=None):
        """act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up): (n, hidden) of x's type, from
        x (n, dim) and weights (hidden, dim) of one type; the biases (hidden) are fp32."""
        d, keep = self._gated(x, w_gate, w_up, b_gate, b_up, act)
        out = self._out(out, (d.n, d.hidden), x.dtype, "out")
        if out.dtype != x.dtype:
            raise TypeError(f"out must have the type {x.dtype}")
        po, _, so = _rows(out, "out")
        ws, at, size = self._gated_workspace(d, 0)
        L._check(self._L.gs_gated_linear_dev(self.ctx.handle, ctypes.byref(d), po, so, at,
                                             size, self._stream()))
        del keep, ws
        return out

    def gated_linear_grad(self, dh, x, w_gate, w_up, b_gate=None, b_up=None, act="silu",
                          dx=None, dw_gate=None, dw_up=None):
        """(dx, dw_gate, dw_up, db_gate, db_up) of gated_linear() from its output's
        gradient and its inputs: in the inputs' type, the biases' in fp32 (None for a bias
        that is None), the weights' and biases' summed over the rows."""
        d, keep = self._gated(x, w_gate, w_up, b_gate, b_up, act)
        self._own(dh, "dh")
        if dh.dtype != x.dtype:
            raise TypeError(f"x is {x.dtype}, dh {dh.dtype}")
        ph, n, sh = _rows(dh, "dh", d.hidden)
        if n != d.n:
            raise ValueError(f"dh must have {d.n} rows, not {n}")
        dx = self._out(dx, x.shape, x.dtype, "dx")
        dw_gate = self._out(dw_gate, w_gate.shape, x.dtype, "dw_gate")
        dw_up = self._out(dw_up, w_up.shape, x.dtype, "dw_up")
        if not dx.dtype == dw_gate.dtype == dw_up.dtype == x.dtype:
            raise TypeError(f"dx, dw_gate and dw_up must have the type {x.dtype}")
        db_gate, db_up = (None if b is None else torch.empty(d.hidden, dtype=torch.float32,
                                                             device=self.device)
                          for b in (b_gate, b_up))
        px, _, sx = _rows(dx, "dx")
        pg, _, sg = _rows(dw_gate, "dw_gate")
        pu, _, su = _rows(dw_up, "dw_up")
        ws, at, size = self._gated_workspace(d, 1)
        L._check(self._L.gs_gated_linear_grad_dev(
            self.ctx.handle, ctypes.byref(d), ph, sh, px, sx, pg, sg, pu, su,
            None if db_gate is None else db_gate.data_ptr(),
            None if db_up is None else db_up.data_ptr(), at, size, self._stream()))
        del keep, ws
        return dx, dw_gate, dw_up, db_gate, db_up

    # ---- gradients of many tensors
    def _tensors(self, tensors, name, like=None):
        """The list as an array of gs_tensor, values in the order in which the tensors
        (or their counterparts in `like`) lie in memory."""
        # a list at a time: tensor by tensor 100 of them took 75 us, so 40
        count = len(tensors)
        plain = set(map(type, tensors)) <= _PLAIN
        if plain:
            types = set(map(_get_dtype, tensors))
            plain = types <= _DTYPES.keys() and set(map(_get_device, tensors)) <= {self._index} and \
                not (torch.is_grad_enabled() and any(map(_get_requires_grad, tensors))) and \
                not any(map(torch.Tensor.is_neg, tensors)) and not _in_forward_mode()
        if not plain:
            for t in tensors:
                self._own(t, name)
            types = set(map(_get_dtype, tensors))
        sizes = array.array("q", map(torch.Tensor.numel, tensors))
        flat = array.array("q", bytes(40 * count))
        flat[0::5] = array.array("q", map(torch.Tensor.data_ptr, tensors))
        flat[1::5] = array.array("q", [1]) * count
        flat[2::5] = flat[3::5] = sizes
        if len(types) == 1:
            flat[4::5] = array.array("q", [_DTYPES[types.pop()]]) * count
        else:
            flat[4::5] = array.array("q", map(_DTYPES.get, map(_get_dtype, tensors)))
        if like is None:
            like = tensors
        if not (all(map(torch.Tensor.is_contiguous, tensors)) and
                (like is tensors or all(map(torch.Tensor.is_contiguous, like)))):
            for k, (t, lead) in enumerate(zip(tensors, like)):
                if t.numel() == 0 or (t.is_contiguous() and lead.is_contiguous()):
                    continue
                if _collapse(lead) is None:  # the order of memory, not that of the dimensions
                    t = t.permute(sorted(range(t.dim()), key=lead.stride, reverse=True))
                rows = _collapse(t)
                if rows is None:
                    raise ValueError(f"{name}[{k}]: the values must lie in rows at one distance" +
                                     (" in grads' order" if like is not tensors else ""))
                flat[5 * k + 1:5 * k + 4] = array.array("q", rows)
        return flat

    def _norm_room(self, flat, count, kind):
        """The norm's number, the norm, the workspace and its size."""
        if kind not in _NORMS:
            raise ValueError(f"kind must be one of {sorted(_NORMS)}")
        # -1 for what the call itself refuses
        size = max(self._L.gs_grad_norm_workspace(flat.buffer_info()[0], count), 0)
        return (_NORMS[kind], torch.empty((), dtype=torch.float32, device=self.device),
                torch.empty(size, dtype=torch.uint8, device=self.device), size)

    def grad_norm(self, grads, kind="l2"):
        """The global norm of a list of fp32 and bf16 tensors, an fp32 scalar on the GPU:
        "l2", the root of the sum of all squares, or "max", the largest size of a value; 0
        for no values, NaN if any value is."""
        grads = list(grads)
        flat = self._tensors(grads, "grads")
        number, norm, ws, size = self._norm_room(flat, len(grads), kind)
        L._check(self._L.gs_grad_norm_dev(self.ctx.handle, flat.buffer_info()[0], len(grads),
                                          number, norm.data_ptr(), ws.data_ptr(), size,
                                          self._stream()))
        return norm

    def clip_grads(self, grads, max_norm, kind="l2", out=None, norm=None):
        """Scales the tensors by min(1, max_norm / (norm + 1e-6)), in place or into the
        tensors `out` (of the same shapes, fp32 or bf16; each in its counterpart's order of
        memory, as one run of values or in the same rows), and returns their global norm from
        before. `norm` (an fp32 scalar on the GPU) is taken instead of it if given, as where it
        is summed over processes. In place nothing is written where the norm is within the
        limit."""
        grads = list(grads)
        flat = self._tensors(grads, "grads")
        to = flat
        if out is None:
            out = grads
        else:
            out = list(out)
            if len(out) != len(grads):
                raise ValueError(f"out has {len(out)} tensors, grads {len(grads)}")
            if any(map(operator.is_not, out, grads)):
                for t in out:
                    if not isinstance(t, torch.Tensor):
                        raise TypeError("out must be torch tensors")
                shapes = list(map(torch.Tensor.size, grads))
                if list(map(torch.Tensor.size, out)) != shapes:
                    k, o = next((k, o) for k, (o, s) in enumerate(zip(out, shapes)) if o.shape != s)
                    raise ValueError(f"out[{k}] must be {tuple(shapes[k])}, not {tuple(o.shape)}")
                to = self._tensors(out, "out", grads)
        max_norm = float(max_norm)
        if not max_norm >= 0.0:
            raise ValueError("max_norm must be a number, at least 0")
        if norm is None:
            number, norm, ws, size = self._norm_room(flat, len(grads), kind)
            ws = ws.data_ptr()
        else:
            number, ws, size = _NORM_GIVEN, None, 0
            self._own(norm, "norm", _PARAM_TYPES)
            if norm.numel() != 1:
                raise ValueError("norm must be one value")
        try:
            torch.autograd.graph.increment_version(out)
        except RuntimeError:  # inference tensors, which have no version, among them
            for t in out:
                _written(t)
        L._check(self._L.gs_grad_clip_dev(self.ctx.handle, flat.buffer_info()[0],
                                          to.buffer_info()[0], len(grads), number,
                                          norm.data_ptr(), max_norm, ws, size, self._stream()))
        return norm

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

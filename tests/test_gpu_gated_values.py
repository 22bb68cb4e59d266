"""Gated projections where single values are not finite or very small, rows in several
pieces, and what lies around the outputs.

One value at a time is infinite or NaN, so that some rows, units or columns of the results
are finite and others are not. Where the formula in 64 bits says NaN, +inf or -inf the
results say the same; everywhere else they are within the tolerances of test_gpu_gated.py
for the inputs before that value was put in: a finite result is a sum of the same products,
or of some of them."""
import ctypes
import functools
import math

import pytest
import torch

from tests.test_gpu_gated import BF16, D64, F32, NAMES, _cuda, _inputs, _reference, ops  # noqa: F401

pytestmark = pytest.mark.gpu

# the ways of field_gated.hip; rows, units and columns that end inside a tile
WAYS = {"few": (37, 40, 24), "few of long rows": (37, 200, 48), "short": (300, 72, 130),
        "tiles": (200, 300, 40), "wide": (4900, 136, 3000)}


def _within(got, ref, what):
    want, tol = ref
    off = (got.to(D64) - want).abs()
    assert got.shape == want.shape and bool((off <= tol).all()), (what, float((off / tol).max()))


# ------------------------------------------------------------------ not finite
# what is put in where, in values of which sign and with which activation; the results that
# are partly finite, and those that are not finite anywhere (the others are everywhere)
INF, NAN = math.inf, math.nan
BAD = {"x inf": ("x", INF, True, "relu", ("h", "dx"), ("dw_gate", "dw_up", "db_gate", "db_up")),
       "x inf, silu": ("x", INF, False, "silu", ("h", "dx"), ("dw_gate", "dw_up", "db_gate", "db_up")),
       "x inf, gelu": ("x", INF, False, "gelu", ("h", "dx"), ("dw_gate", "dw_up", "db_gate", "db_up")),
       "x inf, none": ("x", INF, False, "none", ("h", "dx"), ("dw_gate", "dw_up", "db_gate", "db_up")),
       "x -inf": ("x", -INF, True, "relu", ("h", "dx", "dw_up"), ("dw_gate", "db_gate")),
       "x nan": ("x", NAN, True, "relu", ("h", "dx"), ("dw_gate", "dw_up", "db_gate", "db_up")),
       "w_up -inf": ("wu", -INF, True, "relu", ("h", "dw_gate", "db_gate"), ("dx",)),
       "w_gate inf": ("wg", INF, True, "relu", ("h", "dw_up", "db_up"), ("dx",)),
       "w_gate nan": ("wg", NAN, True, "relu", ("h", "dw_up", "db_up"), ("dx",)),
       "b_gate inf": ("bg", INF, True, "relu", ("h", "dw_up", "db_up"), ("dx",)),
       "b_gate -inf": ("bg", -INF, False, "relu", (), ()),
       "b_up inf": ("bu", INF, True, "relu", ("h", "dw_gate", "db_gate"), ("dx",)),
       "dh inf": ("dh", INF, False, "silu", ("dx", "dw_gate", "dw_up", "db_gate", "db_up"), ()),
       "dh nan": ("dh", NAN, False, "silu", ("dx", "dw_gate", "dw_up", "db_gate", "db_up"), ())}


@functools.lru_cache(maxsize=4)
def _before(way, dtype, positive, act):
    x, wg, wu, bg, bu, dh = _inputs(*WAYS[way], dtype, seed=60)
    if positive:  # every product above 0: no difference of infinities
        x, wg, wu = (t.abs() + 0.1 for t in (x, wg, wu))
        bg, bu, dh = bg.abs(), bu.abs(), dh.abs() + 0.01
    ins = {"x": x, "wg": wg, "wu": wu, "bg": bg, "bu": bu, "dh": dh}
    return ins, {k: t for k, (_, t) in _reference(*ins.values(), act, dtype).items()}


def _plain(x, wg, wu, bg, bu, dh, act):
    x, wg, wu, bg, bu, dh = (t.to(D64) for t in (x, wg, wu, bg, bu, dh))
    gate, up = x @ wg.T + bg, x @ wu.T + bu
    if act == "relu":
        a, slope = torch.relu(gate), (gate > 0).to(D64)
    elif act == "silu":
        s = torch.sigmoid(gate)
        a, slope = gate * s, s * (1 + gate * (1 - s))
    elif act == "gelu":
        phi = 0.5 * torch.erfc(-gate / math.sqrt(2))
        a, slope = gate * phi, phi + gate * torch.exp(-0.5 * gate * gate) / math.sqrt(2 * math.pi)
    else:
        a, slope = gate, torch.ones_like(gate)
    dg, du = dh * up * slope, dh * a
    return {"h": a * up, "dx": dg @ wg + du @ wu, "dw_gate": dg.T @ x, "dw_up": du.T @ x,
            "db_gate": dg.sum(0), "db_up": du.sum(0)}


def _bad_case(way, dtype, bad, spot):
    name, value, positive, act, partly, nowhere = BAD[bad]
    ins, tols = _before(way, dtype, positive, act)
    n, dim, hidden = WAYS[way]
    i, c, u = (n - 1, dim - 1, hidden - 1) if spot == "last" else (n // 2, dim // 3, hidden // 2)
    ins = {**ins, name: ins[name].clone()}
    ins[name][{"x": (i, c), "wg": (u, c), "wu": (u, c), "bg": u, "bu": u, "dh": (i, u)}[name]] = value
    want = _plain(*ins.values(), act)
    for k, t in want.items():
        finite = t.isfinite()
        assert bool(finite.any()) == (k not in nowhere), (k, "somewhere finite")
        assert bool(finite.all()) == (k not in partly + nowhere), (k, "everywhere finite")
    return ins, want, tols, act


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("way,spot", [(w, s) for w in WAYS for s in ("last", "inner")
                                      if (w, s) != ("wide", "inner")])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_value_that_is_not_finite(ops, dtype, way, spot, bad):  # noqa: F811
    ins, want, tols, act = _bad_case(way, dtype, bad, spot)
    *args, dh = _cuda(ins.values())
    got = {"h": ops.gated_linear(*args, act=act),
           **dict(zip(NAMES, ops.gated_linear_grad(dh, *args, act=act)))}
    for k, w in want.items():
        g = got[k].cpu().to(D64)
        assert torch.equal(g.isnan(), w.isnan()), (k, "NaN")
        assert torch.equal(g == INF, w == INF) and torch.equal(g == -INF, w == -INF), (k, "inf")
        on = w.isfinite()
        _within(g[on], (w[on], tols[k][on]), k)


# ------------------------------------------------------------------ small values
@pytest.mark.parametrize("n,dim,hidden", [WAYS[w] for w in WAYS if w != "wide"])
def test_small_fp32_values(ops, n, dim, hidden):  # noqa: F811
    """Bits of an operand below 2^-133 are left out, no more: in x against large weights, and
    in the gradients of gate and up."""
    least = 2.0 ** -133
    g = torch.Generator().manual_seed(61)

    def randn(*s):
        return torch.randn(*s, generator=g)

    dh = torch.zeros(n, hidden)
    for e in (112, 120, 127, 131, 140):
        x, wg, wu = randn(n, dim) * 2.0 ** -60 * 2.0 ** (60 - e), randn(hidden, dim) * 2.0 ** 105, \
            torch.zeros(hidden, dim)
        x[:, 0], wg[:, 0], wu[:, 0] = 1.0, 0.0, 1.0  # up is 1
        want, tol = _reference(x, wg, wu, None, None, dh, "none", F32)["h"]
        out = wg.abs().to(D64).sum(1) * least
        _within(ops.gated_linear(*_cuda((x, wg, wu)), act="none").cpu(), (want, tol + out), e)
    x, wg, wu, bg, bu, dh = _inputs(n, dim, hidden, F32, seed=62)
    dh = dh * 2.0 ** -60 * 2.0 ** -58
    ref = _reference(x, wg, wu, bg, bu, dh, "none", F32)
    rows = (wg.abs() + wu.abs()).to(D64).sum(0) * least
    cols = x.abs().to(D64).sum(0) * least
    for name, t in zip(NAMES, ops.gated_linear_grad(*_cuda((dh, x, wg, wu, bg, bu)), act="none")):
        want, tol = ref[name]
        # sums of fp32 that round below its normal range: 2^-150 each
        tol = tol + (rows if name == "dx" else cols if name.startswith("dw") else 0) + \
            2.0 ** -150 * (n + 2 * hidden)
        _within(t.cpu(), (want, tol), name)


def test_infinite_against_small_fp32_values(ops):  # noqa: F811
    """A value below 2^-133 counts as 0 there, too."""
    x = torch.tensor([[INF, 1.0]], device="cuda").expand(3, 2)
    for small, h in ((1e-30, INF), (1e-38, INF), (2.0 ** -133, INF), (-2.0 ** -133, -INF),
                     (2.0 ** -134, NAN), (0.0, NAN)):
        wg = torch.tensor([[small, 0.0]], device="cuda")
        wu = torch.tensor([[1.0, 0.0]], device="cuda")
        got = ops.gated_linear(x, wg, wu, act="none").cpu()
        want = torch.full((3, 1), h)
        assert torch.equal(got.isnan(), want.isnan()), small
        assert torch.equal(got[~want.isnan()], want[~want.isnan()]), small


# ------------------------------------------------------------------ around the outputs
GUARD, KEPT = 256, 7.0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,dim,hidden", [*WAYS.values(), (1, 1, 1), (3, 5, 7), (65, 129, 33),
                                          (16_500, 72, 130), (20_001, 33, 31), (20_001, 128, 65)])
def test_what_lies_around_the_outputs_stays(ops, dtype, n, dim, hidden):  # noqa: F811
    """A tile's rows before and after each output, and columns beside it."""
    x, wg, wu, bg, bu, dh = args = _cuda(_inputs(n, dim, hidden, dtype, seed=63))
    want = (ops.gated_linear(*args[:5]), *ops.gated_linear_grad(dh, *args[:5]))

    def room(rows, cols):
        r = torch.full((GUARD + rows + GUARD, cols + 11), KEPT, dtype=dtype, device="cuda")
        return r, r[GUARD:GUARD + rows, 3:3 + cols]

    rooms = [room(*t.shape) for t in want[:4]]
    biases = torch.full((2, GUARD + hidden + GUARD), KEPT, device="cuda")
    db = [b[GUARD:GUARD + hidden] for b in biases]
    h, dx, dwg, dwu = (v for _, v in rooms)
    ops.gated_linear(*args[:5], out=h)
    d, keep = ops._gated(x, wg, wu, bg, bu, "silu")
    ws, at, size = ops._gated_workspace(d, 1)
    assert ops._L.gs_gated_linear_grad_dev(
        ops.ctx.handle, ctypes.byref(d), dh.data_ptr(), hidden, dx.data_ptr(), dx.stride(0),
        dwg.data_ptr(), dwg.stride(0), dwu.data_ptr(), dwu.stride(0), db[0].data_ptr(),
        db[1].data_ptr(), at, size, ops._stream()) == 0
    for got, w in zip((h, dx, dwg, dwu, *db), want):
        assert torch.equal(got, w)
        got.fill_(KEPT)
    assert all(bool((r == KEPT).all()) for r, _ in rooms) and bool((biases == KEPT).all())
    del keep, ws


# ------------------------------------------------------------------ pieces
def _on_gpu(n, dim, hidden, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    x = randn(n, dim).to(dtype)
    wg, wu = ((randn(hidden, dim) * 1.5 / math.sqrt(dim)).to(dtype) for _ in range(2))
    return x, wg, wu, 0.3 * randn(hidden), 0.3 * randn(hidden), (randn(n, hidden) * 0.1).to(dtype)


def _pieces(ops, ins, act, dtype):  # noqa: F811
    ref = _reference(*ins, act, dtype)
    *args, dh = ins
    _within(ops.gated_linear(*args, act=act), ref["h"], "h")
    for name, t in zip(NAMES, ops.gated_linear_grad(dh, *args, act=act)):
        _within(t, ref[name], name)
    return ref


@pytest.mark.parametrize("n,dtype", [(3001, F32), (8300, BF16)])
def test_tiles_in_pieces(ops, n, dtype):  # noqa: F811
    """The longest rows: the workspace takes 2688 of fp32 and 8064 of bf16 at a time, the last
    piece is a short one."""
    _pieces(ops, _on_gpu(n, 65536, 20, dtype, 64), "silu", dtype)


def test_wide_bf16_tiles_in_pieces(ops):  # noqa: F811
    """[dgate, dup] of 65536 rows at a time: x read where it is, and laid out (not aligned)."""
    n, dim = 70_001, 136
    x, *rest = _on_gpu(n, dim, 4096, BF16, 65)
    ref = _pieces(ops, (x, *rest), "gelu", BF16)
    room = torch.empty(n, dim + 8, dtype=BF16, device="cuda")
    room[:, 1:dim + 1] = x
    *weights, dh = rest
    for name, t in zip(NAMES, ops.gated_linear_grad(dh, room[:, 1:dim + 1], *weights, act="gelu")):
        _within(t, ref[name], name)


# ------------------------------------------------------------------ very many rows
@pytest.mark.parametrize("n,dtype", [((1 << 29) + 12_345, F32), ((1 << 30) + 12_345, BF16)])
def test_more_rows_than_a_launch_takes(ops, n, dtype):  # noqa: F811
    """Rows of one value: h in two launches (2^22 workgroups in each), the gradients in two and
    four. Few rows have a dh that is not 0, so that the weights' gradients are theirs."""
    some = torch.tensor([0, 1, n // 2 - 1, (1 << 29) - 1, 1 << 29, n - 12_346, n - 2, n - 1], device="cuda")
    x = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(7).sub_(3).to(dtype)[:, None]
    x.mul_(0.375)
    dh = torch.zeros(n, 1, dtype=dtype, device="cuda")
    dh[some] = (torch.arange(8, device="cuda")[:, None] * 0.25 - 0.8).to(dtype)
    some = some.unique()  # two of them are one row of the fp32 case, which is summed once
    _, wg, wu, bg, bu, _ = _inputs(1, 1, 1, dtype, seed=66)
    args = _cuda((wg, wu, bg, bu))
    ref = _reference(x[some].cpu(), wg, wu, bg, bu, dh[some].cpu(), "silu", dtype)
    h = ops.gated_linear(x, *args)
    _within(h[some].cpu(), ref["h"], "h")
    ends = torch.cat([torch.arange(5000, device="cuda"), torch.arange(n - 20_000, n, device="cuda")])
    assert torch.equal(h[ends], ops.gated_linear(x[ends], *args))
    del h
    dx, *rest = ops.gated_linear_grad(dh, x, *args)
    _within(dx[some].cpu(), ref["dx"], "dx")
    assert int(dx.count_nonzero()) <= 8
    for name, t in zip(NAMES[1:], rest):
        _within(t.cpu(), ref[name], name)
    del x, dh, dx, rest
    torch.cuda.empty_cache()

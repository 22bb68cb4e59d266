"""The gated projections against plain 64-bit formulas: types, activations, odd and
empty sizes, strides, values that are not finite, streams, graphs, refusals.

Tolerances are bounds on rounding, written down from the formulas. EPS = 2^-24 is fp32's
rounding, BF = 2^-8 bf16's: half a step, relative to the value."""
import ctypes
import math

import pytest
import torch

from gsplat_tt_amd import _lib as L

pytestmark = pytest.mark.gpu

EPS, BF = torch.finfo(torch.float32).eps / 2, torch.finfo(torch.bfloat16).eps / 2
F32, BF16, D64 = torch.float32, torch.bfloat16, torch.float64
ACTS = ("none", "relu", "silu", "gelu")


@pytest.fixture(scope="module")
def ops():
    from gsplat_tt_amd.field import FieldOps
    o = FieldOps()
    yield o
    o.check()
    o.ctx.close()


def _inputs(n, dim, hidden, dtype, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + n * 31 + dim * 7 + hidden)

    def randn(*s):
        return torch.randn(*s, generator=g)

    x = (randn(n, dim) + 0.3 * randn(dim)).to(dtype)
    wg, wu = ((randn(hidden, dim) * 1.5 / math.sqrt(dim)).to(dtype) for _ in range(2))
    bg, bu = (0.3 * randn(hidden) if bias else None for _ in range(2))
    dh = (randn(n, hidden) * 0.1).to(dtype)
    return x, wg, wu, bg, bu, dh


def _cuda(ts):
    return tuple(None if t is None else t.cuda() for t in ts)


def _act(z, act):
    return {"none": lambda v: v * 1.0, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
            "gelu": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2))}[act](z)


# An activation's and its slope's own error and theirs from their argument's: |act'| and
# |act''| stay below 1.13 (silu: 1.1 and 0.5; gelu: 1.13 and 0.8), and each value is a few
# operations of relative error EPS, some 8 of them hardware functions of 1 unit.
ACT_STEPS = 24


def _reference(x, wg, wu, bg, bu, dh, act, dtype):
    """Values in 64 bits with what each may be off."""
    dim, hidden, n = x.shape[1], wg.shape[0], x.shape[0]
    x, wg, wu, dh = (t.to(D64) for t in (x, wg, wu, dh))
    bg, bu = (torch.zeros(hidden, dtype=D64) if b is None else b.to(D64) for b in (bg, bu))
    gate = (x @ wg.T + bg).requires_grad_()
    up = x @ wu.T + bu
    a = _act(gate, act)
    slope, = torch.autograd.grad(a.sum(), gate)
    gate, a = gate.detach(), a.detach()
    # a sum of dim products: EPS dim of the terms' sizes for the sums in any order, and
    # 8 EPS for the parts of fp32 values that are left out: a value's second part is below
    # 2^-7 of it, the third below 2^-15, and two products of those two are not formed
    zt = EPS * (dim + 12)
    gt = zt * (x.abs() @ wg.abs().T + bg.abs())
    ut = zt * (x.abs() @ wu.abs().T + bu.abs())
    at = 1.13 * gt + ACT_STEPS * EPS * gate.abs()
    st = gt + ACT_STEPS * EPS * (1 + slope.abs())
    half = BF if dtype == BF16 else EPS
    r = {"h": (a * up, at * up.abs() + a.abs() * ut + at * ut + (half + 2 * EPS) * (a * up).abs())}
    dg, du = dh * up * slope, dh * a
    if act == "relu":  # the slope jumps where the gate is within rounding of 0
        st = torch.where(gate.abs() <= gt, torch.ones_like(st), st)
    dgt = dh.abs() * (ut * slope.abs() + up.abs() * st + ut * st) + 3 * EPS * dg.abs()
    dut = dh.abs() * at + 2 * EPS * du.abs()
    for name, d, t in (("db_gate", dg, dgt), ("db_up", du, dut)):
        r[name] = (d.sum(0), t.sum(0) + (n + 4) * EPS * (d.abs() + t).sum(0))
    if dtype == BF16:  # rounded as operands
        dgt, dut = dgt + BF * (dg.abs() + dgt), dut + BF * (du.abs() + dut)
    dgs, dus = dg.abs() + dgt, du.abs() + dut
    dx = dg @ wg + du @ wu
    r["dx"] = (dx, dgt @ wg.abs() + dut @ wu.abs() +
               EPS * (2 * hidden + 12) * (dgs @ wg.abs() + dus @ wu.abs()) + half * dx.abs())
    for name, d, t, s in (("dw_gate", dg, dgt, dgs), ("dw_up", du, dut, dus)):
        v = d.T @ x
        r[name] = (v, t.T @ x.abs() + EPS * (n + 12) * (s.T @ x.abs()) + half * v.abs())
    # the result's own rounding applies to what is off, too
    return {k: (v, t * (1 + 2 * half) + 1e-44) for k, (v, t) in r.items()}


def _check(got, ref, what):
    want, tol = ref
    got = got.detach().cpu().to(D64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    assert (off <= tol).all(), (what, (off / tol).max().item())


NAMES = ("dx", "dw_gate", "dw_up", "db_gate", "db_up")
SIZES = [(1, 1, 1), (1, 64, 256), (2, 3, 5), (7, 8, 16), (33, 512, 70), (64, 32, 32),
         (65, 33, 31), (127, 129, 65), (129, 64, 128), (300, 16, 200), (1000, 75, 201),
         (5, 1000, 17), (513, 128, 64), (2000, 40, 24), (4097, 64, 128), (1, 300, 1000),
         (16, 64, 33), (17, 256, 100), (640, 260, 136), (7, 512, 512), (31, 200, 333), (48, 140, 1000),
         (64, 129, 30), (3586, 100, 300), (200, 128, 2000), (2500, 136, 2500), (3000, 260, 700)]


@pytest.mark.parametrize("n,dim,hidden", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_and_gradients(ops, n, dim, hidden, dtype):
    act = ACTS[(n + dim + hidden) % 4]
    ins = _inputs(n, dim, hidden, dtype)
    ref = _reference(*ins, act, dtype)
    *args, dh = _cuda(ins)
    h = ops.gated_linear(*args, act=act)
    assert h.dtype == dtype
    _check(h, ref["h"], "h")
    grads = ops.gated_linear_grad(dh, *args, act=act)
    for name, g in zip(NAMES, grads):
        assert g.dtype == (F32 if name.startswith("db") else dtype)
        _check(g, ref[name], name)
    again = (ops.gated_linear(*args, act=act), *ops.gated_linear_grad(dh, *args, act=act))
    assert all(torch.equal(a, b) for a, b in zip(again, (h, *grads)))


# 2 hidden / 256 by rows / 256 tiles, at least 448 of them: the wide tiles
WIDE = [(4900, 136, 3000), (3801, 200, 4100), (2601, 145, 5700), (1900, 520, 7400),
        (115_001, 131, 40), (114_944, 256, 128), (23_000, 320, 700)]


@pytest.mark.parametrize("n,dim,hidden", WIDE)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_wide_tiles(ops, n, dim, hidden, dtype):
    test_values_and_gradients(ops, n, dim, hidden, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_wide_tiles_strides_and_values_that_are_not_finite(ops, dtype):
    for n, dim, hidden in ((4900, 136, 3000), (4700, 192, 3100)):
        test_strides_and_alignment(ops, dtype, n, dim, hidden)
    test_values_that_are_not_finite(ops, dtype, 4900, 136, 3000)
    test_broadcast_rows(ops, dtype, 4900, 136, 3000)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bias", [True, False])
def test_activations_and_biases(ops, act, dtype, bias):
    for n, dim, hidden in ((5, 48, 40), (333, 32, 64), (3000, 48, 100)):
        ins = _inputs(n, dim, hidden, dtype, bias, seed=3)
        ref = _reference(*ins, act, dtype)
        *args, dh = _cuda(ins)
        _check(ops.gated_linear(*args, act=act), ref["h"], "h")
        grads = ops.gated_linear_grad(dh, *args, act=act)
        assert (grads[3] is None) == (grads[4] is None) == (not bias)
        for name, g in zip(NAMES, grads):
            if g is not None:
                _check(g, ref[name], name)


def test_one_bias(ops):
    x, wg, wu, bg, bu, dh = _inputs(100, 24, 40, F32, seed=4)
    for one in ((bg, None), (None, bu)):
        ref = _reference(x, wg, wu, *one, dh, "silu", F32)
        *args, d = _cuda((x, wg, wu, *one, dh))
        _check(ops.gated_linear(*args), ref["h"], "h")
        grads = ops.gated_linear_grad(d, *args)
        for name, g in zip(NAMES, grads):
            if g is not None:
                _check(g, ref[name], name)
        assert [g is None for g in grads[3:]] == [b is None for b in one]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,dim,hidden", [(3, 40, 24), (70, 64, 32), (1000, 33, 70), (513, 256, 136)])
def test_strides_and_alignment(ops, dtype, n, dim, hidden):
    """Rows at other distances, one matrix with both weights, any element's address; what
    lies beside the outputs stays."""
    x, wg, wu, bg, bu, dh = _inputs(n, dim, hidden, dtype, seed=5)
    ref = _reference(x, wg, wu, bg, bu, dh, "silu", dtype)

    def room(rows, cols, at, pad):
        return torch.full((rows, cols + pad), 7.0, dtype=dtype, device="cuda"), slice(at, at + cols)

    for at, pad in ((0, 8), (1, 3), (8, 24)):
        def put(t):
            r, c = room(*t.shape, at, pad)
            r[:, c] = t.cuda()
            return r[:, c]

        both, c = room(2 * hidden, dim, at, pad)
        both[:, c] = torch.cat([wg, wu]).cuda()
        args = (put(x), both[:hidden, c], both[hidden:, c], bg.cuda(), bu.cuda())
        h, ch = room(n, hidden, at, pad)
        ops.gated_linear(*args, out=h[:, ch])
        outs = [room(n, dim, at, pad), room(hidden, dim, at, pad), room(hidden, dim, at, pad)]
        grads = ops.gated_linear_grad(put(dh), *args, dx=outs[0][0][:, outs[0][1]],
                                      dw_gate=outs[1][0][:, outs[1][1]],
                                      dw_up=outs[2][0][:, outs[2][1]])
        _check(h[:, ch], ref["h"], "h")
        for name, g in zip(NAMES, grads):
            _check(g, ref[name], name)
        for whole, cols in ((h, ch), *outs):
            whole[:, cols] = 7.0
            assert (whole == 7.0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_broadcast_rows(ops, dtype, n=700, dim=40, hidden=48):
    """One row of x and of dh for all samples (a stride of 0)."""
    x, wg, wu, bg, bu, dh = _inputs(1, dim, hidden, dtype, seed=6)
    many = (x.expand(n, -1), wg, wu, bg, bu, dh.expand(n, -1))
    ref = _reference(*many, "gelu", dtype)
    gx, gd = x.cuda().expand(n, -1), dh.cuda().expand(n, -1)
    args = (gx, *_cuda((wg, wu, bg, bu)))
    h = ops.gated_linear(*args, act="gelu")
    _check(h, ref["h"], "h")
    for name, g in zip(NAMES, ops.gated_linear_grad(gd, *args, act="gelu")):
        _check(g, ref[name], name)
    # one weight for both projections
    same = (x, wg, wg, None, None, dh)
    ref = _reference(*same, "silu", dtype)
    *args, d = _cuda(same)
    args = (args[0], args[1], args[1], None, None)
    _check(ops.gated_linear(*args), ref["h"], "h")
    for name, g in zip(NAMES[:3], ops.gated_linear_grad(d, *args)):
        _check(g, ref[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_rows(ops, dtype):
    x, wg, wu, bg, bu, dh = _cuda(_inputs(0, 20, 30, dtype))
    assert ops.gated_linear(x, wg, wu, bg, bu).shape == (0, 30)
    dx, *rest = ops.gated_linear_grad(dh, x, wg, wu, bg, bu)
    assert dx.shape == (0, 20)
    assert all(not g.any() and g.isfinite().all() for g in rest)
    assert rest[0].shape == (30, 20) and rest[2].shape == (30,)


@pytest.mark.parametrize("n,dim,hidden", [(1, 136, 57_400), (3, 131, 57_500), (70, 136, 57_400)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_rows_of_many_units(ops, n, dim, hidden, dtype):
    """The units alone fill the wide tiles, whose rows are nearly all past the last one."""
    ins = _inputs(n, dim, hidden, dtype)
    ref = _reference(*ins, "silu", dtype)
    *args, dh = _cuda(ins)
    _check(ops.gated_linear(*args), ref["h"], "h")
    for name, g in zip(NAMES, ops.gated_linear_grad(dh, *args)):
        _check(g, ref[name], name)


@pytest.mark.parametrize("dim,hidden", [(200, 30), (136, 57_400)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_rows_of_long_features(ops, dim, hidden, dtype):
    """The weights' gradients are zeros, written over what was there; nothing around them is."""
    x, wg, wu, bg, bu, dh = _cuda(_inputs(0, dim, hidden, dtype))
    assert ops.gated_linear(x, wg, wu, bg, bu).shape == (0, hidden)
    rooms = [torch.full((hidden + 2, dim + 8), 3.0, dtype=dtype, device="cuda") for _ in range(2)]
    outs = [r[1:-1, :dim] for r in rooms]
    dx, *rest = ops.gated_linear_grad(dh, x, wg, wu, bg, bu, dw_gate=outs[0], dw_up=outs[1])
    assert dx.shape == (0, dim) and not any(t.any() for t in rest)
    for r in rooms:
        assert (r[0] == 3).all() and (r[-1] == 3).all() and (r[:, dim:] == 3).all()


@pytest.mark.parametrize("n,dim,hidden", [(4, 40, 24), (300, 32, 64), (300, 72, 130), (200, 300, 40)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_that_are_not_finite(ops, dtype, n, dim, hidden):
    """They act as in plain arithmetic: rows, units and columns without them are as
    before, those with them are what the formula in fp32 says."""
    x, wg, wu, bg, bu, dh = _inputs(n, dim, hidden, dtype, seed=8)
    x, wg = x.abs() + 0.1, wg.abs() + 0.1  # no difference of infinities
    x[1, 2], x[3, 0] = float("inf"), float("nan")
    wu[5, 1], wg[7, 3] = float("-inf"), float("nan")
    dh[2, 9] = float("inf")
    act = "relu"
    f = [t.float() for t in (x, wg, wu)]
    gate, up = f[0] @ f[1].T + bg, f[0] @ f[2].T + bu
    want = torch.relu(gate) * up
    got = ops.gated_linear(*_cuda((x, wg, wu, bg, bu)), act=act).float().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf())
    same = want.isinf()
    assert torch.equal(got[same], want[same])
    dg, du = dh.float() * up * (gate > 0), dh.float() * torch.relu(gate)
    ref = {"dx": dg @ f[1] + du @ f[2], "dw_gate": dg.T @ f[0], "dw_up": du.T @ f[0],
           "db_gate": dg.sum(0), "db_up": du.sum(0)}
    for name, g in zip(NAMES, ops.gated_linear_grad(*_cuda((dh, x, wg, wu, bg, bu)), act=act)):
        g = g.float().cpu()
        assert torch.equal(g.isfinite(), ref[name].isfinite()), name


def test_wide_range_of_values(ops):
    """fp32 values far apart in size keep their digits."""
    g = torch.Generator().manual_seed(9)
    n, dim, hidden = 200, 64, 48
    x = torch.randn(n, dim, generator=g) * 10.0 ** torch.randint(-12, 12, (n, dim), generator=g)
    wg, wu = (torch.randn(hidden, dim, generator=g) *
              10.0 ** torch.randint(-8, 8, (hidden, dim), generator=g) for _ in range(2))
    dh = torch.randn(n, hidden, generator=g) * 10.0 ** torch.randint(-9, 3, (n, hidden), generator=g)
    ref = _reference(x, wg, wu, None, None, dh, "none", F32)
    args = (*_cuda((x, wg, wu)), None, None)
    _check(ops.gated_linear(*args, act="none"), ref["h"], "h")
    for name, t in zip(NAMES[:3], ops.gated_linear_grad(dh.cuda(), *args, act="none")):
        _check(t, ref[name], name)


def test_gradients_match_differences(ops):
    x, wg, wu, bg, bu, dh = (t.to(D64) for t in _inputs(20, 12, 16, F32, seed=10))
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    base = dict(zip(names, (x, wg, wu, bg, bu)))

    def value(p):
        h = _act(p["x"] @ p["w_gate"].T + p["b_gate"], "gelu") * (p["x"] @ p["w_up"].T + p["b_up"])
        return (h * dh).sum()

    args = [t.float().cuda() for t in (x, wg, wu, bg, bu)]
    grads = ops.gated_linear_grad(dh.float().cuda(), *args, act="gelu")
    g = torch.Generator().manual_seed(11)
    for name, grad in zip(names, grads):
        step = torch.randn(base[name].shape, generator=g, dtype=D64)
        step /= step.norm()
        h = 1e-4
        up, down = (value({**base, name: base[name] + s * h * step}) for s in (1, -1))
        slope = (up - down) / (2 * h)
        # truncation h^2 times a third derivative of order 10, fp32 some 100 roundings
        size = grad.double().norm().item()
        assert abs((grad.cpu().to(D64) * step).sum() - slope) <= 1e-6 * 10 + 100 * EPS * size, name


@pytest.mark.parametrize("dim", [24, 140])
def test_many_rows_in_pieces(ops, dim):
    """More rows than one piece of the workspace takes (of the longer rows): the weights'
    sums go over pieces."""
    n, hidden = 90_001, 2000
    g = torch.Generator(device="cuda").manual_seed(12)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    x, wg, wu = randn(n, dim), randn(hidden, dim) / 5, randn(hidden, dim) / 5
    bg, bu, dh = randn(hidden) / 3, randn(hidden) / 3, randn(n, hidden) / 100
    h = ops.gated_linear(x, wg, wu, bg, bu)
    grads = ops.gated_linear_grad(dh, x, wg, wu, bg, bu)
    sums = {k: 0 for k in NAMES[1:]}
    tols = {k: 0 for k in NAMES[1:]}
    step = 10_000
    for lo in range(0, n, step):
        at = slice(lo, lo + step)
        ref = _reference(*(t.cpu() for t in (x[at], wg, wu, bg, bu, dh[at])), "silu", F32)
        _check(h[at], ref["h"], "h")
        _check(grads[0][at], ref["dx"], "dx")
        for k in sums:
            sums[k] = sums[k] + ref[k][0]
            tols[k] = tols[k] + ref[k][1]
    for k, t in zip(NAMES[1:], grads[1:]):
        # the pieces' tolerances have sums of `step` terms; n terms are n / step times that
        _check(t, (sums[k], tols[k] * (n / step)), k)


@pytest.mark.parametrize("n,dim,hidden,dtype", [(1, 64, 100, F32), (40, 64, 256, BF16),
                                                (700, 75, 60, F32), (3000, 64, 128, BF16),
                                                (900, 256, 200, BF16), (4900, 136, 3000, BF16),
                                                (4900, 136, 3000, F32)])
def test_captured_and_replayed(ops, n, dim, hidden, dtype):
    """Two graphs and eager calls between the replays, new inputs in the same buffers."""
    sets = [_cuda(_inputs(n, dim, hidden, dtype, seed=s)) for s in (20, 21, 22)]
    bufs = [t.clone() for t in sets[0]]
    x, wg, wu, bg, bu, dh = bufs

    def run():
        return (ops.gated_linear(x, wg, wu, bg, bu), *ops.gated_linear_grad(dh, x, wg, wu, bg, bu))

    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run()
        graphs.append((g, outs))
    for k in (0, 1, 2, 1):
        for b, t in zip(bufs, sets[k]):
            b.copy_(t)
        want = [t.clone() for t in run()]
        for g, outs in graphs:
            for o in outs:
                o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_streams(ops):
    """Calls on two streams at once, each with outputs and workspace of its own."""
    jobs = [_cuda(_inputs(2000 + 300 * k, 64, 128, BF16, seed=30 + k)) for k in range(2)]
    want = [(ops.gated_linear(*j[:5]), *ops.gated_linear_grad(j[5], *j[:5])) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for _ in range(3):
        for j, s in zip(jobs, streams):
            with torch.cuda.stream(s):
                got.append((ops.gated_linear(*j[:5]), *ops.gated_linear_grad(j[5], *j[:5])))
    torch.cuda.synchronize()
    for k, outs in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(outs, want[k % 2]))


def test_refusals(ops):
    x, wg, wu, bg, bu, dh = _cuda(_inputs(6, 8, 10, F32))
    with pytest.raises(TypeError, match="w_up"):
        ops.gated_linear(x, wg, wu.bfloat16())
    with pytest.raises(ValueError, match="columns"):
        ops.gated_linear(x, wg[:, :7], wu)
    with pytest.raises(ValueError, match="rows"):
        ops.gated_linear(x, wg, wu[:9])
    with pytest.raises(ValueError, match="b_gate"):
        ops.gated_linear(x, wg, wu, bg[:9], bu)
    with pytest.raises(TypeError, match="b_up"):
        ops.gated_linear(x, wg, wu, bg, bu.bfloat16())
    with pytest.raises(ValueError, match="act"):
        ops.gated_linear(x, wg, wu, act="tanh")
    with pytest.raises(ValueError, match="dimensions"):
        ops.gated_linear(x[0], wg, wu)
    with pytest.raises(ValueError, match="contiguous"):
        ops.gated_linear(x, wg.T.contiguous().T, wu)
    with pytest.raises(TypeError, match="type"):
        ops.gated_linear(x.half(), wg.half(), wu.half())
    with pytest.raises(ValueError, match="is on"):
        ops.gated_linear(x.cpu(), wg, wu)
    with pytest.raises(ValueError, match="out"):
        ops.gated_linear(x, wg, wu, out=torch.empty(6, 9, device="cuda"))
    with pytest.raises(TypeError, match="out"):
        ops.gated_linear(x, wg, wu, out=torch.empty(6, 10, device="cuda", dtype=BF16))
    with pytest.raises(ValueError, match="overlap"):
        ops.gated_linear(x, wg, wu, out=torch.empty(1, 10, device="cuda").expand(6, 10))
    with pytest.raises(TypeError, match="dh"):
        ops.gated_linear_grad(dh.bfloat16(), x, wg, wu)
    with pytest.raises(ValueError, match="dh"):
        ops.gated_linear_grad(dh[:5], x, wg, wu)
    with pytest.raises(TypeError, match="dw_up"):
        ops.gated_linear_grad(dh, x, wg, wu, dw_up=torch.empty_like(wu, dtype=BF16))
    with pytest.raises(ValueError, match="requires a gradient"):
        ops.gated_linear(x, wg.clone().requires_grad_(), wu)
    with torch.no_grad():
        assert ops.gated_linear(x, wg.clone().requires_grad_(), wu).shape == (6, 10)
    with pytest.raises(ValueError, match="hidden"):
        ops.gated_linear(x, wg[:0], wu[:0])


def test_closed_context_and_c_boundary(ops):
    from gsplat_tt_amd.field import FieldOps
    x, wg, wu, bg, bu, dh = _cuda(_inputs(6, 8, 10, F32))
    own = FieldOps()
    own.ctx.close()
    for call in (lambda: own.gated_linear(x, wg, wu), lambda: own.gated_linear_grad(dh, x, wg, wu),
                 lambda: own.grad_norm([x]), lambda: own.clip_grads([x.clone()], 1.0)):
        with pytest.raises(ValueError, match="null ctx"):
            call()
    lib = ops._L
    d, keep = ops._gated(x, wg, wu, bg, bu, "silu")
    size = lib.gs_gated_linear_workspace(ctypes.byref(d), 0)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    h = torch.full((6, 10), 3.0, device="cuda")
    args = (ctypes.byref(d), h.data_ptr(), 10)
    if size > 0:
        assert lib.gs_gated_linear_dev(ops.ctx.handle, *args, ws.data_ptr(), size - 1, None) == \
            L.GS_E_INVALID
    assert lib.gs_gated_linear_dev(ops.ctx.handle, ctypes.byref(d), None, 10, ws.data_ptr(), size,
                                   None) == L.GS_E_INVALID
    assert lib.gs_gated_linear_dev(ops.ctx.handle, ctypes.byref(d), h.data_ptr(), 9, ws.data_ptr(),
                                   size, None) == L.GS_E_INVALID
    torch.cuda.synchronize()
    assert (h == 3.0).all()
    # gradients of one bias alone
    size = lib.gs_gated_linear_workspace(ctypes.byref(d), 1)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    want = ops.gated_linear_grad(dh, x, wg, wu, bg, bu)
    outs = [torch.empty_like(t) for t in want]
    for skip in (3, 4):
        ptr = [t.data_ptr() for t in outs]
        ptr[skip] = None
        assert lib.gs_gated_linear_grad_dev(
            ops.ctx.handle, ctypes.byref(d), dh.data_ptr(), 10, ptr[0], 8, ptr[1], 8, ptr[2], 8,
            ptr[3], ptr[4], ws.data_ptr(), size, ops._stream()) == 0
        assert all(torch.equal(a, b) for k, (a, b) in enumerate(zip(outs, want)) if k != skip)
    del keep


# ------------------------------------------------------------------ far apart
@pytest.mark.parametrize("stride", [(1 << 22) - 8, 1 << 22, (1 << 23) + 8])
def test_rows_far_apart(ops, stride):
    """300 rows some megabytes apart, offsets past 32 bits: wide tiles whose rows of x are
    read where they are, or laid out before."""
    n, dim, hidden = 300, 136, 30_000
    x, wg, wu, bg, bu, dh = _inputs(n, dim, hidden, BF16, seed=40)
    room = torch.empty(n * stride, dtype=BF16, device="cuda")
    far = torch.as_strided(room, (n, dim), (stride, 1))
    far.copy_(x)
    near = _cuda((x, wg, wu, bg, bu))
    dh = dh.cuda()
    h = ops.gated_linear(far, *near[1:])
    want = ops.gated_linear(*near)
    assert torch.equal(h, want)
    for a, b in zip(ops.gated_linear_grad(dh, far, *near[1:]), ops.gated_linear_grad(dh, *near)):
        assert torch.equal(a, b)
    ref = _reference(x[:40], wg, wu, bg, bu, dh[:40].cpu(), "silu", BF16)
    _check(h[:40], ref["h"], "h")
    del room, far
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,dim,hidden,dtype", [(700, 72, 33_000, BF16), (400, 600, 25_000, BF16),
                                                (300, 40, 9000, F32), (150, 140, 20_000, F32)])
def test_many_units(ops, n, dim, hidden, dtype):
    """More units than rows: the weights' tiles alone fill the chip."""
    test_values_and_gradients(ops, n, dim, hidden, dtype)


def test_outputs_over_other_tensors_are_refused(ops):
    """They would be read and written at once, or written twice."""
    n = 90
    x, wg, wu, bg, bu, dh = _cuda(_inputs(n, 24, 24, F32, seed=50))
    before = [t.clone() for t in (x, wg, wu, bg, bu, dh)]
    args = (x, wg, wu, bg, bu)
    both = torch.full((48, 24), 3.0, device="cuda")
    for call in (lambda: ops.gated_linear(*args, out=x),
                 lambda: ops.gated_linear(x[:24], wg, wu, out=wu),
                 lambda: ops.gated_linear(*args, out=both[:1].expand(n, 24)),
                 lambda: ops.gated_linear_grad(dh, *args, dx=x),
                 lambda: ops.gated_linear_grad(dh, *args, dx=dh),
                 lambda: ops.gated_linear_grad(dh, *args, dw_gate=wg),
                 lambda: ops.gated_linear_grad(dh, *args, dw_gate=both[:24], dw_up=both[:24]),
                 lambda: ops.gated_linear_grad(dh, *args, dw_gate=both[:24], dw_up=both[23:47])):
        with pytest.raises(ValueError, match="shares memory|overlap"):
            call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((x, wg, wu, bg, bu, dh), before))
    assert (both == 3.0).all()
    # beside each other they are taken, in one matrix by turns of rows too
    want = ops.gated_linear_grad(dh, *args)
    for dw_gate, dw_up in ((both[:24], both[24:]), (both[::2], both[1::2])):
        got = ops.gated_linear_grad(dh, *args, dw_gate=dw_gate, dw_up=dw_up)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    room = torch.zeros(n, 48, device="cuda")
    room[:, :24] = x
    ops.gated_linear(room[:, :24], wg, wu, bg, bu, out=room[:, 24:])
    assert torch.equal(room[:, 24:], ops.gated_linear(*args)) and torch.equal(room[:, :24], x)

"""The feature operators (lookup, group norm, label loss) against plain 64-bit
formulas: types, masks, odd and empty sizes, strides, streams, graphs, refusals.

Tolerances are bounds on fp32 rounding, written down from the formulas: EPS is
the unit roundoff 2^-24, a sum of m terms in any order is off by at most
m EPS sum|terms|, and a bf16 result, of 8 significant bits, is off by 2^-8 of
itself (BF)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from gsplat_tt_amd import _lib as L

pytestmark = pytest.mark.gpu

EPS, BF = 2.0 ** -24, 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16
D64 = torch.float64


@pytest.fixture(scope="module")
def ops():
    from gsplat_tt_amd.field import FieldOps
    o = FieldOps()
    yield o
    o.check()
    o.ctx.close()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype)


def _ids(g, n, rows, masked=0.1):
    ids = torch.randint(0, max(rows, 1), (n,), generator=g)
    return torch.where(torch.rand(n, generator=g) < masked, torch.full_like(ids, -1), ids)


def _close(got, want, tol, what):
    got, want = got.detach().cpu().to(D64), want.to(D64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all(), what
    assert (off <= tol).all(), (what, worst, off.max().item())


# ------------------------------------------------------------------ lookup
@pytest.mark.parametrize("n,rows,dim", [(0, 5, 8), (1, 1, 1), (7, 3, 3), (1000, 169, 32),
                                        (4097, 999, 45), (513, 20, 300), (33, 4, 4096),
                                        (70001, 65536, 27)])
@pytest.mark.parametrize("tt,to", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)])
def test_lookup(ops, n, rows, dim, tt, to):
    g = _gen(n + rows + dim)
    table = _randn(g, rows, dim, dtype=tt)
    ids = _ids(g, n, rows)
    scale = 0.7071
    want = torch.where((ids >= 0)[:, None],
                       table.float()[ids.clamp(min=0)] * np.float32(scale),
                       torch.zeros(1)).to(to)
    for kind in (torch.int32, torch.int64):
        got = ops.lookup(table.cuda(), ids.to(kind).cuda(), scale, dtype=to)
        assert got.dtype == to and torch.equal(got.cpu(), want)


def test_lookup_strides_and_offsets(ops):
    g = _gen(3)
    big = _randn(g, 50, 67).cuda()
    ids = _ids(g, 777, 50).cuda()
    for lo, dim in ((0, 64), (1, 64), (3, 45), (4, 60)):
        table = big[:, lo:lo + dim]
        want = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)] * 2.0, torch.zeros_like(big[:1, :1]))
        room = torch.full((777, 80), 9.0, device="cuda")
        for at in (0, 1, 8):
            room.fill_(9.0)
            ops.lookup(table, ids, 2.0, out=room[:, at:at + dim])
            assert torch.equal(room[:, at:at + dim], want)
            rest = room.clone()
            rest[:, at:at + dim] = 9.0
            assert (rest == 9.0).all()
    rows = ops.lookup(big[:1].expand(50, 67), ids, 1.0)  # one row for every id
    assert torch.equal(rows[ids >= 0], big[:1].expand(int((ids >= 0).sum()), 67))


def test_lookup_range_flag(ops):
    table = torch.ones(4, 5, device="cuda")
    ids = torch.tensor([0, -7, 3, 4, 2 ** 40], device="cuda")
    out = ops.lookup(table, ids)
    assert torch.equal(out.cpu()[:, 0], torch.tensor([1.0, 0.0, 1.0, 0.0, 0.0]))
    with pytest.raises(ValueError, match="past"):
        ops.check()
    ops.check()  # the report is given once
    ops.lookup_grad(torch.ones(5, 5, device="cuda"), ids, 4)
    with pytest.raises(ValueError, match="past"):
        ops.check()
    assert ops.lookup(torch.empty(0, 5, device="cuda"), ids[:0]).shape == (0, 5)
    # a table without rows: every id is past it
    assert not ops.lookup(torch.empty(0, 5, device="cuda"), ids).any()
    with pytest.raises(ValueError, match="past"):
        ops.check()


def _grad_case(n, rows, dim, dtype, seed, hot=0.0):
    g = _gen(seed)
    ids = _ids(g, n, rows)
    if hot:
        ids = torch.where(torch.rand(n, generator=g) < hot, torch.full_like(ids, rows // 2), ids)
    return _randn(g, n, dim, dtype=dtype), ids


def _grad_ref(dout, ids, rows, scale):
    out = torch.zeros(rows, dout.shape[1], dtype=D64)
    size = torch.zeros(rows, dout.shape[1], dtype=D64)
    count = torch.zeros(rows, dtype=D64)
    on = ids >= 0
    out.index_add_(0, ids[on], dout[on].to(D64))
    size.index_add_(0, ids[on], dout[on].to(D64).abs())
    count.index_add_(0, ids[on], torch.ones(int(on.sum()), dtype=D64))
    return out * scale, (count[:, None] + 2) * EPS * size * abs(scale)


@pytest.mark.parametrize("n,rows,dim,hot", [
    (0, 5, 8, 0), (1, 1, 1, 0), (7, 3, 3, 0), (1000, 169, 32, 0), (4097, 999, 45, 0),
    (20000, 1, 64, 0), (30011, 24, 64, 0), (50000, 70000, 16, 0.5), (3000, 7, 513, 0),
    (100003, 300, 48, 0.9), (513, 100000, 3, 0), (4096, 255, 8, 0), (4096, 256, 8, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lookup_grad(ops, n, rows, dim, hot, dtype):
    dout, ids = _grad_case(n, rows, dim, dtype, n + dim, hot)
    want, tol = _grad_ref(dout, ids, rows, 1.5)
    a = ops.lookup_grad(dout.cuda(), ids.cuda(), rows, 1.5, dtype=F32)
    _close(a, want, tol, "dtable")
    b = ops.lookup_grad(dout.cuda(), ids.int().cuda(), rows, 1.5, dtype=F32)
    assert torch.equal(a, b)  # the same sums in the same order
    c = ops.lookup_grad(dout.cuda(), ids.cuda(), rows, 1.5, dtype=BF16)
    assert torch.equal(c, a.to(BF16))


def test_lookup_grad_accumulates_strides_and_masked_values(ops):
    dout, ids = _grad_case(5000, 37, 48, F32, 5)
    want, tol = _grad_ref(dout, ids, 37, 0.5)
    dout[ids < 0] = float("nan")  # masked rows are not read into any sum
    wide = torch.full((5000, 50), float("inf"))
    wide[:, 1:49] = dout
    first = _randn(_gen(6), 37, 64)
    room = first.cuda()
    ops.lookup_grad(wide.cuda()[:, 1:49], ids.cuda(), 37, 0.5, out=room[:, 8:56], accumulate=True)
    got = room.cpu()
    _close(got[:, 8:56], first[:, 8:56].to(D64) + want,
           tol + EPS * 2 * (first[:, 8:56].abs() + want.abs()), "sum")
    assert torch.equal(got[:, :8], first[:, :8]) and torch.equal(got[:, 56:], first[:, 56:])
    # one row repeated for every id (a broadcast gradient)
    one = dout[:1].nan_to_num(1.0)
    want, tol = _grad_ref(one.expand(5000, 48), ids, 37, 1.0)
    _close(ops.lookup_grad(one.cuda().expand(5000, 48), ids.cuda(), 37), want, tol, "broadcast")


def test_lookup_grad_matches_differences(ops):
    g = _gen(8)
    table, ids = _randn(g, 11, 6).to(D64), _ids(g, 200, 11)
    d = _randn(g, 200, 6)

    def value(t):
        rows = torch.where((ids >= 0)[:, None], t[ids.clamp(min=0)] * 1.25, torch.zeros(1, dtype=D64))
        return (rows * d.to(D64)).sum()

    got = ops.lookup_grad(d.cuda(), ids.cuda(), 11, 1.25).cpu().to(D64)
    step = _randn(g, 11, 6).to(D64)
    h = 1e-3  # the value is linear: no truncation error
    slope = (value(table + h * step) - value(table - h * step)) / (2 * h)
    assert abs((got * step).sum() - slope) <= 200 * EPS * d.abs().sum() * 1.25 * step.abs().max()


# ------------------------------------------------------------------ group norm
def _act64(z, act):
    return {"none": lambda v: v * 1, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
            "gelu": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2))}[act](z)


def _norm_ref(x, groups, w, b, act, eps, dy=None):
    """y, mean, rstd, dx, dw, db in 64 bits, and xh, dz."""
    x = x.to(D64)
    bt, c = x.shape[0], x.shape[-1]
    v = x.reshape(bt, -1, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    rstd = ((v - mean).square().mean((1, 3), keepdim=True) + eps) ** -0.5
    xh = (v - mean) * rstd
    w = (torch.ones(c) if w is None else w).to(D64).view(groups, -1)
    b = (torch.zeros(c) if b is None else b).to(D64).view(groups, -1)
    z = (xh * w + b).requires_grad_(dy is not None)
    y = _act64(z, act)
    r = {"y": y.detach().reshape(x.shape), "mean": mean[:, 0, :, 0], "rstd": rstd[:, 0, :, 0],
         "reach": (v.abs().amax((1, 3), keepdim=True) * rstd)}
    if dy is not None:
        dz, = torch.autograd.grad(y, z, dy.to(D64).reshape(v.shape))
        t = dz * w
        m1, m2 = t.mean((1, 3), keepdim=True), (t * xh).mean((1, 3), keepdim=True)
        r["dx"] = (rstd * (t - m1 - xh * m2)).reshape(x.shape)
        r["dw"], r["db"] = (dz * xh).sum((0, 1)).reshape(c), dz.sum((0, 1)).reshape(c)
        # what the terms weigh: a relative error k EPS (1 + reach) of xh moves
        # each factor by as much
        one = 1 + r["reach"]
        size = dy.to(D64).abs().reshape(v.shape) * (1 + w.abs()) * (1 + w.abs() + b.abs())
        r["dw_size"] = (size * (1 + xh.abs()) * one).sum((0, 1)).reshape(c)
        r["db_size"] = (size * one).sum((0, 1)).reshape(c)
        ts = size * (1 + xh.abs()) * one
        r["dx_size"] = (rstd * (ts + (1 + xh.abs()) * ts.mean((1, 3), keepdim=True))).reshape(x.shape)
    r["y_size"] = ((1 + w.abs()) * (r["reach"] + xh.abs() + 1) + b.abs()).reshape(x.shape)
    return r


# rounding steps on the way of one value: the statistics' joins (at most 64 a
# thread and 16 across), the normalisation, exp or erf (a few units), quotients
STEPS = 96

NORM_SIZES = [(1, (1,), 1, 1), (1, (1,), 8, 2), (2, (3, 5), 6, 3), (1, (17, 19), 48, 16),
              (3, (64,), 32, 8), (2, (40, 33), 96, 32), (1, (200, 111), 64, 1),
              (1, (3,), 2100, 7), (5, (7, 9), 40, 40), (2, (65, 64), 20, 5)]


@pytest.mark.parametrize("bt,pixels,c,groups", NORM_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_group_norm(ops, bt, pixels, c, groups, dtype, act):
    g = _gen(c + groups + len(act))
    x = (_randn(g, bt, *pixels, c) * (0.5 + torch.rand(c, generator=g)) +
         _randn(g, c)).to(dtype)
    w, b = 1 + 0.3 * _randn(g, c), 0.3 * _randn(g, c)
    dy = _randn(g, bt, *pixels, c, dtype=dtype)
    r = _norm_ref(x, groups, w, b, act, 1e-5, dy)
    y, mean, rstd = ops.group_norm(x.cuda(), groups, w.cuda(), b.cuda(), act=act)
    out = BF if dtype == BF16 else 0.0
    _close(y, r["y"], STEPS * EPS * r["y_size"] + out * r["y"].abs() + 1e-38, "y")
    _close(mean, r["mean"], STEPS * EPS * (r["reach"][:, 0, :, 0] / r["rstd"]), "mean")
    _close(rstd, r["rstd"], STEPS * EPS * r["rstd"] * (1 + r["reach"][:, 0, :, 0]), "rstd")
    dx, dw, db = ops.group_norm_grad(dy.cuda(), x.cuda(), mean, rstd, groups, w.cuda(), b.cuda(),
                                     act=act)
    # where z is within rounding of relu's kink the slope may be either 0 or 1: the
    # element's own gradient may come or go, in dx and in the sums
    v = x.to(D64).reshape(bt, -1, groups, c // groups)
    rstd64 = r["rstd"][:, None, :, None]
    xh = (v - r["mean"][:, None, :, None]) * rstd64
    z = xh.reshape(x.shape) * w.to(D64) + b.to(D64)
    kink = (z.abs() <= STEPS * EPS * r["y_size"]) if act == "relu" else torch.zeros_like(z).bool()
    own = torch.where(kink, dy.to(D64).abs(), torch.zeros_like(z))
    wown = (own * w.abs().to(D64)).reshape(v.shape)
    own_dx = rstd64 * (wown + wown.mean((1, 3), keepdim=True) +
                       xh.abs() * (wown * xh.abs()).mean((1, 3), keepdim=True))
    own_dw = (own * xh.reshape(x.shape).abs()).reshape(-1, c).sum(0)
    _close(dx, r["dx"], STEPS * EPS * r["dx_size"] + out * r["dx"].abs() + 1e-38 +
           own_dx.reshape(x.shape), "dx")
    _close(dw, r["dw"], STEPS * EPS * r["dw_size"] + own_dw, "dw")
    _close(db, r["db"], STEPS * EPS * r["db_size"] + own.reshape(-1, c).sum(0), "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_far_mean_constant_and_no_parameters(ops, dtype):
    """A mean far above the spread, a constant group (variance 0), and an outlier
    in the first pixel; no weight and bias."""
    g = _gen(1)
    x = _randn(g, 2, 50, 31, 16).to(F32)
    x[0, :, :, :4] += 1000.0
    x[0, :, :, 4:8] = 3.0
    x[1, 0, 0, :] = 3e4
    x = x.to(dtype)
    r = _norm_ref(x, 4, None, None, "silu", 1e-5)
    y, mean, rstd = ops.group_norm(x.cuda(), 4, act="silu")
    out = BF if dtype == BF16 else 0.0
    _close(y, r["y"], STEPS * EPS * r["y_size"] + out * r["y"].abs(), "y")
    _close(rstd, r["rstd"], STEPS * EPS * r["rstd"] * (1 + r["reach"][:, 0, :, 0]), "rstd")


def test_group_norm_strides_inplace_and_empty(ops):
    g = _gen(2)
    room = _randn(g, 3, 20, 21, 40).cuda()
    for lo, c in ((0, 32), (1, 32), (3, 5), (4, 36)):
        x = room[..., lo:lo + c]
        want = ops.group_norm(x.contiguous(), 1, act="gelu")
        got = ops.group_norm(x, 1, act="gelu", out=torch.empty_like(room)[..., :c])
        for a, b in zip(got, want):
            _close(a, b.cpu().to(D64), 64 * EPS * (1 + b.abs().cpu().to(D64)), "strided")
        same = room.clone()
        v = same[..., lo:lo + c]
        ops.group_norm(v, 1, act="gelu", out=v)
        _close(v, want[0].cpu().to(D64), 64 * EPS * (1 + want[0].abs().cpu().to(D64)), "in place")
        assert torch.equal(same[..., :lo], room[..., :lo])
        assert torch.equal(same[..., lo + c:], room[..., lo + c:])
    # images with other images between them
    x = room[::2]
    a, b = ops.group_norm(x, 8, act="relu"), ops.group_norm(x.contiguous(), 8, act="relu")
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for shape in ((0, 4, 8), (2, 0, 8)):
        e = torch.empty(shape, device="cuda")
        y, mean, rstd = ops.group_norm(e, 2)
        dx, dw, db = ops.group_norm_grad(e, e, mean, rstd, 2)
        assert y.shape == dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_group_norm_grad_matches_differences(ops, act):
    g = _gen(4)
    x, w, b = _randn(g, 2, 30, 12), 1 + 0.2 * _randn(g, 12), 0.2 * _randn(g, 12)
    d = _randn(g, 2, 30, 12)
    y, mean, rstd = ops.group_norm(x.cuda(), 3, w.cuda(), b.cuda(), act=act)
    grads = ops.group_norm_grad(d.cuda(), x.cuda(), mean, rstd, 3, w.cuda(), b.cuda(), act=act)

    def value(p):
        return (_norm_ref(p[0], 3, p[1], p[2], act, 1e-5)["y"] * d.to(D64)).sum()

    at = [t.to(D64) for t in (x, w, b)]
    for k, got in enumerate(grads):
        step = _randn(g, *at[k].shape).to(D64)

        def slope(h):
            up, down = list(at), list(at)
            up[k], down[k] = at[k] + h * step, at[k] - h * step
            return (value(up) - value(down)) / (2 * h)

        coarse, fine = slope(2e-3), slope(1e-3)
        # the truncation error falls by 4 with the step: the difference bounds it
        tol = (coarse - fine).abs() + 1e-9 + STEPS * EPS * 20 * d.abs().sum()
        assert abs((got.cpu().to(D64) * step).sum() - fine) <= tol


# ------------------------------------------------------------------ label loss
def _loss_case(n, rows, dim, dtype, seed):
    g = _gen(seed)
    table = _randn(g, rows, dim)
    table /= table.norm(dim=1, keepdim=True).clamp(min=1e-3)
    labels = _ids(g, n, rows)
    feat = _randn(g, n, dim) / math.sqrt(dim) + 0.5 * table[labels.clamp(min=0)]
    weight = torch.rand(n, generator=g)
    return feat.to(dtype), table.to(dtype), labels, weight


def _loss_ref(feat, table, labels, weight, scale):
    f, t = feat.to(D64), table.to(D64)
    on = labels >= 0
    s = scale * f @ t.T
    # a score: dim products and the 6 parts' joins in fp32
    es = (f.shape[1] + 8) * EPS * abs(scale) * (f.abs() @ t.abs().T) + 4 * EPS * s.abs()
    lse = torch.logsumexp(s, 1)
    at = labels.clamp(min=0)[:, None]
    loss = torch.where(on, lse - s.gather(1, at)[:, 0], torch.zeros(1, dtype=D64))
    e = es.amax(1) + 16 * EPS * (1 + lse.abs() + s.abs().amax(1))
    rows = f.shape[0]
    p = torch.exp(s - lse[:, None])
    one = torch.zeros_like(p)
    one[torch.arange(rows), at[:, 0]] = 1.0
    w = torch.where(on, weight.to(D64) * scale, torch.zeros(1, dtype=D64))[:, None]
    gm = w * (p - one)
    eg = w.abs() * (p * 2 * e[:, None] + 4 * EPS * (p + one))
    return dict(loss=loss, lse=torch.where(on, lse, torch.zeros(1, dtype=D64)), e=2 * e, g=gm,
                eg=eg, f=torch.where(on[:, None], f, torch.zeros(1, dtype=D64)), t=t)


def _check_loss(r, loss, lse, dfeat, dtable, dtype):
    _close(loss, r["loss"], r["e"], "loss")
    _close(lse, r["lse"], r["e"], "lse")
    out = BF if dtype == BF16 else 0.0
    g, eg = r["g"].abs(), r["eg"] + (BF if dtype == BF16 else 2.0 ** -22) * r["g"].abs()
    n, rows = g.shape
    _close(dfeat, r["g"] @ r["t"], (eg + (rows + 8) * EPS * g) @ r["t"].abs() +
           out * (r["g"] @ r["t"]).abs() + 1e-38, "dfeat")
    _close(dtable, r["g"].T @ r["f"], (eg + (n + 8) * EPS * g).T @ r["f"].abs() +
           out * (r["g"].T @ r["f"]).abs() + 1e-38, "dtable")


@pytest.mark.parametrize("n,rows,dim", [
    (1, 1, 1), (1, 1200, 64), (5, 2, 3), (128, 128, 64), (129, 130, 65), (300, 1000, 48),
    (2000, 7, 31), (77, 5000, 100), (257, 9000, 16), (200, 333, 300), (64, 300, 520)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss(ops, n, rows, dim, dtype):
    feat, table, labels, weight = _loss_case(n, rows, dim, dtype, n + rows)
    r = _loss_ref(feat, table, labels, weight, 10.0)
    a = [t.cuda() for t in (feat, table, labels, weight)]
    loss, lse = ops.label_loss(a[0], a[1], a[2], scale=10.0)
    _close(loss, r["loss"], r["e"], "loss")
    _close(lse, r["lse"], r["e"], "lse")
    got = ops.label_loss_grad(*a, scale=10.0)
    _check_loss(r, *got, dtype)
    again = ops.label_loss_grad(a[0], a[1], a[2].int(), a[3], scale=10.0)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_masked_rows_hold_anything(ops, dtype):
    feat, table, labels, weight = _loss_case(400, 150, 40, dtype, 9)
    labels[:150] = -1  # a whole tile without a label
    r = _loss_ref(feat, table, labels, weight, 5.0)
    feat[labels < 0] = float("nan")
    feat[3] = float("inf")
    weight[labels < 0] = float("nan")
    a = [t.cuda() for t in (feat, table, labels, weight)]
    loss, lse, dfeat, dtable = ops.label_loss_grad(*a, scale=5.0)
    _check_loss(r, loss, lse, dfeat, dtable, dtype)
    masked = (labels < 0).cuda()
    assert not loss[masked].any() and not lse[masked].any() and not dfeat[masked].any()
    # no label at all
    none = torch.full_like(a[2], -1)
    loss, lse, dfeat, dtable = ops.label_loss_grad(a[0], a[1], none, a[3])
    assert not loss.any() and not dfeat.any() and not dtable.any()


def test_label_loss_large_scores_and_one_label(ops):
    """Scores of thousands, whose exponentials overflow alone; weights of None."""
    feat, table, labels, _ = _loss_case(200, 500, 32, F32, 10)
    ones = torch.ones(200)
    for scale in (3000.0, -50.0, 0.0):
        r = _loss_ref(feat, table, labels, ones, scale)
        got = ops.label_loss_grad(feat.cuda(), table.cuda(), labels.cuda(), scale=scale)
        _check_loss(r, *got, F32)
    # a table of one row: nothing to learn
    loss, lse, dfeat, dtable = ops.label_loss_grad(feat.cuda(), table[:1].cuda(),
                                                   torch.zeros(200, dtype=torch.int32).cuda())
    assert not loss.any() and not dfeat.any() and not dtable.any()


def test_label_loss_strides_range_and_empty(ops):
    feat, table, labels, weight = _loss_case(150, 60, 33, F32, 11)
    r = _loss_ref(feat, table, labels, weight, 4.0)
    wide = torch.full((150, 50), float("nan"))
    wide[:, 5:38] = feat
    wt = torch.full((60, 41), float("nan"))
    wt[:, 1:34] = table
    df, dt = torch.full((150, 40), 7.0).cuda(), torch.full((60, 40), 7.0).cuda()
    got = ops.label_loss_grad(wide.cuda()[:, 5:38], wt.cuda()[:, 1:34], labels.cuda(),
                              weight.cuda(), scale=4.0, dfeat=df[:, 3:36], dtable=dt[:, 3:36])
    _check_loss(r, *got, F32)
    for t in (df, dt):
        assert (t[:, :3] == 7).all() and (t[:, 36:] == 7).all()
    labels[0] = 60
    loss = ops.label_loss(feat.cuda(), table.cuda(), labels.cuda())[0]
    assert loss[0] == 0
    with pytest.raises(ValueError, match="past"):
        ops.check()
    e = torch.empty(0, 33, device="cuda")
    loss, lse, dfeat, dtable = ops.label_loss_grad(e, table.cuda(), labels[:0].cuda())
    assert loss.shape == (0,) and dfeat.shape == (0, 33) and not dtable.any()


def test_label_loss_in_several_pieces(ops):
    """More table rows and more rows than one piece holds; checked on random rows."""
    feat, table, labels, weight = _loss_case(9000, 17000, 24, BF16, 12)
    loss, lse, dfeat, dtable = (t.cpu().to(D64) for t in ops.label_loss_grad(
        *(t.cuda() for t in (feat, table, labels, weight)), scale=8.0))
    f, t, on = feat.cuda().to(D64), table.cuda().to(D64), labels >= 0
    s = 8.0 * f @ t.T
    w = torch.where(on, weight.to(D64) * 8.0, torch.zeros(1, dtype=D64)).cuda()[:, None]
    want = torch.logsumexp(s, 1)
    at = labels.clamp(min=0).cuda()[:, None]
    tol = 64 * EPS * (8.0 * (f.abs() @ t.abs().T).amax(1) + want.abs() + 1)
    off = torch.where(on.cuda(), (loss.cuda() - (want - s.gather(1, at)[:, 0])).abs(), loss.cuda().abs())
    assert (off <= tol).all()
    g = torch.exp(s - want[:, None])
    g.scatter_add_(1, at, torch.full_like(want, -1.0)[:, None])
    g *= w
    for got, ref, size in ((dfeat, g @ t, g.abs() @ t.abs()),
                           (dtable, g.T @ f, g.abs().T @ f.abs())):
        assert ((got.cuda() - ref).abs() <= 1.05 * BF * (size + ref.abs()) + 1e-30).all()


# ------------------------------------------------------------------ larger sizes
@pytest.mark.parametrize("n,rows,dim,hot", [
    (4000, 3000, 64, 0), (4000, 3000, 64, 0.9), (2_200_003, 5000, 3, 0.3), (700_001, 100, 8, 0.5),
    (200_003, 40_000, 20, 0.7), (1025, 129, 130, 0), (4_300_001, 70_000, 2, 0.2)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lookup_grad_of_long_lists(ops, n, rows, dim, hot, dtype):
    test_lookup_grad(ops, n, rows, dim, hot, dtype)


@pytest.mark.parametrize("bt,pixels,c,groups", [(20, (9, 11), 64, 8), (17, (70, 61), 48, 6),
                                                (2, (131, 257), 12, 4), (33, (5,), 7, 7)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_of_batches(ops, bt, pixels, c, groups, dtype):
    test_group_norm(ops, bt, pixels, c, groups, dtype, "silu")


@pytest.mark.parametrize("n,rows,dim", [(1, 1003, 700), (2, 40_001, 33), (8, 2500, 300),
                                        (8, 70_000, 7), (3, 17, 520), (7, 900, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_of_few(ops, n, rows, dim, dtype):
    feat, table, labels, weight = _loss_case(n, rows, dim, dtype, n + dim)
    r = _loss_ref(feat, table, labels, weight, 10.0)
    loss, lse = ops.label_loss(feat.cuda(), table.cuda(), labels.cuda(), scale=10.0)
    _close(loss, r["loss"], r["e"], "loss")
    _close(lse, r["lse"], r["e"], "lse")


@pytest.mark.parametrize("n,rows,dim", [
    (5000, 3000, 16), (20_000, 600, 45), (600, 20_000, 128), (4099, 2500, 48), (3001, 4097, 64),
    (2000, 2500, 129), (1500, 1601, 260), (9, 30_000, 8), (30_000, 3, 60)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_of_many(ops, n, rows, dim, dtype):
    test_label_loss(ops, n, rows, dim, dtype)


@pytest.mark.parametrize("n,dtype", [(9000, F32), (9000, BF16), (25_000, F32), (70_000, BF16)])
def test_label_loss_of_long_rows_in_several_pieces(ops, n, dtype):
    """More samples and more table rows than one piece of score gradients holds."""
    dim, scale, rows = 130, 8.0, 17_000
    host = _loss_case(n, rows, dim, dtype, 13)
    feat, table, labels, weight = (t.cuda() for t in host)
    got = ops.label_loss_grad(feat, table, labels, weight, scale=scale)
    loss, _, dfeat, dtable = (t.to(D64) for t in got)
    t, out, part = table.to(D64), BF if dtype == BF16 else 0.0, BF if dtype == BF16 else 2.0 ** -22
    want_t, tol_t = torch.zeros_like(t), torch.zeros_like(t)
    for i in range(0, n, 5000):
        at = slice(i, i + 5000)
        f, on, y = feat[at].to(D64), labels[at] >= 0, labels[at].clamp(min=0)[:, None]
        s = scale * f @ t.T
        lse = torch.logsumexp(s, 1)
        e = ((dim + 8) * EPS * scale * (f.abs() @ t.abs().T) + 4 * EPS * s.abs()).amax(1)
        e = 2 * (e + 16 * EPS * (1 + lse.abs() + s.abs().amax(1)))
        want = torch.where(on, lse - s.gather(1, y)[:, 0], torch.zeros_like(lse))
        assert ((loss[at] - want).abs() <= e).all()
        p = torch.exp(s - lse[:, None])
        w = torch.where(on, weight[at].to(D64) * scale, torch.zeros_like(lse))[:, None]
        g = p.scatter_add(1, y, torch.full_like(lse, -1.0)[:, None]) * w
        eg = p.scatter_add(1, y, torch.ones_like(lse)[:, None])  # p + one
        eg = w * (2 * p * e[:, None] + 4 * EPS * eg) + part * g.abs()
        ref = g @ t
        tol = (eg + (rows + 8) * EPS * g.abs()) @ t.abs() + out * ref.abs() + 1e-38
        assert ((dfeat[at] - ref).abs() <= tol).all()
        want_t += g.T @ f
        tol_t += (eg + (n + 8) * EPS * g.abs()).T @ f.abs()
    assert ((dtable - want_t).abs() <= tol_t + out * want_t.abs() + 1e-38).all()


@pytest.mark.parametrize("n,dim", [(3, 16), (100, 16), (100, 200)])
def test_label_loss_of_lowest_scores(ops, n, dim):
    """All scores near the lowest values that fp32 holds: finite, and the table's
    rows equal."""
    feat, table = torch.full((n, dim), -1e18).cuda(), torch.full((50, dim), 1e18).cuda()
    labels = torch.arange(n).cuda() % 50
    loss, lse = ops.label_loss(feat, table, labels)
    want = -float(np.float32(1e18)) ** 2 * dim
    assert ((lse.double() - want).abs() <= (dim + 24) * EPS * abs(want)).all()
    assert (loss.abs() <= (dim + 24) * 2 * EPS * abs(want)).all()


def test_offsets_past_32_bits(ops):
    """Rows 2^20 elements apart, and a table of more than 2^32 elements."""
    far = 1 << 20
    room = torch.empty(3000 * far, dtype=BF16, device="cuda")
    view = room.as_strided((3000, 32), (far, 1))
    feat, table, labels, weight = _loss_case(3000, 40, 32, BF16, 14)
    view.copy_(feat)
    a = (table.cuda(), labels.cuda(), weight.cuda())
    near = ops.label_loss_grad(feat.cuda(), *a, scale=3.0)
    assert all(torch.equal(p, q) for p, q in zip(near, ops.label_loss_grad(view, *a, scale=3.0)))
    ids = _ids(_gen(15), 2000, 3000).cuda()
    assert torch.equal(ops.lookup(view, ids), ops.lookup(feat.cuda(), ids))
    assert torch.equal(ops.lookup_grad(view, a[1], 40), ops.lookup_grad(feat.cuda(), a[1], 40))
    x = room.as_strided((1, 3000, 32), (3000 * far, far, 1))
    one, two = ops.group_norm(x, 4, act="silu"), ops.group_norm(feat.cuda()[None], 4, act="silu")
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    del room, view, x
    rows = (1 << 26) + 3  # of 64
    big = torch.empty(rows, 64, dtype=BF16, device="cuda")
    big[-3000:] = 1.0
    big[-3000:, :32] = feat.cuda()
    at = torch.where(ids < 0, ids, ids + rows - 3000)
    assert torch.equal(ops.lookup(big, at)[:, :32], ops.lookup(feat.cuda(), ids))
    del big
    d = _randn(_gen(16), 2000, 64).cuda()
    out = ops.lookup_grad(d, at, rows)
    want, tol = _grad_ref(d.cpu(), ids.cpu(), 3000, 1.0)
    _close(out[-3000:], want, tol, "dtable")
    assert not out[:-3000].any()


@pytest.mark.parametrize("which", ["feat", "table"])
def test_label_loss_grad_matches_differences(ops, which):
    feat, table, labels, weight = _loss_case(40, 30, 8, F32, 13)
    got = ops.label_loss_grad(*(t.cuda() for t in (feat, table, labels, weight)), scale=3.0)
    grad = got[2 if which == "feat" else 3].cpu().to(D64)
    step = _randn(_gen(14), *grad.shape).to(D64)

    def slope(h):
        v = []
        for sign in (1, -1):
            f, t = feat.to(D64), table.to(D64)
            f, t = (f + sign * h * step, t) if which == "feat" else (f, t + sign * h * step)
            v.append((weight.to(D64) * _loss_ref(f, t, labels, weight, 3.0)["loss"]).sum())
        return (v[0] - v[1]) / (2 * h)

    coarse, fine = slope(2e-3), slope(1e-3)
    tol = (coarse - fine).abs() + 1e-9 + 1000 * EPS * grad.abs().sum() * step.abs().max()
    assert abs((grad * step).sum() - fine) <= tol


# ------------------------------------------------------------------ streams, graphs
def test_operators_on_another_stream_and_in_a_graph(ops):
    """One chain of all operators on a side stream and as a replayed HIP graph whose
    inputs change between replays, against the eager results."""
    g = _gen(15)
    table, ids = _randn(g, 30, 32).cuda(), _ids(g, 600, 30).cuda()
    w, b = (1 + 0.1 * _randn(g, 32)).cuda(), (0.1 * _randn(g, 32)).cuda()
    labels = _ids(g, 600, 30).cuda()

    def chain():
        x = ops.lookup(table, ids, 2.0).view(2, 300, 32)
        y, mean, rstd = ops.group_norm(x, 4, w, b, act="silu")
        loss, _, dy, dt = ops.label_loss_grad(y.view(600, 32), table, labels, scale=2.0)
        dx, dw, db = ops.group_norm_grad(dy.view(2, 300, 32), x, mean, rstd, 4, w, b, act="silu")
        ops.lookup_grad(dx.view(600, 32), ids, 30, 2.0, out=dt, accumulate=True)
        return y, loss, dw, db, dt

    eager = [t.clone() for t in chain()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = chain()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(eager, other))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = chain()
    for k in range(4):
        table.mul_(1.0 + 0.1 * k)
        ids.copy_(torch.roll(ids, 7 * k))
        torch.cuda.synchronize()
        eager = [t.clone() for t in chain()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, held)), k


def test_context_stream(ops):
    """The context's own stream through the C ABI."""
    st = ctypes.c_void_p()
    L._check(ops._L.gs_stream(ops.ctx.handle, ctypes.byref(st)))
    assert st.value
    table, ids = torch.randn(9, 12, device="cuda"), torch.arange(9, device="cuda", dtype=torch.int32)
    out = torch.zeros(9, 12, device="cuda")
    torch.cuda.synchronize()
    L._check(ops._L.gs_lookup_dev(ops.ctx.handle, table.data_ptr(), 9, 12, 0, ids.data_ptr(), 0, 9,
                                  12, 1.0, out.data_ptr(), 12, 0, None, st))
    L._check(ops._L.gs_sync(ops.ctx.handle))
    assert torch.equal(out, table)


# ------------------------------------------------------------------ refusals
def test_refusals(ops):
    t = torch.randn(4, 6, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="is on cpu"):
        ops.lookup(t.cpu(), ids)
    with pytest.raises(TypeError, match="type"):
        ops.lookup(t.half(), ids)
    with pytest.raises(TypeError, match="type"):
        ops.lookup(t, ids.float())
    with pytest.raises(ValueError, match="contiguous"):
        ops.lookup(t.T, ids)
    with pytest.raises(ValueError, match="must be"):
        ops.lookup(t, ids, out=torch.empty(3, 5, device="cuda"))
    with pytest.raises(ValueError, match="scale"):
        ops.lookup(t, ids, float("nan"))
    with pytest.raises(ValueError, match="overlap"):
        ops.lookup(t, ids, out=torch.empty(1, 6, device="cuda").expand(3, 6))
    with pytest.raises(ValueError, match="accumulate"):
        ops.lookup_grad(t[:3], ids, 4, accumulate=True)
    with pytest.raises(ValueError, match="values"):
        ops.lookup_grad(t, ids, 4)
    x = torch.randn(2, 8, 9, 6, device="cuda")
    with pytest.raises(ValueError, match="multiple"):
        ops.group_norm(x, 4)
    with pytest.raises(ValueError, match="act"):
        ops.group_norm(x, 2, act="tanh")
    with pytest.raises(ValueError, match="eps"):
        ops.group_norm(x, 2, eps=0.0)
    with pytest.raises(ValueError, match="one distance"):
        ops.group_norm(x[:, :, 1:5], 2)
    with pytest.raises(TypeError, match="type"):
        ops.group_norm(x, 2, weight=torch.ones(6, device="cuda", dtype=BF16))
    with pytest.raises(ValueError, match="values"):
        ops.group_norm(x, 2, weight=torch.ones(5, device="cuda"))
    y, mean, rstd = ops.group_norm(x, 2)
    with pytest.raises(ValueError, match="dy"):
        ops.group_norm_grad(y[:1], x, mean, rstd, 2)
    with pytest.raises(ValueError, match="mean"):
        ops.group_norm_grad(y, x, mean[:1], rstd, 2)
    with pytest.raises(TypeError, match="feat is"):
        ops.label_loss(t.to(BF16), t, torch.zeros(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="columns"):
        ops.label_loss(t, t[:, :5], torch.zeros(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="scale"):
        ops.label_loss(t, t, torch.zeros(4, dtype=torch.int64, device="cuda"), scale=math.inf)
    with pytest.raises(L.GsError, match="limits"):
        ops.label_loss(t, torch.empty(0, 6, device="cuda"),
                       torch.zeros(4, dtype=torch.int64, device="cuda"))


def test_refusals_of_the_c_abi(ops):
    """Status codes and messages; nothing is enqueued."""
    lib, h = ops._L, ops.ctx.handle
    t = torch.full((8, 8), 5.0, device="cuda")
    ids = torch.zeros(8, dtype=torch.int32, device="cuda")
    p, q = t.data_ptr(), ids.data_ptr()
    ok = [h, p, 4, 8, 0, q, 0, 4, 8, 1.0, p, 8, 0, None, None]

    def lookup(**change):
        a = list(ok)
        for k, v in change.items():
            a[int(k[1:])] = v
        return lib.gs_lookup_dev(*a), lib.gs_last_error().decode()

    for change, code, text in (
            (dict(_0=None), L.GS_E_INVALID, "ctx"), (dict(_1=None), L.GS_E_INVALID, "null"),
            (dict(_2=-1), L.GS_E_INVALID, "negative"), (dict(_2=2 ** 30), L.GS_E_CAPACITY, "past"),
            (dict(_4=7), L.GS_E_INVALID, "dtype"), (dict(_5=q + 2), L.GS_E_INVALID, "aligned"),
            (dict(_6=2), L.GS_E_INVALID, "ids64"), (dict(_8=0), L.GS_E_INVALID, "dim"),
            (dict(_8=2 ** 17), L.GS_E_CAPACITY, "dim"), (dict(_10=p + 2), L.GS_E_INVALID, "aligned"),
            (dict(_11=4), L.GS_E_INVALID, "overlap")):
        rc, msg = lookup(**change)
        assert rc == code and text in msg, (change, rc, msg)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda").data_ptr()
    need = lib.gs_lookup_grad_workspace(4, 4, 8)
    for at, size, text in ((ws, need - 1, "too small"), (ws + 8, need, "256-byte"),
                           (None, need, "256-byte")):
        rc = lib.gs_lookup_grad_dev(h, p, 8, 0, q, 0, 4, 8, 1.0, 0, p + 128, 4, 8, 0, at, size,
                                    None, None)
        assert rc == L.GS_E_INVALID and text in lib.gs_last_error().decode()
    torch.cuda.synchronize()
    assert (t == 5.0).all()

"""The feature operators where sizes, values and use leave the ordinary: closed
contexts, grids past a launch's limits, values that are not finite, means far from
0, long batches, streams, gradients that torch would record.

Tolerances are bounds on fp32 rounding (EPS = 2^-24 a rounding), written down from the
formulas."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS, BF = 2.0 ** -24, 2.0 ** -8
F32, BF16, D64 = torch.float32, torch.bfloat16, torch.float64


@pytest.fixture(scope="module")
def ops():
    from gsplat_tt_amd.field import FieldOps
    o = FieldOps()
    yield o
    o.check()
    o.ctx.close()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------------ use
def test_a_closed_context_is_refused():
    from gsplat_tt_amd.field import FieldOps
    ops = FieldOps()
    table, ids = torch.ones(4, 5, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    x = torch.ones(1, 6, 4, device="cuda")
    y, mean, rstd = ops.group_norm(x, 2)
    ops.ctx.close()
    for call in (lambda: ops.lookup(table, ids),
                 lambda: ops.lookup_grad(table[:3], ids, 4),
                 lambda: ops.group_norm(x, 2),
                 lambda: ops.group_norm_grad(y, x, mean, rstd, 2),
                 lambda: ops.label_loss(table[:3], table, ids),
                 lambda: ops.label_loss_grad(table[:3], table, ids)):
        with pytest.raises(ValueError, match="null ctx"):
            call()


# ------------------------------------------------------------------ sizes
def test_group_norm_of_more_groups_than_a_grid_has_blocks(ops):
    """2^24 groups of 4 values: with 256 threads each, 2^32 threads, past a launch."""
    from tests.test_gpu_field import STEPS, _norm_ref
    g = _gen(1)
    x, dy = (_randn(g, 1 << 20, 1, 64, dtype=BF16) for _ in range(2))
    w, b = 1 + 0.3 * _randn(g, 64), 0.3 * _randn(g, 64)
    r = _norm_ref(x, 16, w, b, "silu", 1e-5, dy)
    y, mean, rstd = ops.group_norm(x, 16, w, b, act="silu")
    assert ((y.to(D64) - r["y"]).abs() <= STEPS * EPS * r["y_size"] + BF * r["y"].abs()).all()
    dx, dw, db = ops.group_norm_grad(dy, x, mean, rstd, 16, w, b, act="silu")
    assert ((dx.to(D64) - r["dx"]).abs() <= STEPS * EPS * r["dx_size"] + BF * r["dx"].abs()).all()
    assert ((dw.to(D64) - r["dw"]).abs() <= STEPS * EPS * r["dw_size"]).all()
    assert ((db.to(D64) - r["db"]).abs() <= STEPS * EPS * r["db_size"]).all()


def test_lookup_of_more_rows_than_a_grid_has_blocks(ops):
    """2^27 rows of odd length and stride, 8 a workgroup."""
    n, dim = 1 << 27, 129
    g = _gen(2)
    table = _randn(g, 7, dim, dtype=BF16)
    ids = torch.randint(-1, 7, (n,), generator=g, device="cuda", dtype=torch.int32)
    room = torch.full((n, dim + 1), 5.0, dtype=BF16, device="cuda")
    ops.lookup(table, ids, 1.0, out=room[:, :dim])
    rows = torch.cat([table, torch.zeros(1, dim, dtype=BF16, device="cuda")])
    for lo in range(0, n, 1 << 23):
        at = slice(lo, lo + (1 << 23))
        assert torch.equal(room[at, :dim], rows[ids[at].long()]), lo  # -1: the last, zeros
        assert (room[at, dim] == 5).all()
    del room, ids
    torch.cuda.empty_cache()


def test_label_loss_of_more_samples_than_a_grid_has_blocks(ops):
    """2^29 samples and some, 32 a workgroup in their layout. A table row's sums run over
    a share's products of 16 samples one after the other: 2^24 tiles of 32 in some hundred
    shares make fewer than 2^18 of them."""
    n, rows, scale = (1 << 29) + 37, 3, 2.0
    g = _gen(3)
    feat, table = _randn(g, n, 1, dtype=BF16), _randn(g, rows, 1, dtype=BF16)
    labels = torch.randint(-1, rows, (n,), generator=g, device="cuda", dtype=torch.int32)
    loss, lse, dfeat, dtable = ops.label_loss_grad(feat, table, labels, scale=scale)
    t, want, size = table.to(D64), torch.zeros(rows, 1, dtype=D64, device="cuda"), 0.0
    step = 1 << 24
    for lo in range(0, n, step):
        at = slice(lo, lo + step)
        f, y = feat[at].to(D64), labels[at].long()
        on, y = y >= 0, y.clamp(min=0)[:, None]
        s = scale * f @ t.T
        log = torch.logsumexp(s, 1)
        one = torch.where(on, log - s.gather(1, y)[:, 0], 0.0)
        assert ((loss[at].to(D64) - one).abs() <= 64 * EPS * (1 + s.abs().amax(1))).all(), lo
        assert ((lse[at].to(D64) - torch.where(on, log, 0.0)).abs() <=
                64 * EPS * (1 + s.abs().amax(1))).all(), lo
        p = torch.exp(s - log[:, None])
        d = p.scatter_add(1, y, torch.full_like(s[:, :1], -1.0)) * scale * on[:, None]
        # the products' left operands and the result are rounded to bf16
        near = 1.05 * BF * (d.abs() @ t.abs() + (d @ t).abs()) + 64 * EPS
        assert ((dfeat[at].to(D64) - d @ t).abs() <= near).all(), lo
        want += d.T @ f
        size += (d.abs().T @ f.abs())
    assert ((dtable.to(D64) - want).abs() <= (BF + 2.0 ** 18 * EPS) * size + BF * want.abs()).all()
    del feat, labels, loss, lse, dfeat
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ group norm's exactness
@pytest.mark.parametrize("pixels,c,groups", [((9, 11), 16, 4), ((200, 111), 64, 2), ((70, 61), 6, 2)])
@pytest.mark.parametrize("act", ["none", "relu"])
def test_group_norm_far_means_cost_no_digits(ops, pixels, c, groups, act):
    """From the statistics as they were returned, y, dx and the parameters' gradients
    carry the roundings of the differences from the mean alone, however far it is: a
    handful a value, and those of sums over a thread's pixels and a tree."""
    g = _gen(c)
    x = _randn(g, 2, *pixels, c) + 3e4 * (1 + torch.rand(c, generator=g, device="cuda") // 0.5)
    per = c // groups
    x = x.view(2, -1, groups, per)
    x = (x - x.mean((1, 3), keepdim=True) + 3e4).view(2, *pixels, c)
    w, b, dy = 1 + 0.3 * _randn(g, c), 0.3 * _randn(g, c), _randn(g, 2, *pixels, c)
    y, mean, rstd = ops.group_norm(x, groups, w, b, act=act)
    dx, dw, db = ops.group_norm_grad(dy, x, mean, rstd, groups, w, b, act=act)
    v = x.to(D64).view(2, -1, groups, per)
    m, r = (t.to(D64).view(2, 1, groups, 1) for t in (mean, rstd))
    w64, b64 = w.to(D64).view(groups, per), b.to(D64).view(groups, per)
    xh = (v - m) * r
    z = xh * w64 + b64
    near = 4 * EPS * ((xh * w64).abs() + z.abs())
    want = z if act == "none" else z.clamp(min=0)
    assert ((y.to(D64).view(v.shape) - want).abs() <= near).all()
    dz = dy.to(D64).view(v.shape) * (1.0 if act == "none" else (z > 0))
    assert act == "none" or not (z.abs() <= near).any()  # no slope is in doubt
    steps = 96 * EPS
    t = dz * w64
    m1, m2 = t.mean((1, 3), keepdim=True), (t * xh).mean((1, 3), keepdim=True)
    a1, a2 = t.abs().mean((1, 3), keepdim=True), (t * xh).abs().mean((1, 3), keepdim=True)
    off = (dx.to(D64).view(v.shape) - r * (t - m1 - xh * m2)).abs()
    assert (off <= steps * r * (t.abs() + a1 + xh.abs() * a2)).all()
    for got, terms in ((dw, dz * xh), (db, dz)):
        off = (got.to(D64).view(groups, per) - terms.sum((0, 1))).abs()
        assert (off <= steps * terms.abs().sum((0, 1))).all()


@pytest.mark.parametrize("pixels,c,groups", [((9, 11), 16, 4), ((200, 111), 64, 2), ((70, 61), 6, 2)])
@pytest.mark.parametrize("value", [1000.0, -77.7, 2e19])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_of_constant_groups(ops, pixels, c, groups, value, dtype):
    """A constant image has its value as the mean, variance 0, and the bias as output."""
    x = torch.full((2, *pixels, c), value, dtype=dtype, device="cuda")
    b = _randn(_gen(4), c)
    y, mean, rstd = ops.group_norm(x, groups, None, b)
    assert (mean == x.flatten()[0].float()).all()
    assert ((rstd.to(D64) - 1e-5 ** -0.5).abs() <= 8 * EPS * 1e-5 ** -0.5).all()
    assert torch.equal(y, b.to(dtype).expand(x.shape))


# ------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("n,dim", [(37, 16), (64, 16), (200, 100), (37, 200)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_of_masked_samples_against_any_table(ops, n, dim, dtype):
    """With no label no table value reaches a result, beside padding too."""
    g = _gen(n * dim)
    feat, table = _randn(g, n, dim, dtype=dtype), _randn(g, 50, dim, dtype=dtype)
    table[3, 0], table[9, 1], table[11] = math.nan, math.inf, -math.inf
    none = torch.full((n,), -1, device="cuda")
    for got in ops.label_loss_grad(feat, table, none, scale=2.0):
        assert not got.any()


@pytest.mark.parametrize("n,dim", [(37, 16), (64, 16), (200, 100), (37, 200)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_row_of_score_minus_infinity_has_no_gradient(ops, n, dim, dtype):
    """One labelled sample among masked ones, whose score of one row is -inf."""
    g = _gen(n * dim)
    feat, none = _randn(g, n, dim, dtype=dtype), torch.full((n,), -1, device="cuda")
    table = _randn(g, 50, dim, dtype=dtype)
    table[11, 0] = -math.inf
    feat[7] = feat[7].abs() + 0.5
    none[7] = 4
    dtable = ops.label_loss_grad(feat, table, none, scale=2.0)[3]
    assert torch.isfinite(dtable).all() and not dtable[11].any() and dtable[4].any()


def _same(got, want, tol):
    """Equal where not finite, within tol elsewhere."""
    got, fine = got.to(D64), torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    there = ~fine & ~torch.isnan(want)
    assert torch.equal(got[there], want[there])
    assert ((got - want).abs() <= tol)[fine].all()


def _loss64(feat, table, labels, scale):
    f, t = feat.to(D64), table.to(D64)
    on, y = labels >= 0, labels.clamp(min=0)[:, None]
    f = torch.where(on[:, None], f, 0.0)  # masked samples hold anything
    s = scale * (f @ t.T)
    log = torch.logsumexp(s, 1)
    loss = torch.where(on, log - s.gather(1, y)[:, 0], 0.0)
    p = torch.exp(s - log[:, None])
    d = torch.where(on[:, None], p.scatter_add(1, y, torch.full_like(s[:, :1], -1.0)) * scale, 0.0)
    return loss, torch.where(on, log, 0.0), d, s


@pytest.mark.parametrize("n,rows,dim", [(5, 40, 16), (101, 70, 16), (77, 300, 48), (300, 40, 100),
                                        (45, 200, 130), (200, 140, 300)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_of_infinite_values(ops, n, rows, dim, dtype):
    """Infinite table values and features give the scores that arithmetic gives: a row
    of score -inf drops out, +inf and NaN show."""
    g = _gen(n + dim)
    feat, table = _randn(g, n, dim).abs().to(dtype) + 0.25, _randn(g, rows, dim, dtype=dtype)
    labels = torch.randint(-1, rows, (n,), generator=g, device="cuda")
    labels[0] = -1  # masked
    labels[1:3] = 0
    labels = torch.where(labels == 5, 6, labels)
    scale = 0.5
    table[5, dim // 2] = -math.inf
    table[5, 1] = -math.inf
    loss, log, d, s = _loss64(feat, table, labels, scale)
    assert torch.isfinite(loss).all() and (s[labels >= 0, 5] == -math.inf).all()
    finite = torch.where(torch.isfinite(s), s, 0.0).abs()
    size = scale * (feat.to(D64).abs() @ torch.where(torch.isinf(table), 0, table).to(D64).abs().T)
    near = ((dim + 32) * EPS * size.amax(1) + 32 * EPS * (1 + finite.amax(1)))
    a = ops.label_loss(feat, table, labels, scale=scale)
    b = ops.label_loss_grad(feat, table, labels, scale=scale)
    for got in (a, b):
        _same(got[0], loss, 2 * near)
        _same(got[1], log, 2 * near)
    # gradients: the dropped row gets none; dfeat is not a number in the infinite columns
    part = BF if dtype == BF16 else 2.0 ** -22
    f = torch.where((labels >= 0)[:, None], feat, 0).to(D64)
    t = torch.where(torch.isinf(table), 0, table).to(D64)
    e = part + 2 * near[:, None] + (n + rows + 32) * EPS
    tol = ((d.abs() * e + e * torch.exp(s - log[:, None]).nan_to_num(0.0) * scale))
    _same(b[3], d.T @ f, tol.T @ f + BF * (d.T @ f).abs() * (dtype == BF16) + 1e-30)
    want = d @ t
    want[:, [1, dim // 2]] = math.nan
    want[labels < 0] = 0.0
    _same(b[2], want, tol @ t.abs() + BF * want.abs().nan_to_num(0.0) * (dtype == BF16) + 1e-30)
    # features: +inf and -inf scores of one sample, and both infinite
    feat[2, 3], feat[1, 1], feat[0, 0] = math.inf, math.inf, math.nan
    table[:, 3] = table[:, 3].abs() + 0.25
    table[[0, 5, 7], 3] = -1.0
    loss, log, d, s = _loss64(feat, table, labels, scale)
    assert torch.isinf(log[2]) and (s[2] == -math.inf).any() and torch.isinf(loss[2])
    finite = torch.where(torch.isfinite(s), s, 0.0).abs()
    size = scale * (torch.where(torch.isfinite(feat), feat, 0).to(D64).abs() @ t.abs().T)
    near = ((dim + 32) * EPS * (size.amax(1) + 1) + 32 * EPS * (1 + finite.amax(1)))
    for got in (ops.label_loss(feat, table, labels, scale=scale),
                ops.label_loss_grad(feat, table, labels, scale=scale)):
        _same(got[0], loss, 2 * near)
        _same(got[1], log, 2 * near)


@pytest.mark.parametrize("pixels", [1, 3000])
def test_gelu_keeps_its_digits(ops, pixels):
    """gelu and its slope over the line, in one launch and in three. z comes from the
    bias alone (x is constant). Phi(-|z|) = exp(-z^2 / 2) R: the exponent's rounding
    moves the exponential by z^2 EPS, exponential, quotient, polynomial and products
    take 16 EPS, and the polynomial's own error 4 EPS."""
    c = 4096
    z = torch.linspace(-9.0, 9.0, c, device="cuda")
    x, dy = torch.zeros(1, pixels, c, device="cuda"), torch.zeros(1, pixels, c, device="cuda")
    dy[:, 0] = 1.0
    y, mean, rstd = ops.group_norm(x, 1, None, z, act="gelu")
    _, _, db = ops.group_norm_grad(dy, x, mean, rstd, 1, None, z, act="gelu")
    z = z.to(D64)
    phi = 0.5 * torch.erfc(-z / math.sqrt(2))
    tail = 0.5 * torch.erfc(z.abs() / math.sqrt(2))
    off = (20 + z * z) * EPS * tail + 2 * EPS * phi  # of Phi
    assert ((y.to(D64)[0, 0] - z * phi).abs() <= z.abs() * off + EPS * (z * phi).abs()).all()
    bell = z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    assert ((db.to(D64) - (phi + bell)).abs() <= off + (8 + z * z) * EPS * bell.abs() +
            2 * EPS * (phi + bell).abs()).all()


@pytest.mark.parametrize("batch,pixels,c", [(65_000, 4, 16), (1 << 18, 1, 64), (70_001, 3, 5),
                                            (3000, 40, 300)])
def test_group_norm_grad_of_long_batches(ops, batch, pixels, c):
    """The parameters' gradients of many images: sums in a tree, whose error grows by a
    rounding a level and not by one an image. A constant gradient rounds the same way at
    every step of a long chain."""
    g = _gen(batch)
    x = _randn(g, batch, pixels, c)
    dy = torch.full_like(x, 1.1)
    y, mean, rstd = ops.group_norm(x, 1)
    _, dw, db = ops.group_norm_grad(dy, x, mean, rstd, 1)
    d = float(dy.flatten()[0])
    steps = 64 * EPS  # 40 in a row and 24 joined at most
    total = batch * pixels * d
    assert ((db.to(D64) - total).abs() <= steps * total).all()
    xh = (x.to(D64) - mean.to(D64)[:, :, None]) * rstd.to(D64)[:, :, None]
    assert ((dw.to(D64) - (xh * d).sum((0, 1))).abs() <= steps * (xh.abs() * d).sum((0, 1))).all()


def test_inputs_that_record_a_gradient_are_refused(ops):
    """The operators are not part of torch's graph: in grad mode a tensor that requires a
    gradient is an error, not a constant. Given outputs count as written in place."""
    table = torch.randn(6, 4, device="cuda", requires_grad=True)
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    x = torch.randn(1, 6, 4, device="cuda")
    w = torch.ones(4, device="cuda", requires_grad=True)
    y, mean, rstd = ops.group_norm(x, 2)
    for call in (lambda: ops.lookup(table, ids),
                 lambda: ops.lookup(table.detach(), ids, out=table[:3]),
                 lambda: ops.lookup_grad(table[:3], ids, 4),
                 lambda: ops.group_norm(x, 2, w),
                 lambda: ops.group_norm(x, 2, None, w),
                 lambda: ops.group_norm_grad(y, x, mean, rstd, 2, w),
                 lambda: ops.label_loss(table[:3], table.detach(), ids),
                 lambda: ops.label_loss_grad(table[:3].detach(), table, ids)):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
    with torch.no_grad():
        a = ops.lookup(table, ids)
    assert torch.equal(a, ops.lookup(table.detach(), ids)) and torch.equal(a, table.detach()[ids])
    out = torch.zeros(3, 4, device="cuda")
    for call in (lambda: ops.lookup(table.detach(), ids, out=out),
                 lambda: ops.lookup_grad(a, ids, 3, out=out),
                 lambda: ops.group_norm(out.view(1, 3, 4), 2, out=out.view(1, 3, 4)),
                 lambda: ops.label_loss_grad(a, table.detach(), ids, dfeat=out)):
        before = out._version
        call()
        assert out._version > before


def test_check_waits_for_every_stream(ops):
    """A report of a call that still waits on another stream is not missed."""
    table = torch.ones(4, 5, device="cuda")
    ids = torch.tensor([0, 9], device="cuda")
    ops.lookup(table, ids[:1])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second or so
        ops.lookup(table, ids)
    with pytest.raises(ValueError, match="past"):
        ops.check()
    ops.check()


def test_lookup_grad_without_rows_reports_ids(ops):
    """Into a table without rows every id is past it; masked ones are not reported."""
    dout = torch.ones(700, 5, device="cuda")
    ids = torch.full((700,), -1, device="cuda")
    assert ops.lookup_grad(dout, ids, 0).shape == (0, 5)
    ops.check()
    ids[-1] = 0
    ops.lookup_grad(dout, ids.int(), 0)
    with pytest.raises(ValueError, match="past"):
        ops.check()


def test_lookup_grad_of_few_ids_into_a_large_table(ops):
    """Clearing what belongs to the table's rows is the whole chip's work: it costs about
    as much as filling the table, not one workgroup's time."""
    n, rows = 5000, (1 << 27) + 1
    g = _gen(5)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    dout, out = _randn(g, n, 2), torch.empty(rows, 2, device="cuda")

    def best(call):
        times = []
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    took = best(lambda: ops.lookup_grad(dout, ids, rows, out=out))
    assert took <= 10 * best(lambda: out.zero_()) + 1.0
    ops.lookup_grad(dout, ids, rows, out=out)
    want = torch.zeros(rows, 2, device="cuda").index_add_(0, ids, dout)
    assert ((out - want).abs() <= 4 * EPS * want.abs() + 1e-6).all()
    del out, want
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ pieces that add up in place
@pytest.mark.parametrize("n,rows,dim,dtype", [(19_501, 20_000, 768, F32),
                                              (30_011, 32_003, 512, BF16)])
def test_label_loss_pieces_add_up_without_slices(ops, n, rows, dim, dtype):
    """Several pieces whose sums have one share: they go straight onto the earlier
    pieces' sums, of the table and (fp32) of the samples too."""
    scale, g = 8.0, _gen(6)
    out, part = (BF, BF) if dtype == BF16 else (0.0, 2.0 ** -22)
    table = _randn(g, rows, dim)
    table /= table.norm(dim=1, keepdim=True)
    labels = torch.randint(-1, rows, (n,), generator=g, device="cuda")
    feat = (_randn(g, n, dim) / math.sqrt(dim) + 0.5 * table[labels.clamp(min=0)]).to(dtype)
    table = table.to(dtype)
    got = ops.label_loss_grad(feat, table, labels, scale=scale)
    loss, _, dfeat, dtable = (t.to(D64) for t in got)
    t = table.to(D64)
    want_t, tol_t = torch.zeros_like(t), torch.zeros_like(t)
    for i in range(0, n, 4000):
        at = slice(i, i + 4000)
        f, on, y = feat[at].to(D64), labels[at] >= 0, labels[at].clamp(min=0)[:, None]
        s = scale * f @ t.T
        log = torch.logsumexp(s, 1)
        e = ((dim + 8) * EPS * scale * (f.abs() @ t.abs().T) + 4 * EPS * s.abs()).amax(1)
        e = 2 * (e + 16 * EPS * (1 + log.abs() + s.abs().amax(1)))
        want = torch.where(on, log - s.gather(1, y)[:, 0], 0.0)
        assert ((loss[at] - want).abs() <= e).all()
        p = torch.exp(s - log[:, None])
        w = torch.where(on, scale, 0.0)[:, None].to(D64)
        d = p.scatter_add(1, y, torch.full_like(log, -1.0)[:, None]) * w
        ed = p.scatter_add(1, y, torch.ones_like(log)[:, None])
        ed = w * (2 * p * e[:, None] + 4 * EPS * ed) + part * d.abs()
        ref = d @ t
        tol = (ed + (rows + 8) * EPS * d.abs()) @ t.abs() + out * ref.abs() + 1e-38
        assert ((dfeat[at] - ref).abs() <= tol).all()
        want_t += d.T @ f
        tol_t += (ed + (n + 8) * EPS * d.abs()).T @ f.abs()
    assert ((dtable - want_t).abs() <= tol_t + out * want_t.abs() + 1e-38).all()

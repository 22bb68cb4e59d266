"""The global norm of many tensors and clipping against plain 64-bit formulas: types,
sizes, strides, values that are not finite, lists of one to thousands, streams, graphs,
refusals.

Tolerances are bounds on rounding: EPS = 2^-24 is fp32's, BF = 2^-8 bf16's, half a step
relative to the value."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS, BF = torch.finfo(torch.float32).eps / 2, torch.finfo(torch.bfloat16).eps / 2
F32, BF16, D64 = torch.float32, torch.bfloat16, torch.float64


@pytest.fixture(scope="module")
def ops():
    from gsplat_tt_amd.field import FieldOps
    o = FieldOps()
    yield o
    o.check()
    o.ctx.close()


def _list(shapes, dtypes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * 10.0 ** (k % 5 - 3)).to(dtypes[k % len(dtypes)])
            for k, s in enumerate(shapes)]


def _norm(ts, kind):
    vs = [t.to(D64).flatten() for t in ts if t.numel()]
    if not vs:
        return 0.0
    v = torch.cat(vs)
    return float(v.square().sum().sqrt() if kind == "l2" else v.abs().max())


def _norm_is(got, ts, kind):
    assert got.shape == () and got.dtype == F32
    want = _norm([t.cpu() for t in ts], kind)
    # the squares' sum in 64 bits (2^-53 a term), its root rounded once
    assert abs(float(got) - want) <= (0 if kind == "max" else 1.001 * EPS * want), (float(got), want)
    return want


SHAPES = {"one value": [(1,)], "scalar": [()], "small": [(7, 32), (32,), (3, 5, 2)],
          "empty ones": [(0,), (5,), (3, 0), (2, 2)], "nothing": [(0, 4)], "no tensors": [],
          "odd": [(4095,), (4096,), (4097,), (1, 3), (65537,), (12289,)],
          "scene": [(3001, 3), (3001, 3), (3001, 4), (3001,), (3001, 16, 3)],
          "large": [(3_000_017,), (5,), (777, 1001)],
          "many": [(1 + 37 * k % 101,) for k in range(700)]}


@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F32, BF16, BF16)])
@pytest.mark.parametrize("kind", ["l2", "max"])
def test_norm_and_clip(ops, name, dtypes, kind):
    ts = _list(SHAPES[name], dtypes)
    dev = [t.cuda() for t in ts]
    got = ops.grad_norm(dev, kind=kind)
    want = _norm_is(got, ts, kind)
    for share in (0.3, 2.0):
        limit = share * want
        factor = min(1.0, limit / (want + 1e-6))
        for out_types in ((F32,), (BF16, F32)):
            outs = [torch.full(t.shape, 9.0, dtype=out_types[k % len(out_types)], device="cuda")
                    for k, t in enumerate(ts)]
            n = ops.clip_grads(dev, limit, kind=kind, out=outs)
            assert torch.equal(n, got)
            for t, d, o in zip(ts, dev, outs):
                v = t.to(D64) * factor
                # norm, factor and product are rounded once each
                tol = 4 * EPS * v.abs() + (BF * v.abs() * 1.01 if o.dtype == BF16 else 0) + 1e-44
                assert ((o.cpu().to(D64) - v).abs() <= tol).all()
                assert torch.equal(d.cpu(), t)  # the inputs stay
        place = [t.clone() for t in dev]
        n = ops.clip_grads(place, limit, kind=kind)
        assert torch.equal(n, got)
        for t, p in zip(ts, place):
            if share > 1:
                assert torch.equal(p.cpu(), t)
            v = t.to(D64) * factor
            tol = 4 * EPS * v.abs() + (BF * v.abs() * 1.01 if p.dtype == BF16 else 0) + 1e-44
            assert ((p.cpu().to(D64) - v).abs() <= tol).all()


def test_sizes_of_values(ops):
    """Squares past fp32's range and below it."""
    for size in (1e-40, 3e-39, 1e-25, 1e25, 3e38):
        t = torch.full((1000,), size, device="cuda")
        got = float(ops.grad_norm([t]))
        # values as they are held
        want = float(t[0].double()) * math.sqrt(1000)
        if want < 3.4e38:
            assert abs(got - want) <= 1.001 * EPS * want + 1e-45
        else:
            assert got == math.inf
    mixed = [torch.tensor([1e20, 1e-20], device="cuda"), torch.tensor([3e-30], device="cuda")]
    assert float(ops.grad_norm(mixed)) == float(torch.tensor(1e20))


@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_that_are_not_finite(ops, kind, dtype):
    g = torch.randn(5000, generator=torch.Generator().manual_seed(1)).to(dtype)
    for at in (0, 3, 4999):
        bad = g.clone()
        bad[at] = float("nan")
        dev = [g.cuda(), bad.cuda()]
        assert ops.clip_grads(dev, 1.0, kind=kind).isnan()
        assert all(t.isnan().all() for t in dev)
        bad[at] = -float("inf")
        dev = [g.cuda(), bad.cuda()]
        assert float(ops.clip_grads(dev, 1.0, kind=kind)) == math.inf
        assert not dev[0].any()
        assert dev[1][at].isnan() and int(dev[1].isnan().sum()) == 1
    zeros = [torch.zeros(10, dtype=dtype, device="cuda")]
    assert float(ops.clip_grads(zeros, 0.0, kind=kind)) == 0.0 and not zeros[0].any()
    one = [torch.ones(10, dtype=dtype, device="cuda")]
    ops.clip_grads(one, 0.0, kind=kind)
    assert not one[0].any()
    one = [torch.ones(10, dtype=dtype, device="cuda")]
    ops.clip_grads(one, math.inf, kind=kind)
    assert (one[0] == 1).all()


def test_strides(ops):
    base = torch.randn(60, 50, generator=torch.Generator().manual_seed(2))
    views = {"columns": lambda t: t[:, 3:20], "one column": lambda t: t[:, 7], "rows": lambda t: t[::3],
             "transposed": lambda t: t.T, "transposed columns": lambda t: t[:, 1:9].T,
             "three": lambda t: t.view(60, 10, 5).permute(2, 0, 1), "offset": lambda t: t.view(-1)[1:1002],
             "every second": lambda t: t[:, ::2], "one row": lambda t: t[4:5, 2:9]}
    for dtype in (F32, BF16):
        for name, view in views.items():
            big = base.to(dtype).cuda()
            t = view(big)
            want = _norm_is(ops.grad_norm([t, t]), [t, t], "l2")
            limit, keep = 0.5 * want, big.clone()
            factor = limit / (want + 1e-6)
            v = t.cpu().to(D64) * factor
            tol = 4 * EPS * v.abs() + (BF * v.abs() * 1.01 if dtype == BF16 else 0)
            room = torch.full_like(big, 5.0, dtype=F32)
            ops.clip_grads([t], limit / math.sqrt(2), out=[view(room)])
            # of one of the two: its norm is 1 / sqrt(2) of theirs
            assert ((view(room).cpu().to(D64) - v).abs() <= 4 * EPS * v.abs() + 1e-6 * v.abs()).all(), name
            view(room).fill_(5.0)
            assert (room == 5).all(), name
            whole = torch.full(t.shape, 5.0, device="cuda") if t.is_contiguous() or name in (
                "columns", "one column", "rows", "every second", "one row") else None
            if whole is not None:
                ops.clip_grads([t], limit, out=[whole], norm=torch.tensor(want, device="cuda"))
                assert ((whole.cpu().to(D64) - v).abs() <= 4 * EPS * v.abs()).all(), name
            ops.clip_grads([t], limit, norm=torch.tensor(want, device="cuda"))
            assert ((t.cpu().to(D64) - v).abs() <= tol).all(), name
            t.copy_(view(keep))
            assert torch.equal(big, keep), name
    # a row for all (an input alone), and columns of one matrix as outputs of their own
    row = torch.randn(1, 40, device="cuda").expand(30, 40)
    _norm_is(ops.grad_norm([row]), [row], "l2")
    big = base.cuda()
    parts = [big[:, :10], big[:, 10:30], big[:, 30:]]
    want = big.clone()
    n = ops.clip_grads(parts, 1.0)
    assert ((big - want / (n + 1e-6)).abs() <= 4 * EPS * want.abs()).all()


def test_norm_given(ops):
    t = torch.ones(100, device="cuda")
    norm = torch.tensor(40.0, device="cuda")
    got = ops.clip_grads([t], 10.0, norm=norm)
    assert got is norm
    assert (t - 0.25).abs().max() <= 2 * EPS
    ops.clip_grads([t], 10.0, norm=torch.tensor([[1.0]], device="cuda"))
    assert (t - 0.25).abs().max() <= 2 * EPS


def test_parameters_and_inference_tensors(ops):
    """Tensors that are parameters, or made under inference_mode, among others; versions of
    what is written are counted."""
    p = torch.nn.Parameter(torch.ones(30, device="cuda"))
    with torch.inference_mode():
        i = torch.ones(20, device="cuda")
    t = torch.ones(50, device="cuda")
    version = t._version
    with torch.no_grad():
        n = ops.clip_grads([p, i, t], 1.0)
    assert abs(float(n) - 10.0) <= 1e-6 and t._version == version + 1
    for x in (p, i, t):
        assert (x.detach() - 0.1).abs().max() <= 4 * EPS
    with pytest.raises(ValueError, match="requires a gradient"):
        ops.grad_norm([p])
    n = ops.grad_norm(x.detach() for x in (p, t))  # any iterable
    assert abs(float(n) - 80 ** 0.5 / 10) <= 1e-6


def test_results_do_not_change_from_run_to_run(ops):
    ts = [torch.randn(n, device="cuda") for n in (5_000_011, 3, 100_003)]
    first = ops.grad_norm(ts)
    assert all(torch.equal(ops.grad_norm(ts), first) for _ in range(5))


@pytest.mark.parametrize("shapes", ["small", "scene", "many"])
def test_captured_and_replayed(ops, shapes):
    sets = [[t.cuda() for t in _list(SHAPES[shapes], (F32, BF16), seed=s)] for s in range(3)]
    bufs = [t.clone() for t in sets[0]]
    outs = [torch.empty(t.shape, device="cuda") for t in bufs]
    ops.clip_grads(bufs, 0.5, out=outs)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norm = ops.clip_grads(bufs, 0.5, out=outs)
        graphs.append((g, norm))
    for k in (0, 1, 2, 1):
        for b, t in zip(bufs, sets[k]):
            b.copy_(t)
        want = ops.clip_grads(bufs, 0.5, out=outs).clone()
        eager = [o.clone() for o in outs]
        for g, norm in graphs:
            for o in outs:
                o.fill_(3.0)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(norm, want)
            assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_streams(ops):
    jobs = [[torch.randn(300_000 + k, device="cuda") for _ in range(3)] for k in range(2)]
    want = [ops.grad_norm(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for _ in range(3):
        for j, s in zip(jobs, streams):
            with torch.cuda.stream(s):
                got.append(ops.grad_norm(j))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[k % 2]) for k, g in enumerate(got))


def test_refusals(ops):
    t = torch.ones(4, 6, device="cuda")
    with pytest.raises(TypeError, match="type"):
        ops.grad_norm([t, t.half()])
    with pytest.raises(TypeError, match="tensor"):
        ops.grad_norm([t, None])
    with pytest.raises(ValueError, match="is on"):
        ops.grad_norm([t.cpu()])
    with pytest.raises(ValueError, match="kind"):
        ops.grad_norm([t], kind="l1")
    with pytest.raises(ValueError, match="requires a gradient"):
        ops.grad_norm([t.clone().requires_grad_()])
    big = torch.ones(4, 5, 6, device="cuda")
    with pytest.raises(ValueError, match="distance"):
        ops.grad_norm([big[:, :2, :3]])
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            ops.clip_grads([t], bad)
    with pytest.raises(ValueError, match="tensors"):
        ops.clip_grads([t], 1.0, out=[])
    with pytest.raises(ValueError, match="must be"):
        ops.clip_grads([t], 1.0, out=[t.view(6, 4)])
    with pytest.raises(ValueError, match="order"):
        ops.clip_grads([t.T], 1.0, out=[torch.empty(6, 4, device="cuda")])
    with pytest.raises(ValueError, match="one value"):
        ops.clip_grads([t], 1.0, norm=torch.ones(2, device="cuda"))
    with pytest.raises(TypeError, match="norm"):
        ops.clip_grads([t], 1.0, norm=torch.ones(1, device="cuda", dtype=BF16))
    # what would be written twice, or read and written
    room = torch.ones(100, device="cuda")
    for ins, outs in (([t, t], None), ([room[:60], room[50:]], None),
                      ([room[:50], room[50:]], [room[50:], room[:50]]),
                      ([room[:40]], [room[1:41]]), ([t], [t[:1].expand(4, 6)]),
                      ([room[:4].expand(5, 4)], None), ([room[:50], room[50:]], [room[:50], room[:50]]),
                      ([room[:40]], [room.view(BF16)[:40]])):
        before = room.clone()
        with pytest.raises(ValueError, match="shares memory|overlap"):
            ops.clip_grads(ins, 1e-3, out=outs, norm=torch.ones((), device="cuda"))
        torch.cuda.synchronize()
        assert torch.equal(room, before) and (t == 1).all()
    with pytest.raises(ValueError, match="shares memory"):
        ops.clip_grads([room], 1e-3, norm=room[3])
    same = [t, t]  # the norm alone may name a tensor twice
    assert abs(float(ops.grad_norm(same)) - math.sqrt(48)) <= 1e-6


def test_c_boundary(ops):
    from gsplat_tt_amd import _lib as L
    lib, h = ops._L, ops.ctx.handle
    t = torch.ones(1 << 16, device="cuda")
    one = (L.GsTensor * 1)(L.GsTensor(t.data_ptr(), 1, t.numel(), 0, 0, 0))
    at = ctypes.addressof(one)
    size = lib.gs_grad_norm_workspace(at, 1)
    ws = torch.empty(size + 256, dtype=torch.uint8, device="cuda")
    norm = torch.zeros(1, device="cuda")
    st = ops._stream()
    assert lib.gs_grad_norm_dev(h, at, 1, 0, norm.data_ptr(), ws.data_ptr(), size, st) == 0
    assert float(norm) == 256.0
    for args in ((at, 1, 2, norm.data_ptr(), ws.data_ptr(), size), (at, -1, 0, norm.data_ptr(), ws.data_ptr(), size),
                 (None, 1, 0, norm.data_ptr(), ws.data_ptr(), size), (at, 1, 0, None, ws.data_ptr(), size),
                 (at, 1, 0, norm.data_ptr(), ws.data_ptr(), size - 1),
                 (at, 1, 0, norm.data_ptr(), ws.data_ptr() + 8, size)):
        assert lib.gs_grad_norm_dev(h, *args, st) == L.GS_E_INVALID
    assert lib.gs_grad_clip_dev(h, at, at, 1, -1, norm.data_ptr(), -1.0, None, 0, st) == L.GS_E_INVALID
    assert lib.gs_grad_clip_dev(h, at, at, 1, -1, None, 1.0, None, 0, st) == L.GS_E_INVALID
    two = (L.GsTensor * 1)(L.GsTensor(t.data_ptr(), 2, t.numel(), 5, 0, 0))
    assert lib.gs_grad_clip_dev(h, at, ctypes.addressof(two), 1, -1, norm.data_ptr(), 1.0,
                                None, 0, st) == L.GS_E_INVALID

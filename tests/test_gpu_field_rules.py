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

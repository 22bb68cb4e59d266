"""The label head with a hidden layer and clipped gradients: lookup, norm, gated
projections, label loss and clipping together, against autograd in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D64 = torch.float64


def _reference(head, images, view_ids, labels):
    p = {k: v.cpu().to(D64).requires_grad_() for k, v in head.params.items()}
    x = images.cpu().to(D64)
    x = x + p["appearance"][view_ids.cpu().long()].view(x.shape)
    c = x.shape[-1]
    y = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), head.GROUPS, p["weight"], p["bias"])
    y = torch.nn.functional.silu(y).permute(0, 2, 3, 1).reshape(-1, c)
    gate = y @ p["w_gate"].T + p["b_gate"]
    y = gate * torch.sigmoid(gate) * (y @ p["w_up"].T + p["b_up"])
    loss = torch.nn.functional.cross_entropy(head.SCALE * y @ p["table"].T, labels.cpu().long(),
                                             ignore_index=-1)
    loss.backward()
    return loss.detach(), {k: t.grad for k, t in p.items()}


def _case():
    from gsplat_tt_amd.field import FieldOps
    from gsplat_tt_amd.label_head import LabelHead
    ops = FieldOps()
    g = torch.Generator().manual_seed(3)
    views, h, w, c = 3, 21, 34, 24
    images = torch.randn(views, h, w, c, generator=g).cuda()
    labels = torch.randint(-1, 6, (views * h * w,), generator=g).cuda()
    view_ids = torch.arange(views, device="cuda", dtype=torch.int32).repeat_interleave(h * w)
    head = LabelHead(ops, c, 6, views, hidden=40)
    head.params["appearance"] += 0.1 * torch.arange(views, device="cuda")[:, None]
    head.params["b_gate"] += 0.1
    return ops, head, (images, view_ids, labels)


def test_gradients():
    ops, head, batch = _case()
    loss, grads = head.gradients(*batch)
    want, ref = _reference(head, *batch)
    assert set(grads) == set(ref) == set(head.params)
    # fp32 against 64 bits: some 1e3 roundings of 6e-8 on the way of each value
    assert abs(float(loss) - float(want)) <= 1e-4 * abs(float(want))
    for k, g in grads.items():
        size = ref[k].abs().max()
        assert (g.cpu().to(D64) - ref[k]).abs().max() <= 1e-4 * size + 1e-7, k
    # along a direction, against differences of the loss in 64 bits
    g = torch.Generator().manual_seed(4)
    step = {k: torch.randn(v.shape, generator=g, dtype=D64) for k, v in ref.items()}
    slope = sum((grads[k].cpu().to(D64) * s).sum() for k, s in step.items())
    keep = {k: v.clone() for k, v in head.params.items()}
    values, h = [], 1e-4
    for sign in (1, -1):
        head.params = {k: v.to(D64) + sign * h * step[k].cuda() for k, v in keep.items()}
        values.append(float(_reference(head, *batch)[0]))
    # fp32 gradients as above, truncation of order h^2
    size = sum((ref[k].abs() * s.abs()).sum() for k, s in step.items())
    assert abs(slope - (values[0] - values[1]) / (2 * h)) <= 1e-4 * size + 1e-4
    ops.ctx.close()


def test_steps_with_clipped_gradients():
    """A step takes the gradients scaled to the limit: with an Adam that starts at 0 the
    first step is the gradient's sign, whatever its size, so the moments are compared."""
    ops, head, batch = _case()
    _, grads = head.gradients(*batch)
    total = float(torch.cat([g.flatten().double() for g in grads.values()]).norm())
    for limit in (0.01 * total, 2 * total):
        ops2, other, _ = _case()
        other.step(*batch, max_norm=limit)
        factor = min(1.0, limit / (total + 1e-6))
        for k, g in grads.items():
            want = g.double() * factor * (1 - 0.9)
            # the norm, the factor, the product, lerp's weight and product
            assert (other._moments[k][0].double() - want).abs().max() <= \
                10 * 2.0 ** -24 * want.abs().max(), k
        ops2.ctx.close()
    first = float(head.step(*batch, max_norm=1.0))
    for _ in range(3):
        loss = head.step(*batch, max_norm=1.0)
    assert loss.isfinite() and first > 0
    per_pixel = head.loss(*batch)
    assert not per_pixel[batch[2] < 0].any() and per_pixel.isfinite().all()
    ops.check()
    ops.ctx.close()


def test_command_with_a_hidden_layer(capsys):
    from gsplat_tt_amd import label_head
    label_head.main(["--gaussians", "3000", "--steps", "3", "--hidden", "32", "--clip", "1.0"])
    assert "labelled pixels" in capsys.readouterr().out

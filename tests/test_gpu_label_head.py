"""The operators together: the label head's gradients against autograd in 64 bits,
and a short training run on rendered features."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D64 = torch.float64


def _reference(head, images, view_ids, labels):
    p = {k: v.cpu().to(D64).requires_grad_() for k, v in head.params.items()}
    x = images.cpu().to(D64)
    x = x + p["appearance"][view_ids.cpu().long()].view(x.shape)
    v, h, w, c = x.shape
    y = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), head.GROUPS, p["weight"], p["bias"])
    y = torch.nn.functional.silu(y).permute(0, 2, 3, 1).reshape(-1, c)
    loss = torch.nn.functional.cross_entropy(head.SCALE * y @ p["table"].T, labels.cpu().long(),
                                             ignore_index=-1)
    loss.backward()
    return loss.detach(), {k: t.grad for k, t in p.items()}


def test_label_head_gradients_and_training():
    from gsplat_tt_amd.field import FieldOps
    from gsplat_tt_amd.label_head import LabelHead, synthetic
    ops = FieldOps()
    images, view_ids, labels = synthetic(ops, gaussians=5000, views=3, height=45, width=62)
    assert images.shape == (3, 45, 62, 24) and torch.isfinite(images).all()
    assert 0 < int((labels < 0).sum()) < labels.numel() // 2
    head = LabelHead(ops, 24, 6, 3)
    head.params["appearance"] += 0.1 * torch.arange(3, device="cuda")[:, None]
    loss, grads = head.gradients(images, view_ids, labels)
    want, ref = _reference(head, images, view_ids, labels)
    # fp32 against 64 bits: some 1e3 roundings of 6e-8 on the way of each value
    assert abs(float(loss) - float(want)) <= 1e-4 * abs(float(want))
    for k, g in grads.items():
        size = ref[k].abs().max()
        assert (g.cpu().to(D64) - ref[k]).abs().max() <= 1e-4 * size + 1e-7, k
    first = float(head.step(images, view_ids, labels))
    for _ in range(30):
        last = float(head.step(images, view_ids, labels))
    assert last < 0.7 * first
    per_pixel = head.loss(images, view_ids, labels)
    assert not per_pixel[labels < 0].any()
    ops.check()
    ops.ctx.close()

"""A label head on rendered features: the feature operators used together.

    python -m gsplat_tt_amd.label_head [--gaussians N] [--steps K]

A synthetic scene's Gaussians carry codes into a codebook of feature rows
(`lookup`), which the rasterizer renders three channels at a time into feature
images. `LabelHead` adds a learned appearance row per view (`lookup` again), runs
a group norm with silu, and scores every pixel against a table of label rows
(`label_loss`). A step is the whole forward and backward through
`label_loss_grad`, `group_norm_grad` and `lookup_grad`, then Adam on the head's
parameters. Pixels that show no Gaussian are masked.
"""
from __future__ import annotations

import argparse

import numpy as np
import torch

from . import _lib as L
from . import scenes
from .field import FieldOps


class LabelHead:
    """Appearance rows, norm and label table over (views, H, W, channels) features."""

    GROUPS, SCALE = 4, 4.0

    def __init__(self, ops: FieldOps, channels: int, labels: int, views: int, seed: int = 0):
        g = torch.Generator().manual_seed(seed)

        def param(t):
            return t.to(ops.device, torch.float32)

        self.ops, self.labels, self.views = ops, labels, views
        self.params = {"appearance": param(torch.zeros(views, channels)),
                       "weight": param(torch.ones(channels)),
                       "bias": param(torch.zeros(channels)),
                       "table": param(torch.randn(labels, channels, generator=g) /
                                      channels ** 0.5)}
        self._moments = {k: (torch.zeros_like(v), torch.zeros_like(v))
                         for k, v in self.params.items()}
        self._steps = 0

    def _features(self, images, view_ids):
        """The table's input: rows (pixels, channels), and what the backward needs."""
        p = self.params
        rows = self.ops.lookup(p["appearance"], view_ids)
        x = images + rows.view(images.shape)
        y, mean, rstd = self.ops.group_norm(x, self.GROUPS, p["weight"], p["bias"], act="silu")
        return y.view(-1, y.shape[-1]), (x, mean, rstd)

    def loss(self, images, view_ids, labels):
        """The cross entropy of every pixel, 0 for masked ones."""
        feat, _ = self._features(images, view_ids)
        return self.ops.label_loss(feat, self.params["table"], labels, scale=self.SCALE)[0]

    def gradients(self, images, view_ids, labels):
        """(mean loss over the pixels with a label, gradients of the parameters); the
        mean stays on the GPU."""
        p = self.params
        feat, (x, mean, rstd) = self._features(images, view_ids)
        on = (labels >= 0).float()
        weight = on / on.sum().clamp(min=1)
        loss, _, dfeat, dtable = self.ops.label_loss_grad(feat, p["table"], labels, weight,
                                                          scale=self.SCALE)
        dx, dweight, dbias = self.ops.group_norm_grad(dfeat.view(x.shape), x, mean, rstd,
                                                      self.GROUPS, p["weight"], p["bias"],
                                                      act="silu")
        dapp = self.ops.lookup_grad(dx.view(feat.shape), view_ids, self.views)
        return (loss * weight).sum(), {"appearance": dapp, "weight": dweight, "bias": dbias,
                                       "table": dtable}

    def step(self, images, view_ids, labels, lr=0.02, betas=(0.9, 0.99), eps=1e-8):
        """One Adam step; returns the mean loss before it."""
        loss, grads = self.gradients(images, view_ids, labels)
        self._steps += 1
        for k, g in grads.items():
            m, v = self._moments[k]
            m.lerp_(g, 1 - betas[0])
            v.lerp_(g * g, 1 - betas[1])
            mh, vh = m / (1 - betas[0] ** self._steps), v / (1 - betas[1] ** self._steps)
            self.params[k] -= lr * mh / (vh.sqrt() + eps)
        return loss


def render_features(ctx: L.Context, scene, cam_poses, features, K, height, width):
    """(views, height, width, channels) feature images on the GPU: the scene rendered
    with its Gaussians' features as colours, three channels at a time."""
    cov = scenes.cov3d(scene.scales, scene.quats)
    n, channels = features.shape
    if channels % 3:
        raise ValueError("the channels are rendered three at a time")
    feat = features.detach().cpu().numpy().astype(np.float32)
    out = np.empty((len(cam_poses), height, width, channels), np.float32)
    for c in range(0, channels, 3):
        ctx.set_scene(scene.means, cov, scene.opacities, feat[:, c:c + 3])
        for v, w2c in enumerate(cam_poses):
            out[v, :, :, c:c + 3] = ctx.render(L.make_view(w2c, K, height, width))[0]
    return torch.from_numpy(out).cuda(ctx.device_index)


def synthetic(ops: FieldOps, gaussians=20_000, codes=60, labels=6, views=4, channels=24,
              height=120, width=160, seed=7):
    """Feature images, view ids and labels of a synthetic scene: codes by place, a
    label per code, pixels labelled by the code they show most of."""
    g = torch.Generator().manual_seed(seed)
    scene, _ = scenes.config1(seed=seed, n=gaussians)
    means = torch.from_numpy(scene.means)
    centers = means[torch.randperm(gaussians, generator=g)[:codes]]
    code = torch.cdist(means, centers).argmin(1).to(ops.device, torch.int32)
    of_code = torch.arange(codes) % labels
    codebook = torch.randn(codes, channels, generator=g).to(ops.device)
    features = ops.lookup(codebook, code)
    K = scenes.intrinsics(width * 0.78, width * 0.78, width / 2, height / 2)
    poses = [scenes.look_at_w2c((0.6 * np.cos(a), 0.4 * np.sin(a), 0.0), (0.0, 0.0, 5.0))
             for a in np.linspace(0, 2 * np.pi, views, endpoint=False)]
    images = render_features(ops.ctx, scene, poses, features, K, height, width)
    pad = -labels % 3
    one = torch.eye(labels + pad)[of_code][code.long().cpu()]
    shown = render_features(ops.ctx, scene, poses, one, K, height, width)
    most, label = shown.max(-1)
    label = torch.where(most > 0.2, label, torch.full_like(label, -1)).view(-1)
    view_ids = torch.arange(views, device=ops.device, dtype=torch.int32)
    return images, view_ids.repeat_interleave(height * width), label


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--gaussians", type=int, default=20_000)
    ap.add_argument("--steps", type=int, default=60)
    args = ap.parse_args(argv)
    ops = FieldOps()
    images, view_ids, labels = synthetic(ops, gaussians=args.gaussians)
    head = LabelHead(ops, images.shape[-1], 6, images.shape[0])
    for k in range(args.steps):
        loss = head.step(images, view_ids, labels)
        if k % 10 == 0 or k == args.steps - 1:
            print(f"step {k}: loss {float(loss):.4f}", flush=True)
    ops.check()
    feat, _ = head._features(images, view_ids)
    on = labels >= 0
    right = ((feat @ head.params["table"].T).argmax(1) == labels)[on].float().mean()
    print(f"{int(on.sum())} labelled pixels of {labels.numel()}, {float(right):.3f} of them right")


if __name__ == "__main__":
    main()

"""A feature decoder's gated projections and the clipping of gradients, as measurable
cases.

gated   the gated projections of a feed-forward block, act(x Wg^T + bg) * (x Wu^T + bu):
        features of pixels or Gaussians into hidden values, from which a label table
        scores. Alone (rendering, picking) or with the gradients (a training step).
clip    the global norm of many tensors' gradients (the root of the sum of all squares,
        or the largest size of a value), and their scaling down to a limit, into
        buffers of the optimizer's type or in place.
norm    the global norm alone.

Everything is drawn on the GPU from the seed.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_OPS = None


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one picked pixel through a small decoder: launch latency is all of it
        _gated("gated_one", 1, 64, 256, "silu", "f32", False, False),
        # a handful of picked pixels with wide features: the weights' bytes
        _gated("gated_few", 33, 512, 2048, "gelu", "bf16", True, False),
        # a 480 x 640 feature image rendered through its decoder
        _gated("gated_view", 307_200, 64, 256, "silu", "bf16", True, False),
        # 720p of 128 channels, exact decoding with fp32 features
        _gated("gated_view_f32", 921_600, 128, 128, "silu", "f32", True, False),
        # one batch of training pixels, odd row lengths
        _gated("gated_train_odd", 10_007, 75, 201, "gelu", "f32", True, True),
        # a training step on a 480 x 640 feature image
        _gated("gated_train_view", 307_200, 64, 128, "silu", "bf16", True, True),
        # fp32 features of 50K Gaussians, a wide decoder
        _gated("gated_train_f32", 50_021, 256, 1024, "silu", "f32", False, True),
        # open-vocabulary features of a batch of pixels, the widest decoder
        _gated("gated_train_wide", 100_003, 512, 2048, "silu", "bf16", False, True),
        # a label head's parameters: a handful of small tensors
        _grads("clip_head", "head", 6, 2048, "f32", "l2", "into", 0.5),
        # a 1M-Gaussian degree-3 scene's gradients: means, scales, rotations,
        # opacities and SH coefficients, clipped into the optimizer's buffers
        _grads("clip_scene", "scene", 5, 1_000_000, "f32", "l2", "into", 5.0),
        # decoders of many scenes, bf16 gradients under the limit, in place
        _grads("clip_calm", "layers", 60, 5_000_000, "bf16", "l2", "place", 1e9),
        # the largest gradient over many tensors of odd sizes
        _grads("norm_many", "layers", 301, 20_011, "f32", "max", "norm", 0.0),
    ]


def _gated(name, n, dim, hidden, act, dtype, bias, train):
    return {"name": name, "kind": "gated", "n": n, "dim": dim, "hidden": hidden, "act": act,
            "dtype": dtype, "bias": bias, "train": train}


def _grads(name, shapes, count, size, dtype, norm, to, limit):
    """`size`: the scene's Gaussians, or the values of the largest tensor; `to`: "into"
    fp32 buffers, in "place", or the "norm" alone."""
    return {"name": name, "kind": "grads", "shapes": shapes, "count": count, "size": size,
            "dtype": dtype, "norm": norm, "to": to, "limit": limit}


MOST = 100_003 * 512 * 2048


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    dtype = rng.choice(("f32", "bf16"))
    if rng.random() < 0.65:
        train = rng.random() < 0.5
        # feature lengths of tables and images, odd ones among them
        dim = rng.choice((3, 8, 16, 27, 32, 48, 64, 75, 100, 128, 256, 512, size(1, 1024)))
        hidden = rng.choice((16, 64, 128, 256, 512, 1000, 1024, 2048, size(1, 4096)))
        # a product of fp32 values costs about eight of bf16
        most = MOST // (8 if dtype == "f32" else 1)
        n = size(1, min(1_000_000, most // (dim * hidden), 300_000_000 // (dim + hidden)))
        # relu's slope jumps: where a gate is within rounding of 0 it is 0 or 1 by chance,
        # which is more than fp32 gradients may be off, and less than bf16 ones may
        acts = ("none", "silu", "gelu") if train and dtype == "f32" else \
            ("none", "relu", "silu", "gelu")
        c = _gated("", n, dim, hidden, rng.choice(acts), dtype, rng.random() < 0.5, train)
    else:
        to = rng.choice(("into", "into", "place", "norm"))
        limit = 1e9 if to == "place" else rng.choice((0.01, 1.0, 100.0))
        norm = rng.choice(("l2", "l2", "max"))
        if rng.random() < 0.25:
            c = _grads("", "scene", 5, size(100, 1_000_000), dtype, norm, to, limit)
        else:
            count = size(1, 400 if to == "norm" else 60)
            c = _grads("", rng.choice(("head", "layers")), count,
                       size(16, min(10_000_000, 200_000_000 // count)), dtype, norm, to, limit)
    del c["name"]
    return c


def _shapes(case):
    n, count = case["size"], case["count"]
    if case["shapes"] == "scene":
        return [(n, 3), (n, 3), (n, 4), (n,), (n, 16, 3)]
    if case["shapes"] == "head":
        # tables and their biases by turns
        return [(max(1, n // 32), 32) if i % 2 == 0 else (min(n, 32),) for i in range(count)]
    # sizes spread over three orders of magnitude, odd ones among them, the largest first
    return [(max(1, int(n * 1000.0 ** (-i / count))),) for i in range(count)]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=DEV)

    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "grads":
        # every tensor's gradients have a size of their own
        grads = [randn(*s).mul_(10.0 ** (i % 5 - 4)).to(dtype)
                 for i, s in enumerate(_shapes(case))]
        state = {"case": case, "grads": grads}
        if case["to"] == "into":
            state["out"] = [torch.empty(t.shape, device=DEV) for t in grads]
        return state
    n, dim, hidden = case["n"], case["dim"], case["hidden"]
    # normalised features: each channel has an offset and a spread of its own
    x = randn(n, dim).mul_(0.5 + 0.2 * randn(dim).abs()).add_(0.3 * randn(dim))
    state = {"case": case, "x": x.to(dtype),
             "w_gate": (randn(hidden, dim) * 1.5 / math.sqrt(dim)).to(dtype),
             "w_up": (randn(hidden, dim) / math.sqrt(dim)).to(dtype),
             "b_gate": 0.3 * randn(hidden) if case["bias"] else None,
             "b_up": 0.3 * randn(hidden) if case["bias"] else None}
    if case["train"]:
        state["dh"] = randn(n, hidden).mul_(1e-2).to(dtype)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    global _OPS
    if _OPS is None:
        from gsplat_tt_amd import field
        _OPS = field.FieldOps()
    case = state["case"]
    if case["kind"] == "grads":
        if case["to"] == "norm":
            return {"norm": _OPS.grad_norm(state["grads"], kind=case["norm"])}
        out = state.get("out", state["grads"])
        norm = _OPS.clip_grads(state["grads"], case["limit"], kind=case["norm"], out=out)
        return {"norm": norm, "grads": out}
    x, wg, wu, bg, bu = (state[k] for k in ("x", "w_gate", "w_up", "b_gate", "b_up"))
    h = _OPS.gated_linear(x, wg, wu, bg, bu, act=case["act"])
    if not case["train"]:
        return h
    dx, dwg, dwu, dbg, dbu = _OPS.gated_linear_grad(state["dh"], x, wg, wu, bg, bu,
                                                    act=case["act"])
    out = {"h": h, "dx": dx, "dw_gate": dwg, "dw_up": dwu}
    return {**out, "db_gate": dbg, "db_up": dbu} if case["bias"] else out


def _run_plain(state):
    case = state["case"]
    if case["kind"] == "grads":
        return _grads_plain(state)
    x, wg, wu = (state[k].float() for k in ("x", "w_gate", "w_up"))
    gate, up = x @ wg.T, x @ wu.T
    if case["bias"]:
        gate, up = gate + state["b_gate"], up + state["b_up"]
    act = case["act"]
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-gate))
        a, slope = gate * s, s * (1.0 + gate * (1.0 - s))
    elif act == "gelu":
        phi = 0.5 * torch.erfc(gate * -math.sqrt(0.5))
        a = gate * phi
        slope = phi + gate * torch.exp(-0.5 * gate * gate) / math.sqrt(2 * math.pi)
    elif act == "relu":
        a, slope = gate.clamp(min=0), (gate > 0).float()
    else:
        a, slope = gate, torch.ones_like(gate)
    dtype = state["x"].dtype
    h = (a * up).to(dtype)
    if not case["train"]:
        return h
    dh = state["dh"].float()
    dgate, dup = dh * up * slope, dh * a
    out = {"h": h, "dx": (dgate @ wg + dup @ wu).to(dtype), "dw_gate": (dgate.T @ x).to(dtype),
           "dw_up": (dup.T @ x).to(dtype)}
    return {**out, "db_gate": dgate.sum(0), "db_up": dup.sum(0)} if case["bias"] else out


def _grads_plain(state):
    case, grads = state["case"], state["grads"]
    if case["norm"] == "l2":
        norm = torch.stack([t.double().square().sum() for t in grads]).sum().sqrt().float()
    else:
        norm = torch.stack([t.abs().max().float() for t in grads]).max()
    if case["to"] == "norm":
        return {"norm": norm}
    factor = (case["limit"] / (norm + 1e-6)).clamp(max=1.0)
    if case["to"] == "into":
        for t, o in zip(grads, state["out"]):
            torch.mul(t.float(), factor, out=o)
        return {"norm": norm, "grads": state["out"]}
    for t in grads:
        t.copy_(t.float() * factor)
    return {"norm": norm, "grads": grads}


# ------------------------------------------------------------------ what a pass needs
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "grads":
        values = sum(math.prod(s) for s in _shapes(case))
        # in place and under the limit nothing has to be written
        out = 4 if case["to"] == "into" else 0
        return {"bytes": values * (e + out) + 4, "flops": values * (3 if out else 2)}
    n, dim, hidden = case["n"], case["dim"], case["hidden"]
    weights = 2 * hidden * dim
    # forward: x, weights in, h out; with gradients also dh in, dx and the weights' out
    values = n * dim + weights + n * hidden
    flops = 4 * n * dim * hidden
    if case["train"]:
        return {"bytes": 2 * values * e + (16 * hidden if case["bias"] else 0),
                "flops": 3 * flops}
    return {"bytes": values * e + (8 * hidden if case["bias"] else 0), "flops": flops}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    d = torch.float64
    if case["kind"] == "grads":
        if case["norm"] == "l2":
            total = sum(torch.linalg.vector_norm(t.to(d)) ** 2 for t in state["grads"])
            norm = total ** 0.5
        else:
            norm = max(t.to(d).abs().amax() for t in state["grads"])
        if case["to"] == "norm":
            return {"norm": norm}
        factor = min(1.0, case["limit"] / (float(norm) + 1e-6))
        return {"norm": norm, "grads": [t.to(d) * factor for t in state["grads"]]}
    hidden, train = case["hidden"], case["train"]
    act = {"none": lambda v: v * 1.0, "relu": torch.relu, "silu": lambda v: v * v.sigmoid(),
           "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2))}[case["act"]]
    w = torch.cat([state["w_gate"], state["w_up"]]).to(d)
    b = torch.zeros(2 * hidden, dtype=d, device=DEV)
    if case["bias"]:
        b = torch.cat([state["b_gate"], state["b_up"]]).to(d)
    h, dx, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, 2 ** 26 // hidden)
    for lo in range(0, case["n"], step):
        x = state["x"][lo:lo + step].to(d)
        z = torch.addmm(b, x, w.T).requires_grad_(train)
        y = act(z[:, :hidden]) * z[:, hidden:]
        h.append(y.detach())
        if train:
            dz, = torch.autograd.grad(y, z, state["dh"][lo:lo + step].to(d))
            dx.append(dz @ w)
            dw += dz.T @ x
            db += dz.sum(0)
    if not train:
        return torch.cat(h)
    out = {"h": torch.cat(h), "dx": torch.cat(dx), "dw_gate": dw[:hidden], "dw_up": dw[hidden:]}
    return {**out, "db_gate": db[:hidden], "db_up": db[hidden:]} if case["bias"] else out

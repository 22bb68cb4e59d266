"""The feature operators at the sizes their users run them, as measurable cases.

Learned features on splats take four kinds of work:

lookup  rows of a feature table by id, scaled: spherical-harmonics codes of a
        compressed scene, one learned appearance row per training view.
grad    the table's gradient: the sum of the rows' gradients per id.
norm    group norm with an activation over channels-last feature images, alone
        (rendering) or with its gradients (a training step).
loss    softmax cross entropy of per-pixel features against a table of labels or
        codes, alone (evaluation, picking) or with its gradients.

Ids and labels below 0 are masked. Everything is drawn on the GPU from the seed.
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
        # one batch of training pixels, each with its view's appearance row (a
        # capture of 169 training views): launch latency is all of it
        _lookup("lookup_views", 4096, 169, 32, "f32", True),
        # a compressed outdoor scene: the 15 x 3 higher-degree coefficients of
        # 6M Gaussians from a codebook of 65536 rows, odd row length
        _lookup("lookup_sh_6m", 6_000_000, 65536, 45, "f32", False),
        # appearance gradients of a 480 x 640 image's pixels drawn from 24 views:
        # few rows, each the sum of many
        _grad("grad_views", 307_200, 24, 64, "bf16", True),
        # codebook gradients of a 1M-Gaussian degree-3 scene, codes used unevenly
        _grad("grad_sh_1m", 1_000_000, 4096, 48, "f32", False),
        # a thumbnail's feature image in a viewer
        _norm("norm_thumb", 1, 60, 80, 32, 8, "silu", "f32", False),
        # a 720p feature image of 64 channels
        _norm("norm_720p", 1, 720, 1280, 64, 8, "silu", "bf16", False),
        # a training step on two small images of odd size, three channels a group
        _norm("norm_train_odd", 2, 333, 501, 48, 16, "relu", "f32", True),
        # a training step on a batch of quarter-size views
        _norm("norm_train_batch", 8, 240, 320, 128, 32, "gelu", "bf16", True),
        # the score of one picked pixel against a label table
        _loss("loss_one", 1, 1200, 64, "f32", False),
        # evaluation of a 480 x 640 label image
        _loss("loss_eval", 307_200, 150, 32, "bf16", False),
        # training codes of a degree-3 codebook from a batch of samples
        _loss("loss_train_codes", 10_007, 8192, 48, "f32", True),
        # open-vocabulary features of a batch of pixels, wide features
        _loss("loss_train_open", 30_011, 32_003, 512, "bf16", True),
    ]


def _lookup(name, n, rows, dim, dtype, ids64):
    return {"name": name, "kind": "lookup", "n": n, "rows": rows, "dim": dim, "dtype": dtype,
            "ids64": ids64}


def _grad(name, n, rows, dim, dtype, ids64):
    return {"name": name, "kind": "grad", "n": n, "rows": rows, "dim": dim, "dtype": dtype,
            "ids64": ids64}


def _norm(name, b, h, w, c, groups, act, dtype, train):
    return {"name": name, "kind": "norm", "b": b, "h": h, "w": w, "c": c, "groups": groups,
            "act": act, "dtype": dtype, "train": train}


def _loss(name, n, rows, dim, dtype, train):
    return {"name": name, "kind": "loss", "n": n, "rows": rows, "dim": dim, "dtype": dtype,
            "train": train}


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    kind = rng.choice(("lookup", "grad", "norm", "norm", "loss", "loss"))
    dtype = rng.choice(("f32", "bf16"))
    if kind == "lookup" or kind == "grad":
        # 3: colours; 12 to 48: SH coefficients; up to 512: features
        dim = rng.choice((3, 12, 16, 27, 32, 45, 48, 64, 75, 128, 256, 512))
        rows = size(8, 200_000)
        n = size(1, min(6_000_000, 2 ** 28 // dim) if kind == "lookup" else
                 min(3_000_000, 2 ** 27 // dim))
        c = (_lookup if kind == "lookup" else _grad)("", n, rows, dim, dtype, rng.random() < 0.5)
    elif kind == "norm":
        groups = rng.choice((1, 2, 4, 8, 16, 32))
        ch = groups * rng.choice((1, 2, 3, 4, 5, 8, 16))
        b = rng.choice((1, 1, 2, 3, 4, 8))
        w = size(1, 1300)
        h = max(1, int(w * rng.uniform(0.5, 1.0)))
        h = max(1, min(h, 78_000_000 // (b * w * ch)))
        c = _norm("", b, h, w, ch, groups, rng.choice(("none", "relu", "silu", "gelu")), dtype,
                  rng.random() < 0.5)
    else:
        dim = rng.choice((3, 8, 16, 31, 32, 48, 64, 100, 128, 256, 512))
        rows = size(2, 33_000)
        n = size(1, min(400_000, 450_000_000 // rows, 60_000_000_000 // (rows * dim)))
        c = _loss("", n, rows, dim, dtype, rng.random() < 0.6)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=DEV)

    def rand(*s):
        return torch.rand(*s, generator=g, device=DEV)

    dtype = DTYPES[case["dtype"]]
    if case["kind"] in ("lookup", "grad"):
        n, rows, dim = case["n"], case["rows"], case["dim"]
        ids = _uneven(rand(n), rows, randn(rows))
        ids = torch.where(rand(n) < 0.02, torch.full_like(ids, -1), ids)
        ids = ids if case["ids64"] else ids.int()
        state = {"case": case, "ids": ids, "scale": math.sqrt(dim)}
        if case["kind"] == "lookup":
            state["table"] = (randn(rows, dim) / math.sqrt(dim)).to(dtype)
        else:
            state["dout"] = (randn(n, dim) * 1e-2).to(dtype)
        return state
    if case["kind"] == "norm":
        b, h, w, c = case["b"], case["h"], case["w"], case["c"]
        # feature images: each channel has an offset and a spread of its own
        x = randn(b, h, w, c).mul_(0.5 + rand(c)).add_(randn(c)).to(dtype)
        state = {"case": case, "x": x, "weight": 1 + 0.2 * randn(c), "bias": 0.2 * randn(c)}
        if case["train"]:
            state["dy"] = randn(b, h, w, c).mul_(1e-2).to(dtype)
        return state
    n, rows, dim = case["n"], case["rows"], case["dim"]
    table = randn(rows, dim)
    table /= table.norm(dim=1, keepdim=True)
    labels = _uneven(rand(n), rows, randn(rows))
    # features lie near their label's row, as they do some way into training
    feat = randn(n, dim) / math.sqrt(dim) + 0.5 * table[labels]
    labels = torch.where(rand(n) < 0.05, torch.full_like(labels, -1), labels)
    state = {"case": case, "feat": feat.to(dtype), "table": table.to(dtype), "labels": labels,
             "scale": 10.0}
    if case["train"]:
        count = (labels >= 0).sum().clamp(min=1)
        state["row_weight"] = torch.ones(n, device=DEV) / count
    return state


def _uneven(u, rows, key):
    """Ids below `rows`, the k-th most used about as often as 1/(k + 8), in random order."""
    rank = (8.0 * ((rows + 8.0) / 8.0) ** u.double() - 8.0).long().clamp(0, rows - 1)
    return torch.argsort(key)[rank]


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    global _OPS
    if _OPS is None:
        from gsplat_tt_amd import field
        _OPS = field.FieldOps()
    case, kind = state["case"], state["case"]["kind"]
    if kind == "lookup":
        return _OPS.lookup(state["table"], state["ids"], state["scale"])
    if kind == "grad":
        return _OPS.lookup_grad(state["dout"], state["ids"], case["rows"], state["scale"])
    if kind == "norm":
        y, mean, rstd = _OPS.group_norm(state["x"], case["groups"], state["weight"],
                                        state["bias"], act=case["act"])
        if not case["train"]:
            return y
        dx, dw, db = _OPS.group_norm_grad(state["dy"], state["x"], mean, rstd, case["groups"],
                                          state["weight"], state["bias"], act=case["act"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if not case["train"]:
        return _OPS.label_loss(state["feat"], state["table"], state["labels"],
                               scale=state["scale"])[0]
    loss, _, df, dt = _OPS.label_loss_grad(state["feat"], state["table"], state["labels"],
                                           state["row_weight"], scale=state["scale"])
    return {"loss": loss, "dfeat": df, "dtable": dt}


def _run_plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "lookup":
        table, ids = state["table"], state["ids"].long()
        valid = (ids >= 0) & (ids < case["rows"])
        rows = table[ids.clamp(0, case["rows"] - 1)].float() * state["scale"]
        return torch.where(valid[:, None], rows, torch.zeros_like(rows)).to(table.dtype)
    if kind == "grad":
        dout, ids, rows = state["dout"], state["ids"].long(), case["rows"]
        valid = (ids >= 0) & (ids < rows)
        acc = torch.zeros(rows + 1, case["dim"], device=dout.device)
        acc.index_add_(0, torch.where(valid, ids, torch.full_like(ids, rows)), dout.float())
        return (acc[:rows] * state["scale"]).to(dout.dtype)
    if kind == "norm":
        return _norm_plain(state)
    feat, table, labels = state["feat"].float(), state["table"].float(), state["labels"]
    valid = labels >= 0
    safe = labels.clamp(min=0)[:, None]
    logits = state["scale"] * (feat @ table.T)
    lse = torch.logsumexp(logits, 1)
    loss = torch.where(valid, lse - logits.gather(1, safe)[:, 0], torch.zeros_like(lse))
    if not case["train"]:
        return loss
    w = torch.where(valid, state["row_weight"] * state["scale"], torch.zeros_like(lse))
    g = (logits - lse[:, None]).exp_()
    g.scatter_add_(1, safe, torch.full_like(lse, -1.0)[:, None])
    g *= w[:, None]
    return {"loss": loss, "dfeat": (g @ table).to(state["feat"].dtype),
            "dtable": (g.T @ feat).to(state["table"].dtype)}


def _norm_plain(state, eps=1e-5):
    case, x = state["case"], state["x"]
    shape = (case["b"], case["h"] * case["w"], case["groups"], case["c"] // case["groups"])
    xf = x.float().view(shape)
    mean = xf.mean((1, 3), keepdim=True)
    var = (xf - mean).square().mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    xh = (xf - mean) * rstd
    weight, bias = state["weight"].view(shape[2:]), state["bias"].view(shape[2:])
    z = xh * weight + bias
    act = case["act"]
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        y, slope = z * s, s * (1.0 + z * (1.0 - s))
    elif act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        y = z * phi
        slope = phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    elif act == "relu":
        y, slope = z.clamp(min=0), (z > 0).float()
    else:
        y, slope = z, torch.ones_like(z)
    y = y.to(x.dtype).view(x.shape)
    if not case["train"]:
        return y
    dz = state["dy"].float().view(shape) * slope
    dweight, dbias = (dz * xh).sum((0, 1)).view(-1), dz.sum((0, 1)).view(-1)
    dxh = dz * weight
    dx = rstd * (dxh - dxh.mean((1, 3), keepdim=True)
                 - xh * (dxh * xh).mean((1, 3), keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype).view(x.shape), "dweight": dweight, "dbias": dbias}


# ------------------------------------------------------------------ what a pass needs
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] in ("lookup", "grad"):
        n, rows, dim = case["n"], case["rows"], case["dim"]
        touched = min(n, rows) if case["kind"] == "lookup" else rows
        return {"bytes": n * (8 if case["ids64"] else 4) + (n + touched) * dim * e,
                "flops": n * dim}
    if case["kind"] == "norm":
        values = case["b"] * case["h"] * case["w"] * case["c"]
        # forward: x in, y out; with gradients also dy in, dx out
        return {"bytes": values * e * (4 if case["train"] else 2) + 8 * case["c"],
                "flops": values * (30 if case["train"] else 10)}
    n, rows, dim = case["n"], case["rows"], case["dim"]
    return {"bytes": (n + rows) * dim * e * (2 if case["train"] else 1) + n * 12,
            "flops": n * rows * dim * (6 if case["train"] else 2)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    d = torch.float64
    if case["kind"] == "lookup":
        out = torch.zeros(case["n"], case["dim"], dtype=d, device=DEV)
        seen = (state["ids"] >= 0).nonzero()[:, 0]
        out[seen] = state["table"].to(d)[state["ids"][seen].long()] * state["scale"]
        return out
    if case["kind"] == "grad":
        # running sums over the rows in id order, differenced at each id's end
        out = torch.zeros(case["rows"], case["dim"], dtype=d, device=DEV)
        seen = (state["ids"] >= 0).nonzero()[:, 0]
        order = seen[torch.argsort(state["ids"][seen].long(), stable=True)]
        total = torch.cumsum(state["dout"][order].to(d), 0)
        total = torch.cat([torch.zeros_like(out[:1]), total])
        count = torch.bincount(state["ids"][seen].long(), minlength=case["rows"])
        end = torch.cumsum(count, 0)
        return (total[end] - total[end - count]) * state["scale"]
    return _norm_exact(state) if case["kind"] == "norm" else _loss_exact(state)


def _norm_exact(state):
    case, d = state["case"], torch.float64
    b, c, groups = case["b"], case["c"], case["groups"]
    per = c // groups
    out = {k: torch.empty(b, case["h"] * case["w"], c, dtype=d, device=DEV)
           for k in (("y", "dx") if case["train"] else ("y",))}
    dweight, dbias = (torch.zeros(c, dtype=d, device=DEV) for _ in range(2))
    for i in range(b):
        for k in range(groups):
            at = slice(k * per, (k + 1) * per)
            x = state["x"][i, :, :, at].to(d).reshape(-1, per)
            weight, bias = state["weight"][at].to(d), state["bias"][at].to(d)
            var, mean = torch.var_mean(x, correction=0)
            scale = (var + 1e-5) ** -0.5
            xh = (x - mean) * scale
            z = (weight * xh + bias).requires_grad_(case["train"])
            y = {"none": lambda v: v * 1.0, "relu": torch.relu, "silu": lambda v: v * v.sigmoid(),
                 "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2))}[case["act"]](z)
            out["y"][i, :, at] = y.detach()
            if case["train"]:
                dz, = torch.autograd.grad(y, z, state["dy"][i, :, :, at].to(d).reshape(-1, per))
                dweight[at] += (dz * xh).sum(0)
                dbias[at] += dz.sum(0)
                t = dz * weight
                out["dx"][i, :, at] = scale * (t - t.mean() - xh * (t * xh).mean())
    out = {k: v.view(state["x"].shape) for k, v in out.items()}
    return {**out, "dweight": dweight, "dbias": dbias} if case["train"] else out["y"]


def _loss_exact(state):
    case, d = state["case"], torch.float64
    n, rows, dim = case["n"], case["rows"], case["dim"]
    table = state["table"].to(d)
    loss = torch.zeros(n, dtype=d, device=DEV)
    dfeat = torch.zeros(n, dim, dtype=d, device=DEV)
    dtable = torch.zeros(rows, dim, dtype=d, device=DEV)
    step = max(1, 2 ** 28 // rows)
    for lo in range(0, n, step):
        at = lo + (state["labels"][lo:lo + step] >= 0).nonzero()[:, 0]
        feat, label = state["feat"][at].to(d), state["labels"][at]
        score = (feat @ table.T) * state["scale"]
        prob = torch.softmax(score, 1)
        one = torch.arange(len(at), device=DEV)
        loss[at] = torch.log_softmax(score, 1)[one, label].neg()
        if case["train"]:
            prob[one, label] -= 1
            prob *= (state["row_weight"][at].to(d) * state["scale"])[:, None]
            dfeat[at] = prob @ table
            dtable += prob.T @ feat
    return {"loss": loss, "dfeat": dfeat, "dtable": dtable} if case["train"] else loss

"""What is measured of the operators on feature maps: layer_norm, the 8-bit
activation checkpoints (pack8, unpack8, checkpoint8) and label_loss.

A trainer that gives each Gaussian a feature vector besides its colour renders
it like a colour (render(colors=...)), normalises every pixel's vector, and
compares it with the embeddings of a label set: segment identities, classes or
the entries of a codebook. rows are the pixels of the views of a step (or the
pixels sampled from them), channels the feature's length.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
BLOCK = 128          # channels that share one scale of the 8-bit form


def listed():
    return [
        # one query's feature vector (a click in the viewer): latency only
        dict(name="norm-one", op="norm", rows=1, channels=512, dtype="bf16", saved="full",
             train=False),
        # one 800x800 view with 64-channel features, a training step
        dict(name="norm-frame", op="norm", rows=640_000, channels=64, dtype="fp32", saved="full",
             train=True),
        # 262144 sampled pixels with long (image encoder sized) features
        dict(name="norm-long", op="norm", rows=262_144, channels=512, dtype="bf16", saved="full",
             train=True),
        # the same view, the map held in 8 bits for the backward pass
        dict(name="norm-frame-8bit", op="norm", rows=640_000, channels=64, dtype="fp32",
             saved="int8", train=True),
        # a few sampled pixels of a narrow odd-sized feature
        dict(name="pack-small", op="pack", rows=5_000, channels=19, dtype="fp16"),
        # one 1600x900 view's map, held and read back
        dict(name="pack-frame", op="pack", rows=1_440_000, channels=32, dtype="fp32"),
        # one view through normalisation and loss, its map held in 8 bits
        dict(name="segment-frame", op="segment", rows=640_000, channels=32, classes=128,
             dtype="fp32"),
        # the smallest loss of use: 1000 sampled pixels, segment identities in a byte image
        dict(name="labels-pixels", op="labels", rows=1_000, channels=16, classes=200,
             dtype="fp32", labels="uint8", bias=True, reduction="mean", train=True),
        # one 800x800 view of 16-channel identity features
        dict(name="labels-frame", op="labels", rows=640_000, channels=16, classes=256,
             dtype="fp32", labels="int64", bias=True, reduction="mean", train=True),
        # sampled pixels of odd-sized features against a few thousand classes
        dict(name="labels-odd", op="labels", rows=100_003, channels=77, classes=4_099,
             dtype="fp32", labels="int32", bias=False, reduction="none", train=True),
        # long features against a codebook, the largest
        dict(name="labels-codebook", op="labels", rows=65_536, channels=512, classes=8_192,
             dtype="bf16", labels="int64", bias=False, reduction="mean", train=True),
        # evaluation of a 1600x900 view: every pixel's loss, no gradient
        dict(name="labels-eval", op="labels", rows=1_440_000, channels=64, classes=1_203,
             dtype="bf16", labels="int64", bias=True, reduction="none", train=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "pack", "segment", "labels", "labels", "labels"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    if op in ("norm", "pack"):
        channels = _log(rng, 3, 2048)
        rows = _log(rng, 1, min(1_440_000, 134_217_728 // channels))
        case = dict(op=op, rows=rows, channels=channels, dtype=dtype)
        if op == "norm":
            case["train"] = rng.random() < 0.8
            case["saved"] = rng.choice(["full", "int8"])
        return case
    if op == "segment":
        return dict(op=op, rows=_log(rng, 64, 640_000), channels=_log(rng, 3, 32),
                    classes=_log(rng, 2, 128), dtype="fp32")     # rendered maps are fp32
    channels = _log(rng, 3, 512)
    classes = _log(rng, 2, 32_768)
    rows = _log(rng, 1, min(1_440_000, 65_536 * 512 * 8_192 // (channels * classes)))
    return dict(op=op, rows=rows, channels=channels, classes=classes, dtype=dtype,
                labels=rng.choice(["uint8" if classes <= 255 else "int32", "int32", "int64"]),
                bias=rng.random() < 0.5, reduction=rng.choice(["mean", "sum", "none"]),
                train=rng.random() < 0.8)


def _ignored(case):
    return 255 if case.get("labels") == "uint8" else -100


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dt = DTYPES[case["dtype"]]
    n, d = case["rows"], case["channels"]
    s = {"case": case}
    if case["op"] in ("norm", "pack"):
        # rendered features: a spread per channel, an offset per pixel (its opacity)
        x = randn(n, d) * (0.5 + torch.rand(d, generator=g, device="cuda")) + 0.3 * randn(n, 1)
        s["x"] = x.to(dt)
        if case["op"] == "norm":
            s["weight"] = (1.0 + 0.1 * randn(d)).to(dt)
            s["bias"] = (0.1 * randn(d)).to(dt)
            s["grad"] = randn(n, d).to(dt)
    else:
        v = case["classes"]
        classes = randn(v, d) * (2.0 / math.sqrt(d))
        labels = torch.randint(0, v, (n,), generator=g, device="cuda")
        # features part of the way to their class, as in the middle of training
        x = randn(n, d) + 1.25 * classes[labels]
        # unlabelled stretches of the image, a tenth of it
        runs = torch.rand((n + 63) // 64, generator=g, device="cuda") < 0.1
        labels[runs.repeat_interleave(64)[:n]] = _ignored(case)
        s["x"] = x.to(dt)
        s["classes"] = classes.to(dt)
        s["labels"] = labels.to(getattr(torch, case.get("labels", "int64")))
        if case["op"] == "segment":
            s["weight"] = (1.0 + 0.1 * randn(d)).to(dt)
            s["bias"] = (0.1 * randn(d)).to(dt)
        else:
            s["class_bias"] = 0.5 * randn(v) if case["bias"] else None
            s["grad"] = randn(n).abs() if case["reduction"] == "none" else None
    if own:
        for k in ("x", "weight", "bias", "classes", "class_bias"):
            if s.get(k) is not None and case.get("train", True) and case["op"] != "pack":
                s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------ plain form

def _pack(x):
    """codes and scales of x in the 8-bit form, all in 32 bits: per BLOCK
    channels of a row, inv = 127 / a and scale = a / 127 of the largest
    magnitude a (0 below 1e-30), codes = round half even(x * inv)."""
    n, d = x.shape
    nb = (d + BLOCK - 1) // BLOCK
    xf = torch.zeros(n, nb * BLOCK, device=x.device)
    xf[:, :d] = x.float()
    xf = xf.view(n, nb, BLOCK)
    a = xf.abs().amax(2, keepdim=True)
    live = a >= 1e-30
    top = torch.full_like(a, 127.0)      # two tensors: a correctly rounded quotient
    inv = torch.where(live, torch.div(top, a), torch.zeros_like(a))
    scale = torch.where(live, torch.div(a, top), torch.zeros_like(a))
    codes = torch.round(xf * inv).clamp(-127, 127)
    return codes, scale


def _unpack(codes, scale, d):
    return (codes * scale).flatten(1)[:, :d]


def _norm(x, weight, bias):
    xf = x.float()
    mean = xf.mean(1, keepdim=True)
    rstd = torch.rsqrt(((xf - mean) ** 2).mean(1, keepdim=True) + EPS)
    return (xf - mean) * rstd * weight.float() + bias.float(), mean, rstd


def _norm_backward(xf, mean, rstd, weight, g):
    xh = (xf - mean) * rstd
    wg = g * weight.float()
    dx = rstd * (wg - wg.mean(1, keepdim=True) - xh * (wg * xh).mean(1, keepdim=True))
    return dx, (g * xh).sum(0), g.sum(0)


def _chunk(n, v):
    return max(1, min(n, (1 << 28) // v))


def _labels(x, classes, bias, labels, ignored, reduction, grad, train):
    """loss and gradients (x, classes, bias) in 32 bits."""
    n, v = x.shape[0], classes.shape[0]
    wf = classes.float()
    live = labels != ignored
    count = live.sum().clamp_min(1).float()
    rows = live.float()
    if reduction == "mean":
        rows = rows / count
    elif reduction == "none" and grad is not None:
        rows = rows * grad.float()
    loss = torch.empty(n, device=x.device)
    dx = torch.empty(x.shape, device=x.device)
    dw, db = torch.zeros_like(wf), torch.zeros(v, device=x.device)
    step = _chunk(n, v)
    for i in range(0, n, step):
        j = slice(i, min(n, i + step))
        lv = live[j]
        xf = x[j].float() * lv[:, None]
        z = xf @ wf.t()
        if bias is not None:
            z = z + bias.float()
        m = z.amax(1, keepdim=True)
        e = torch.exp(z - m)
        lab = torch.where(lv, labels[j].long(), torch.zeros_like(labels[j], dtype=torch.long))
        zl = z.gather(1, lab[:, None])
        el = e.gather(1, lab[:, None])
        # the others' share by itself: 1 - p of a confident row keeps its digits
        others = e.scatter(1, lab[:, None], 0.0).sum(1, keepdim=True)
        t = others + el
        row = torch.where(zl == m, torch.log1p(others), torch.log(t) + (m - zl))
        loss[j] = row[:, 0] * lv
        if train:
            p = (e / t).scatter(1, lab[:, None], -others / t)
            p = p * rows[j, None]
            dx[j] = p @ wf
            dw += p.t() @ xf
            db += p.sum(0)
    if reduction == "mean":
        loss = loss.sum() / count
    elif reduction == "sum":
        loss = loss.sum()
    return loss, dx, dw, db


def _plain(s):
    case, x = s["case"], s["x"]
    dt, d = x.dtype, x.shape[1]
    if case["op"] == "pack":
        codes, scale = _pack(x)
        return {"scales": scale[..., 0], "values": _unpack(codes, scale, d).to(dt)}
    if case["op"] == "norm":
        y, mean, rstd = _norm(x, s["weight"], s["bias"])
        if not case["train"]:
            return {"y": y.to(dt)}
        xf = x.float() if case["saved"] == "full" else _unpack(*_pack(x), d)
        dx, dw, db = _norm_backward(xf, mean, rstd, s["weight"], s["grad"].float())
        return {"y": y.to(dt), "dx": dx.to(dt), "dweight": dw.to(dt), "dbias": db.to(dt)}
    if case["op"] == "segment":
        y, _, _ = _norm(x, s["weight"], s["bias"])
        loss = _labels(y, s["classes"], None, s["labels"], -100, "mean", None, False)[0]
        held = _unpack(*_pack(x), d)
        y, mean, rstd = _norm(held, s["weight"], s["bias"])
        _, dy, dc, _ = _labels(y, s["classes"], None, s["labels"], -100, "mean", None, True)
        dx, dw, db = _norm_backward(held, mean, rstd, s["weight"], dy)
        return {"loss": loss, "dx": dx, "dweight": dw, "dbias": db, "dclasses": dc}
    loss, dx, dw, db = _labels(x, s["classes"], s["class_bias"], s["labels"], _ignored(case),
                               case["reduction"], s["grad"], case["train"])
    out = {"loss": loss}
    if case["train"]:
        out["dx"], out["dclasses"] = dx.to(dt), dw.to(dt)
        if s["class_bias"] is not None:
            out["dclass_bias"] = db
    return out


# ------------------------------------------------------------------ the framework's

def _own(s):
    from metal_gauss_b200.activations import checkpoint8, pack8, unpack8
    from metal_gauss_b200.labels import label_loss
    from metal_gauss_b200.layernorm import layer_norm

    case, x = s["case"], s["x"]
    if case["op"] == "pack":
        codes, scales = pack8(x)
        return {"scales": scales, "values": unpack8(codes, scales, dtype=x.dtype)}
    if case["op"] == "norm":
        y = layer_norm(x, s["weight"], s["bias"], eps=EPS, saved=case["saved"])
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, s["weight"], s["bias"]), s["grad"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "segment":
        def segment(x, weight, bias, classes):
            return label_loss(layer_norm(x, weight, bias, eps=EPS), classes, s["labels"])

        leaves = (x, s["weight"], s["bias"], s["classes"])
        loss = checkpoint8(segment, *leaves)
        dx, dw, db, dc = torch.autograd.grad(loss, leaves)
        return {"loss": loss.detach(), "dx": dx, "dweight": dw, "dbias": db, "dclasses": dc}
    loss = label_loss(x, s["classes"], s["labels"], bias=s["class_bias"],
                      ignore_index=_ignored(case), reduction=case["reduction"])
    if not case["train"]:
        return {"loss": loss}
    leaves = [x, s["classes"]] + ([s["class_bias"]] if s["class_bias"] is not None else [])
    grads = torch.autograd.grad(loss, leaves, s["grad"])
    return {"loss": loss.detach(), **dict(zip(("dx", "dclasses", "dclass_bias"), grads))}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass has to do

def work(case):
    n, d, b = case["rows"], case["channels"], BYTES[case["dtype"]]
    blocks = (d + BLOCK - 1) // BLOCK
    if case["op"] == "pack":
        # x in and back out; the 8-bit form written once and read once
        return {"bytes": 2 * n * d * b + 2 * n * (d + 4 * blocks), "flops": 4 * n * d}
    if case["op"] == "norm":
        if not case["train"]:
            return {"bytes": 2 * n * d * b + 2 * d * b, "flops": 7 * n * d}
        # x, y, its gradient, dx; the backward pass reads x again, or its 8-bit
        # form, which the forward pass wrote
        held = n * d * b if case["saved"] == "full" else 2 * n * (d + 4 * blocks)
        return {"bytes": 4 * n * d * b + held + 16 * n + 4 * d * b, "flops": 20 * n * d}
    v = case["classes"]
    lab = n * {"uint8": 1, "int32": 4, "int64": 8}[case.get("labels", "int64")]
    if case["op"] == "segment":
        return {"bytes": 2 * n * d * b + 2 * n * (d + 4 * blocks) + 2 * lab + 2 * v * d * b,
                "flops": 8 * n * d * v + 30 * n * d}
    if not case["train"]:
        return {"bytes": n * d * b + v * d * b + lab + 4 * n, "flops": 2 * n * d * v}
    return {"bytes": 2 * n * d * b + 2 * v * d * b + lab
            + (8 * n if case["reduction"] == "none" else 4), "flops": 6 * n * d * v}


# ------------------------------------------------------------------ in 64 bits

def _held64(x):
    """x as the 8-bit form gives it back: the form is defined by 32-bit
    quotients and products, each correctly rounded; code * scale in 64 bits."""
    n, d = x.shape
    out = torch.empty(n, d, dtype=torch.float64, device=x.device)
    scales = []
    for c in range(0, d, BLOCK):
        part = x[:, c:c + BLOCK].float()
        top = part.abs().max(dim=1, keepdim=True).values
        scale = torch.div(top, torch.full_like(top, 127.0))
        inv = torch.div(torch.full_like(top, 127.0), top)
        dead = (top < 1e-30).expand_as(part)
        codes = torch.round(part * inv).masked_fill(dead, 0.0).clamp(-127.0, 127.0)
        scale = scale.masked_fill(top < 1e-30, 0.0)
        out[:, c:c + BLOCK] = codes.double() * scale.double()
        scales.append(scale)
    return out, torch.cat(scales, 1).double()


def _norm64(x, weight, bias):
    var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
    inv = 1.0 / torch.sqrt(var + EPS)
    return torch.addcmul(bias, (x - mean) * inv, weight), mean, inv


def _norm64_adjoint(x, mean, inv, weight, gy):
    hat = (x - mean) * inv
    d_hat = gy * weight
    d = x.shape[1]
    proj = (d_hat * hat).sum(1, keepdim=True) / d
    return ((d_hat - d_hat.sum(1, keepdim=True) / d - hat * proj) * inv,
            torch.einsum("nd,nd->d", gy, hat), gy.sum(0))


def _labels64(x, w, bias, labels, ignored, reduction, grad, train):
    n, d = x.shape
    keep = torch.nonzero(labels != ignored)[:, 0]
    total = max(1, keep.numel())
    per_row = torch.zeros(n, dtype=torch.float64, device=x.device)
    dx = torch.zeros(n, d, dtype=torch.float64, device=x.device)
    dw = torch.zeros_like(w)
    db = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device)
    for rows in keep.split(max(1, (1 << 27) // w.shape[0])):
        xr, lab = x[rows], labels[rows].long()
        logits = torch.mm(xr, w.t())
        if bias is not None:
            logits += bias
        logp = torch.log_softmax(logits, dim=1)
        per_row[rows] = -logp[torch.arange(rows.numel(), device=x.device), lab]
        if train:
            gz = logp.exp_()
            gz[torch.arange(rows.numel(), device=x.device), lab] -= 1.0
            if reduction == "mean":
                gz /= total
            elif reduction == "none":
                gz *= grad[rows, None]
            dx[rows] = torch.mm(gz, w)
            dw += torch.mm(gz.t(), xr)
            db += gz.sum(0)
    loss = {"none": per_row, "sum": per_row.sum(), "mean": per_row.sum() / total}[reduction]
    return loss, dx, dw, db


def exact(case, seed):
    s = prepare(case, seed)
    f = {k: t.detach().double() for k, t in s.items()
         if torch.is_tensor(t) and t.is_floating_point()}
    x = s["x"].detach()
    if case["op"] == "pack":
        held, scales = _held64(x)
        return {"scales": scales, "values": held}
    if case["op"] == "norm":
        y, mean, inv = _norm64(f["x"], f["weight"], f["bias"])
        if not case["train"]:
            return {"y": y}
        kept = f["x"] if case["saved"] == "full" else _held64(x)[0]
        dx, dw, db = _norm64_adjoint(kept, mean, inv, f["weight"], f["grad"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "segment":
        y, _, _ = _norm64(f["x"], f["weight"], f["bias"])
        loss = _labels64(y, f["classes"], None, s["labels"], -100, "mean", None, False)[0]
        held = _held64(x)[0]
        y, mean, inv = _norm64(held, f["weight"], f["bias"])
        _, dy, dc, _ = _labels64(y, f["classes"], None, s["labels"], -100, "mean", None, True)
        dx, dw, db = _norm64_adjoint(held, mean, inv, f["weight"], dy)
        return {"loss": loss, "dx": dx, "dweight": dw, "dbias": db, "dclasses": dc}
    loss, dx, dw, db = _labels64(f["x"], f["classes"], f.get("class_bias"), s["labels"],
                                 _ignored(case), case["reduction"], f.get("grad"),
                                 case["train"])
    out = {"loss": loss}
    if case["train"]:
        out["dx"], out["dclasses"] = dx, dw
        if s["class_bias"] is not None:
            out["dclass_bias"] = db
    return out

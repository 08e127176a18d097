"""Label supervision of rendered feature maps.

`label_loss` compares every pixel's feature vector with the embeddings of a
label set (segment identities, classes, the entries of a codebook) and is the
cross entropy of the softmax over them. It stands beside the image losses of
ssim.py for feature maps that the rasteriser draws as explicit colours. The
(pixels, classes) logits are never stored: the forward pass walks the classes
in tiles with a running maximum and sum, the backward pass computes the tiles
again (`mg_label_loss_forward`, `mg_label_loss_backward`).
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr
from .activations import DTYPES, check_cuda, dtype_code, once, wants_grad

MAX_CHANNELS, MAX_CLASSES = 512, 1 << 20      # MG_LABEL_MAX_CHANNELS, MG_LABEL_MAX_CLASSES
REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
LABEL_BYTES = {torch.uint8: 1, torch.int32: 4, torch.int64: 8}


_FORWARD = _lib.Launcher("mg_label_loss_forward")
_BACKWARD = _lib.Launcher("mg_label_loss_backward")
_SCRATCH = _lib.SizeOf("mg_label_loss_scratch_bytes")


def _forward(features, classes, labels, bias, scale, ignore_index, reduction, train):
    """The loss and what the backward pass needs; stats is (2 n + 1,): the two
    values of each row and the count of live ones."""
    d, v = features.shape[-1], classes.shape[0]
    n = labels.numel()
    code = DTYPES[features.dtype]
    x = features.detach().contiguous()
    w = classes.detach().contiguous()
    lab = labels.contiguous()
    b = None if bias is None else bias.detach().to(torch.float32).contiguous()
    loss = torch.empty(labels.shape if reduction == 0 else (), dtype=torch.float32,
                       device=x.device)
    stats = torch.empty(2 * n + 1, dtype=torch.float32, device=x.device) if train else None
    at = ptr(stats)
    nbytes = _SCRATCH(x.get_device(), n, d, v, code, 0)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _FORWARD(x.get_device(), ptr(x), ptr(w), code, ptr(b), ptr(lab), LABEL_BYTES[lab.dtype],
             ignore_index, n, d, v, scale, reduction, ptr(loss), at,
             at + 8 * n if train and reduction else None, ptr(scratch), nbytes)
    return loss, (x, w, lab, b, stats)


class _LabelLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, classes, labels, bias, scale, ignore_index, reduction):
        loss, kept = _forward(features, classes, labels, bias, scale, ignore_index, reduction,
                              True)
        ctx.save_for_backward(*kept)
        ctx.meta = (scale, ignore_index, reduction)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return loss

    @staticmethod
    @once
    def backward(ctx, grad):
        x, w, lab, b, stats = ctx.saved_tensors
        scale, ignore_index, reduction = ctx.meta
        need_x, need_w, _, need_b = ctx.needs_input_grad[:4]
        d, v, n = x.shape[-1], w.shape[0], lab.numel()
        code = DTYPES[x.dtype]
        g = grad.to(torch.float32).contiguous()
        dx = torch.empty_like(x) if need_x else None
        dw = torch.empty_like(w) if need_w else None
        db = torch.empty(v, dtype=torch.float32, device=x.device) if need_b else None
        nbytes = _SCRATCH(x.get_device(), n, d, v, code, 1)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        at = stats.data_ptr()
        _BACKWARD(x.get_device(), ptr(x), ptr(w), code, ptr(b), ptr(lab), LABEL_BYTES[lab.dtype],
                  ignore_index, n, d, v, scale, reduction, ptr(g), at,
                  at + 8 * n if reduction else None, ptr(dx), ptr(dw), ptr(db), ptr(scratch),
                  nbytes)
        if db is not None and ctx.bias_dtype != torch.float32:
            db = db.to(ctx.bias_dtype)
        return dx, dw, None, db, None, None, None


def label_loss(features: torch.Tensor, classes: torch.Tensor, labels: torch.Tensor,
               bias: torch.Tensor | None = None, scale: float = 1.0, ignore_index: int = -100,
               reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of softmax(scale * features @ classes.T + bias) against
    labels, differentiable in features, classes and bias.

    features (..., channels), up to 512 channels; classes (n_classes,
    channels) of the same type (float32, bfloat16 or float16); scale a number
    (a tensor that needs a gradient is refused); labels (...) uint8, int32 or
    int64; bias (n_classes,) float32 or of the features' type, -infinity taking
    a class out (whose embedding is finite all the same). Pixels labelled ignore_index have loss 0 and
    no gradient whatever their features hold, and do not count in a mean. The
    result is float32: one value for reduction "mean" (0 when no pixel takes
    part) or "sum", labels' shape for "none". A row with an infinite logit has
    loss NaN; logits have to stay within float32's range. Another label outside
    [0, n_classes) makes the loss NaN and is recorded in the device error word
    (`_lib.check_device_error`)."""
    dtype_code(features, "label_loss: features")
    if features.dim() < 1 or not 1 <= features.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"label_loss: features must be (..., channels) with 1 to {MAX_CHANNELS} "
                         f"channels, got {tuple(features.shape)}")
    if classes.dim() != 2 or classes.shape[1] != features.shape[-1] or \
            not 1 <= classes.shape[0] <= MAX_CLASSES:
        raise ValueError(f"label_loss: classes must be (n_classes, {features.shape[-1]}) with 1 "
                         f"to {MAX_CLASSES} classes, got {tuple(classes.shape)}")
    if classes.dtype != features.dtype:
        raise TypeError(f"label_loss: features are {features.dtype}, classes {classes.dtype}")
    if labels.dtype not in LABEL_BYTES:
        raise TypeError(f"label_loss: labels must be uint8, int32 or int64, got {labels.dtype}")
    if labels.shape != features.shape[:-1]:
        raise ValueError(f"label_loss: labels must be {tuple(features.shape[:-1])}, got "
                         f"{tuple(labels.shape)}")
    if bias is not None:
        if tuple(bias.shape) != (classes.shape[0],):
            raise ValueError(f"label_loss: bias must be ({classes.shape[0]},), got "
                             f"{tuple(bias.shape)}")
        if bias.dtype not in (torch.float32, features.dtype):
            raise TypeError(f"label_loss: bias must be float32 or {features.dtype}, got "
                            f"{bias.dtype}")
    for t, what in ((classes, "classes"), (labels, "labels"), (bias, "bias")):
        if t is not None and t.device != features.device:
            raise RuntimeError(f"label_loss: features on {features.device}, {what} on {t.device}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"label_loss: reduction must be one of {tuple(REDUCTIONS)}, got "
                         f"{reduction!r}")
    if torch.is_tensor(scale) and wants_grad(scale):
        raise TypeError("label_loss: scale is a number and has no gradient; to learn it, multiply "
                        "the features or the classes by it")
    check_cuda(features, "label_loss: features")
    args = (features, classes, labels, bias, float(scale), int(ignore_index),
            REDUCTIONS[reduction])
    if not wants_grad(features, classes, bias):
        return _forward(*args, False)[0]
    return _LabelLoss.apply(*args)

"""Layer normalisation of per-pixel feature vectors, forward and backward.

`layer_norm` normalises the last dimension of a rendered feature map (any
(..., channels) tensor) before it is compared with class embeddings
(`labels.label_loss`). One kernel each way plus the join of the weight's and
bias's gradients (`mg_layer_norm_forward`, `mg_layer_norm_backward`); sums are
fp32 in a fixed order, so equal calls give equal bits.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr
from .activations import BLOCK, DTYPES, check_cuda, dtype_code, once, wants_grad

MAX_CHANNELS = 8192      # MG_LAYER_NORM_MAX_CHANNELS
_FORWARD = _lib.Launcher("mg_layer_norm_forward")
_BACKWARD = _lib.Launcher("mg_layer_norm_backward")
_SCRATCH = _lib.SizeOf("mg_layer_norm_backward_scratch_bytes")


def _forward(x, weight, bias, eps, train, saved):
    """y and what the backward pass needs: x, or codes and scales; mean and
    rstd as one (2 n,) tensor."""
    d = x.shape[-1]
    n = x.numel() // d
    params = weight if weight is not None else bias
    pcode = 0 if params is None else DTYPES[params.dtype]
    x = x.detach().contiguous()
    w = None if weight is None else weight.detach().contiguous()
    b = None if bias is None else bias.detach().contiguous()
    y = torch.empty_like(x)
    stats = codes = scales = None
    mean = rstd = None
    if train:
        stats = torch.empty(2 * n, dtype=torch.float32, device=x.device)
        mean = stats.data_ptr()
        rstd = mean + 4 * n
        if saved == "int8":
            codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
            scales = torch.empty((n, -(-d // BLOCK)), dtype=torch.float32, device=x.device)
    _FORWARD(x.get_device(), ptr(x), DTYPES[x.dtype], ptr(w), ptr(b), pcode, n, d, eps, ptr(y),
             mean, rstd, ptr(codes), ptr(scales))
    return y, (x if codes is None else None, codes, scales, w, stats), pcode


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, saved):
        y, kept, ctx.pcode = _forward(x, weight, bias, eps, True, saved)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    @once
    def backward(ctx, dy):
        x, codes, scales, w, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        d = dy.shape[-1]
        n = dy.numel() // d
        pdtype = (torch.float32, torch.bfloat16, torch.float16)[ctx.pcode]
        dy = dy.contiguous()
        dx = torch.empty_like(dy) if need_x else None
        dw = torch.empty(d, dtype=pdtype, device=dy.device) if need_w else None
        db = torch.empty(d, dtype=pdtype, device=dy.device) if need_b else None
        scratch, nbytes = None, 0
        if need_w or need_b:
            nbytes = _SCRATCH(dy.get_device(), n, d)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dy.device)
        mean = stats.data_ptr()
        _BACKWARD(dy.get_device(), ptr(dy), ptr(x), ptr(codes), ptr(scales), DTYPES[dy.dtype],
                  ptr(w), ctx.pcode, mean, mean + 4 * n, n, d, ptr(dx), ptr(dw), ptr(db),
                  ptr(scratch), nbytes)
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5,
               saved: str = "full") -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of
    x (..., channels), differentiable in x, weight and bias. x is float32,
    bfloat16 or float16; weight and bias (channels,) have x's type or float32,
    both the same. saved="int8" holds x for the backward pass in 8 bits
    (activations.pack8) in place of x itself: y is unchanged, the gradients
    are the formula's at the x that reads back, with the mean and deviation of
    the true x."""
    dtype_code(x, "layer_norm: x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"layer_norm: x must be (..., channels) with 1 to {MAX_CHANNELS} "
                         f"channels, got {tuple(x.shape)}")
    if saved not in ("full", "int8"):
        raise ValueError(f"layer_norm: saved must be 'full' or 'int8', got {saved!r}")
    if torch.is_tensor(eps) and wants_grad(eps):
        raise TypeError("layer_norm: eps is a number and has no gradient")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"layer_norm: {what} must be ({x.shape[-1]},), got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"layer_norm: {what} must be {x.dtype} or float32, got {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"layer_norm: x on {x.device}, {what} on {t.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    check_cuda(x, "layer_norm: x")
    if not wants_grad(x, weight, bias):
        return _forward(x, weight, bias, float(eps), False, saved)[0]
    return _LayerNorm.apply(x, weight, bias, float(eps), saved)

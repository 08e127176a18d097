"""Activation checkpoints in 8 bits.

What follows a feature map in the graph (normalisation, products, a loss) holds
it and its own intermediate maps for the backward pass. `pack8` puts a map into
one byte per element and one fp32 scale per 128 channels (`mg_pack8`), `unpack8`
reads it back, and `checkpoint8(fn, x, ...)` runs a segment of the graph whose
input is held in that form and computed again in the backward pass.
`layernorm.layer_norm(saved="int8")` uses the same form without the second
forward pass. What the rasteriser itself holds for the map's own gradient is
untouched by this.

    a = largest magnitude of 128 channels of a row (fewer at its end)
    scale = a / 127,  code = round half even(x * (127 / a)),  value = code * scale

so a value comes back within a / 254 of itself.
"""

from __future__ import annotations

import contextlib
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import ptr

_PACK, _UNPACK = _lib.Launcher("mg_pack8"), _lib.Launcher("mg_unpack8")
BLOCK = 128
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # MG_F32, MG_BF16, MG_F16


def wants_grad(*tensors: torch.Tensor | None) -> bool:
    """Whether an operator on these goes through its autograd function: one of
    them needs a gradient, or a forward-mode level is open (the function then
    refuses an input that carries a tangent, which a detached one would lose)."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def once(backward):
    """The backward of an autograd function that has no second derivative:
    torch's own guard where a graph of it is being built, none of its cost
    where not."""
    guarded = torch.autograd.function.once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


def dtype_code(t: torch.Tensor, what: str) -> int:
    if t.dtype not in DTYPES:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return DTYPES[t.dtype]


def check_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} is on '{t.device}': the CUDA backend needs CUDA tensors and "
                           "does not move data or fall back")


def _rows(t: torch.Tensor, what: str) -> tuple[int, int]:
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{what} must be (..., channels) with at least one channel, "
                         f"got {tuple(t.shape)}")
    return t.numel() // t.shape[-1], t.shape[-1]


def pack8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (..., channels) in 8 bits: codes int8 (..., channels) and scales
    float32 (..., ceil(channels / 128)), neither differentiable in x. 128
    channels with an infinity or a NaN among them read back as NaN; below 1e-30
    they read back as 0."""
    code, (n, d) = dtype_code(x, "pack8: x"), _rows(x, "pack8: x")
    check_cuda(x, "pack8: x")
    x = x.detach().contiguous()
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty((*x.shape[:-1], -(-d // BLOCK)), dtype=torch.float32, device=x.device)
    _PACK(x.get_device(), ptr(x), code, n, d, ptr(codes), ptr(scales))
    return codes, scales


def unpack8(codes: torch.Tensor, scales: torch.Tensor,
            dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The tensor that `pack8` gave codes and scales for, as `dtype`. It has no
    gradient: scales that need one are refused."""
    if scales.requires_grad and torch.is_grad_enabled():
        raise TypeError("unpack8: scales need a gradient, and unpack8 has none")
    if codes.dtype != torch.int8 or scales.dtype != torch.float32:
        raise TypeError(f"unpack8 takes int8 codes and float32 scales, got {codes.dtype} and "
                        f"{scales.dtype}")
    if dtype not in DTYPES:
        raise TypeError(f"unpack8: dtype must be float32, bfloat16 or float16, got {dtype}")
    n, d = _rows(codes, "unpack8: codes")
    want = (*codes.shape[:-1], -(-d // BLOCK))
    if tuple(scales.shape) != want:
        raise ValueError(f"unpack8: scales must be {want} for codes {tuple(codes.shape)}, "
                         f"got {tuple(scales.shape)}")
    if scales.device != codes.device:
        raise RuntimeError(f"unpack8: codes on {codes.device}, scales on {scales.device}")
    check_cuda(codes, "unpack8: codes")
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 8:
        codes = codes.clone()
    x = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    _UNPACK(codes.get_device(), ptr(codes), ptr(scales), n, d, DTYPES[dtype], ptr(x))
    return x


def _parameters(fn) -> tuple[torch.Tensor, ...]:
    """The parameters that a module (or a module's method, or a partial of
    either) trains."""
    while isinstance(fn, functools.partial):
        fn = fn.func
    module = fn if isinstance(fn, torch.nn.Module) else getattr(fn, "__self__", None)
    if not isinstance(module, torch.nn.Module):
        return ()
    return tuple(p for p in module.parameters() if p.requires_grad)


def _refuse_other_leaves(out: torch.Tensor, leaves: list[torch.Tensor]) -> None:
    """Raises when out's graph ends in a tensor that is none of leaves."""
    known = {id(t) for t in leaves}
    seen, todo = set(), [out.grad_fn]
    while todo:
        node = todo.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        if node.name() == "torch::autograd::AccumulateGrad" and id(node.variable) not in known:
            raise RuntimeError(f"checkpoint8: fn uses a tensor {tuple(node.variable.shape)} that "
                               "needs a gradient and is none of its arguments: pass it as an "
                               "argument, or detach it")
        todo.extend(n for n, _ in node.next_functions)


def _autocast_state() -> tuple[bool, torch.dtype]:
    return torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda")


def _autocast(state: tuple[bool, torch.dtype]):
    """The mixed precision of state, without the cache of cast parameters: one
    cast without a graph must not serve a later use that needs it, nor one from
    outside a segment's own graph."""
    enabled, dtype = state
    if not enabled and not torch.is_autocast_enabled("cuda"):
        return contextlib.nullcontext()
    return torch.autocast("cuda", dtype=dtype, enabled=enabled, cache_enabled=False)


def _one_tensor(out) -> torch.Tensor:
    if not torch.is_tensor(out):
        raise TypeError(f"checkpoint8: fn must return one tensor, got {type(out).__name__}")
    return out


class _Checkpoint8(torch.autograd.Function):
    """Inputs: fn, the number of its arguments after x, x, those, and the
    parameters that fn brings along."""

    @staticmethod
    def forward(ctx, fn, count, x, *rest):
        args = rest[:count]
        ctx.fn, ctx.count, ctx.dtype = fn, count, x.dtype
        ctx.where = [i for i, a in enumerate(args) if torch.is_tensor(a)]
        ctx.others = [None if torch.is_tensor(a) else a for a in args]
        codes, scales = pack8(x)
        ctx.save_for_backward(codes, scales, *(args[i] for i in ctx.where), *rest[count:])
        ctx.autocast = _autocast_state()
        with torch.no_grad(), _autocast(ctx.autocast):
            return _one_tensor(fn(x, *args))

    @staticmethod
    @once
    def backward(ctx, grad):
        codes, scales, *tensors = ctx.saved_tensors
        need = ctx.needs_input_grad[2:]
        x = unpack8(codes, scales, ctx.dtype)
        args = list(ctx.others)
        with torch.enable_grad(), _autocast(ctx.autocast):
            x.requires_grad_(need[0])
            for i, t in zip(ctx.where, tensors):
                args[i] = t.detach().requires_grad_(need[1 + i])
            out = ctx.fn(x, *args)
        inputs = [x, *args, *tensors[len(ctx.where):]]
        leaves = [t for t, k in zip(inputs, need) if k]
        _refuse_other_leaves(out, leaves)
        if out.requires_grad:
            found = iter(torch.autograd.grad(out, leaves, grad, allow_unused=True))
        else:      # none of them was used
            found = iter([None] * len(leaves))
        return (None, None) + tuple(next(found) if k else None for k in need)


def checkpoint8(fn, x: torch.Tensor, *args) -> torch.Tensor:
    """fn(x, *args), differentiable in x, the tensors among args and, where fn
    is a module or a module's method, the module's parameters; it holds x in 8
    bits and nothing that fn computes: the backward pass reads x back and runs
    fn again. The result is fn's own; the gradients are those of fn at the x
    that was read back. fn must return one tensor and do the same work both
    times (no random numbers, no running statistics); it runs under the forward
    pass's autocast state both times. Every other tensor that needs a gradient
    has to be an argument: one that fn closes over, or that sits in a list
    among args, makes the backward pass raise. Where no gradient of those
    inputs is wanted, fn runs by itself and nothing is held."""
    dtype_code(x, "checkpoint8: x")
    _rows(x, "checkpoint8: x")
    check_cuda(x, "checkpoint8: x")
    params = _parameters(fn)
    if not wants_grad(x, *(a for a in args if torch.is_tensor(a)), *params):
        return _one_tensor(fn(x, *args))
    return _Checkpoint8.apply(fn, len(args), x, *args, *params)

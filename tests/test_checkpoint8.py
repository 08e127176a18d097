"""checkpoint8 as modules, closures and mixed precision use it."""

import functools

import pytest
import torch

from metal_gauss_b200 import activations
from metal_gauss_b200.activations import checkpoint8, pack8
from metal_gauss_b200.labels import label_loss
from metal_gauss_b200.layernorm import layer_norm
from test_features import gen, held8

pytestmark = pytest.mark.gpu


class Head(torch.nn.Module):
    """Normalisation and a label loss whose embeddings the module owns."""

    def __init__(self, channels, classes, seed):
        super().__init__()
        g = gen(seed)
        self.weight = torch.nn.Parameter(torch.randn(channels, generator=g, device="cuda"))
        self.classes = torch.nn.Parameter(torch.randn(classes, channels, generator=g, device="cuda"))
        self.frozen = torch.nn.Parameter(torch.randn(channels, generator=g, device="cuda"),
                                         requires_grad=False)

    def forward(self, x, labels):
        return label_loss(layer_norm(x, self.weight, self.frozen), self.classes, labels)

    def scaled(self, x, labels, scale):
        return label_loss(layer_norm(x, self.weight), self.classes, labels, scale=scale)


def case(seed=1, n=70, d=48, v=9):
    g = gen(seed)
    x = torch.randn(n, d, generator=g, device="cuda", requires_grad=True)
    return x, torch.randint(0, v, (n,), generator=g, device="cuda"), Head(d, v, seed)


@pytest.mark.parametrize("form", ["module", "method", "partial"])
def test_a_modules_parameters_get_their_gradients(cuda, form):
    x, lab, head = case()
    fn, args = {"module": (head, (lab,)), "method": (head.scaled, (lab, 0.5)),
                "partial": (functools.partial(head.scaled, scale=0.5), (lab,))}[form]
    params = (head.weight, head.classes)
    got = torch.autograd.grad(checkpoint8(fn, x, *args) * 3, (x, *params))
    xr = held8(x).requires_grad_(True)
    want = torch.autograd.grad(fn(xr, *args) * 3, (xr, *params))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # through backward(), also where x itself needs no gradient
    (checkpoint8(fn, x.detach(), *args) * 3).backward()
    assert all(torch.equal(p.grad, q) for p, q in zip(params, want[1:]))
    assert head.frozen.grad is None
    # asked for the input's gradient alone
    (gx,) = torch.autograd.grad(checkpoint8(fn, x, *args) * 3, x)
    assert torch.equal(gx, want[0])
    # a parameter that trains no more
    head.weight.requires_grad_(False)
    gx, gc = torch.autograd.grad(checkpoint8(fn, x, *args) * 3, (x, head.classes))
    assert torch.equal(gx, want[0]) and torch.equal(gc, want[2])
    head.weight.requires_grad_(True)
    # a leaf of a module as a plain argument
    w = head.weight
    (got,) = torch.autograd.grad(checkpoint8(lambda t, u: (t * u).sum(), x, w), w)
    want = held8(x).double().sum(0)
    assert float((got.double() - want).abs().max()) <= 72 * 2.0 ** -24 * float(held8(x).abs().sum(0).max())


def test_a_parameter_changed_before_the_backward_pass_is_refused(cuda):
    x, lab, head = case(2)
    loss = checkpoint8(head, x, lab)
    with torch.no_grad():
        head.classes.mul_(2)
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


def test_tensors_that_fn_closes_over_are_refused(cuda):
    """Their gradients would be lost: leaves, results of other operators, a
    module inside a lambda, a tensor in a list."""
    x, lab, head = case(3)
    w = torch.ones(48, device=cuda, requires_grad=True)
    calls = [lambda: checkpoint8(lambda t: layer_norm(t, w), x),
             lambda: checkpoint8(lambda t: t * (w * 2), x),
             lambda: checkpoint8(lambda t: head(t, lab), x),
             lambda: checkpoint8(lambda t, u: t * u * w, x, w),
             lambda: checkpoint8(lambda t, several: t * several[0], x, [w])]
    held = w * 2
    calls.append(lambda: checkpoint8(lambda t: t + held, x))
    for call in calls:
        out = call()
        with pytest.raises(RuntimeError, match="argument"):
            torch.autograd.grad(out.sum(), x)
    # what needs no gradient may be closed over, and so may anything that is detached
    d = w.detach()
    (got,) = torch.autograd.grad(checkpoint8(lambda t: t * d + w.detach(), x).sum(), x)
    assert torch.equal(got, torch.ones_like(x))


def test_a_segment_that_uses_no_input(cuda):
    x, lab, head = case(4)
    y = checkpoint8(lambda t: t.detach() * 2, x)
    assert torch.equal(y, x.detach() * 2)
    (got,) = torch.autograd.grad(y.sum(), x, allow_unused=True)
    assert got is None
    (got,) = torch.autograd.grad(checkpoint8(lambda t: t, x), x, torch.full_like(x, 3.0))
    assert torch.equal(got, torch.full_like(x, 3.0))


@pytest.mark.parametrize("inside", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_segment_runs_again_in_the_forward_passs_precision(cuda, dtype, inside):
    """Mixed precision in the forward pass, the backward pass outside it or in
    another one; the same parameter used beside the segment keeps its own
    gradient."""
    g = gen(5)
    x = torch.randn(64, 48, generator=g, device=cuda, requires_grad=True)
    w = torch.randn(32, 48, generator=g, device=cuda, requires_grad=True)
    seen = []

    def segment(t, u):
        y = torch.nn.functional.linear(t, u)
        seen.append(y.dtype)
        return y.float().square().mean()

    def step(run, t):
        with torch.autocast("cuda", dtype=dtype):
            loss = run(segment, t, w) + torch.nn.functional.linear(x.detach(), w).float().mean()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=inside):
            return loss.detach(), *torch.autograd.grad(loss, (t, w))

    got = step(checkpoint8, x)
    assert seen == [dtype, dtype]
    xr = held8(x).requires_grad_(True)
    want = step(lambda f, *a: f(*a), xr)
    assert torch.equal(got[1], want[1])
    # the two uses of w in one sum: half a step of dtype for each cast gradient
    eps = torch.finfo(dtype).eps
    assert float((got[2] - want[2]).abs().max()) <= 2 * eps * float(want[2].abs().max())
    # and without mixed precision the segment never enters it
    seen.clear()
    loss = checkpoint8(segment, x, w)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        torch.autograd.grad(loss, x)
    assert seen == [torch.float32, torch.float32]


def test_nothing_is_packed_where_no_gradient_is_wanted(cuda, monkeypatch):
    x, lab, head = case(6)
    calls = []

    def counted(t):
        calls.append(t.shape)
        return pack8(t)

    monkeypatch.setattr(activations, "pack8", counted)
    with torch.no_grad():
        assert torch.equal(checkpoint8(head, x, lab), head(x, lab))
    d = x.detach()
    assert torch.equal(checkpoint8(lambda t, k: t * k, d, 2.0), d * 2)
    assert not calls
    # a closure over a module then trains it as it would by itself
    (got,) = torch.autograd.grad(checkpoint8(lambda t: head(t, lab), d), head.classes)
    (want,) = torch.autograd.grad(head(d, lab), head.classes)
    assert torch.equal(got, want) and not calls
    with pytest.raises(TypeError, match="one tensor"):
        checkpoint8(lambda t: (t, t), d)
    assert checkpoint8(head, x, lab).requires_grad and len(calls) == 1


class Doubled(torch.autograd.Function):
    """A user's function with an attribute called variable."""

    @staticmethod
    def forward(ctx, t):
        ctx.variable = torch.zeros(1)
        return t * 2

    @staticmethod
    def backward(ctx, grad):
        return grad * 2


def test_users_functions_and_segments_within_segments(cuda):
    x, lab, head = case(7)
    (got,) = torch.autograd.grad(checkpoint8(lambda t: Doubled.apply(t), x).sum(), x)
    assert torch.equal(got, torch.full_like(x, 2.0))
    # a segment within a segment: both inputs are read back from 8 bits
    params = (head.weight, head.classes)

    class Outer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.head = head

        def forward(self, t):
            return checkpoint8(self.head, t * 1.5, lab)

    got = torch.autograd.grad(checkpoint8(Outer(), x), (x, *params))
    xr = held8(x).requires_grad_(True)
    inner = held8(xr.detach() * 1.5).requires_grad_(True)
    di, *want = torch.autograd.grad(head(inner, lab), (inner, *params))
    assert all(torch.equal(a, b) for a, b in zip(got, (di * 1.5, *want)))

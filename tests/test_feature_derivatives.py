"""Derivatives that layer_norm, label_loss and checkpoint8 do not have are
refused, not dropped."""

import pytest
import torch
from torch.autograd import forward_ad

from metal_gauss_b200.activations import checkpoint8, unpack8, wants_grad
from metal_gauss_b200.labels import label_loss
from metal_gauss_b200.layernorm import layer_norm


def test_an_open_forward_mode_level_goes_through_the_autograd_function():
    x = torch.zeros(3)
    assert not wants_grad(x, None)
    assert wants_grad(x, x.clone().requires_grad_(True))
    with torch.no_grad():
        assert not wants_grad(x.clone().requires_grad_(True))
    with forward_ad.dual_level():
        assert wants_grad(forward_ad.make_dual(x, x)) and wants_grad(x)
        with torch.no_grad():      # which does not switch forward mode off
            assert wants_grad(forward_ad.make_dual(x, x))
    assert not wants_grad(x)


def test_numbers_that_need_a_gradient_are_refused():
    """A learned temperature would get none. (What passes goes on to the next
    refusal, of CPU tensors.)"""
    x, c, lab = torch.zeros(4, 8), torch.zeros(3, 8), torch.zeros(4, dtype=torch.int64)
    k = torch.tensor(0.5, requires_grad=True)
    with pytest.raises(TypeError, match="scale"):
        label_loss(x, c, lab, scale=k)
    with pytest.raises(TypeError, match="eps"):
        layer_norm(x, eps=k)
    for ok in (0.5, torch.tensor(0.5)):
        with pytest.raises(RuntimeError, match="CUDA"):
            label_loss(x, c, lab, scale=ok)
        with pytest.raises(RuntimeError, match="CUDA"):
            layer_norm(x, eps=ok)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        label_loss(x, c, lab, scale=k)


def test_scales_that_need_a_gradient_are_refused():
    codes, scales = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1, requires_grad=True)
    with pytest.raises(TypeError, match="gradient"):
        unpack8(codes, scales)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        unpack8(codes, scales)
    with pytest.raises(RuntimeError, match="CUDA"):
        unpack8(codes, scales.detach())


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused(cuda):
    g = torch.Generator(device=cuda).manual_seed(3)
    x, t = torch.randn(2, 20, 8, generator=g, device=cuda).unbind(0)
    w, c = torch.randn(8, generator=g, device=cuda), torch.randn(6, 8, generator=g, device=cuda)
    b = torch.randn(6, generator=g, device=cuda)
    lab = torch.randint(0, 6, (20,), generator=g, device=cuda)
    plain = layer_norm(x, w, w), label_loss(x, c, lab, bias=b)
    with forward_ad.dual_level():
        def dual(v):
            return forward_ad.make_dual(v, torch.ones_like(v))

        calls = [lambda: layer_norm(dual(x)), lambda: layer_norm(x, dual(w)),
                 lambda: layer_norm(x, w, dual(w), saved="int8"),
                 lambda: label_loss(dual(x), c, lab), lambda: label_loss(x, dual(c), lab),
                 lambda: label_loss(x, c, lab, bias=dual(b)),
                 lambda: checkpoint8(lambda u: u * 2, dual(x))]
        for call in calls:
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
                call()
        # tensors without a tangent are computed as ever
        assert torch.equal(layer_norm(x, w, w), plain[0])
        assert torch.equal(label_loss(x, c, lab, bias=b), plain[1])
    for f in (layer_norm, lambda u: label_loss(u, c, lab)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (t,))

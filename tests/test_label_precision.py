"""How many bits of the logits' gradient G reach dx and dclasses: more than the
features' type has. Embeddings and features lie close to a constant, so that
the products are differences of nearly equal sums: an error of G of 2^-8 of
itself (one bf16 number) would be 2^-3 of the result, far above the result's own
rounding."""

import pytest
import torch

from metal_gauss_b200.labels import label_loss
from test_features import BF16, F16, F32, U, gen, half

pytestmark = pytest.mark.gpu

# What is left out of G: two bf16 parts leave 2^-8 of 2^-8 of an entry; fp16
# embeddings are two parts too, and the product of both second parts (2^-8 of
# each) is not taken. fp32: three parts, and of nine products the six of 2^-24
# and more, in the logits too.
PARTS = {BF16: 2.0 ** -16, F16: 2 * 2.0 ** -16, F32: 6 * U}


def formula(x, w, lab, grad, held=None):
    """dx, dclasses in 64 bits, and the magnitudes that their errors scale with;
    G held in `held`'s type where it is given."""
    x, w, grad = x.double(), w.double(), grad.double()
    z = x @ w.t()
    p = torch.softmax(z, 1)
    G = (p - torch.nn.functional.one_hot(lab, w.shape[0])) * grad[:, None]
    if held is not None:
        G = G.to(held).double()
    return G @ w, G.t() @ x, G.abs() @ w.abs(), G.abs().t() @ x.abs(), (x.abs() @ w.abs().t()).max()


# channels that hold something, channels: on the SM and through scratch
@pytest.mark.parametrize("d", [8, 64, 300, 512])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_the_logits_gradient_is_wider_than_the_features(cuda, d, dtype):
    g = gen(d)
    n, v, used = 3 * 200, 40, 8
    x, w = torch.zeros(n, d, device=cuda), torch.zeros(v, d, device=cuda)
    x[:, :used] = 0.125 * (1 + torch.randn(n, used, generator=g, device=cuda) / 32)
    w[:, :used] = 1 + torch.randn(v, used, generator=g, device=cuda) / 32
    x, w = x.to(dtype), w.to(dtype)
    lab = torch.randint(0, v, (n // 3,), generator=g, device=cuda).repeat_interleave(3)
    grad = torch.tensor([1.0, 0.7, -1.7], device=cuda).repeat(n // 3)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = torch.autograd.grad(label_loss(xl, wl, lab, reduction="none"), (xl, wl), grad)
    dx, dw, mx, mw, mag = formula(x, w, lab, grad)
    # an entry of G: differences of logits of up to `used` products, exp and log: a few u
    rel = 4 * (used + 8) * U * float(mag) + 64 * U + PARTS[dtype]
    tx = (rel + (v + 8) * U) * mx
    tw = (rel + (n + 8) * U) * mw
    tiny = 2.0 ** -25 * (dtype == F16)
    for a, want, t in ((got[0], dx, tx), (got[1], dw, tw)):
        bound = t + half(dtype) * (want.abs() + t) + tiny
        assert ((a.double() - want).abs() <= bound).all()
    # G in one number of the 16-bit type would be outside
    if dtype != F32:
        one = formula(x, w, lab, grad, BF16)
        for a, want, t in ((one[0], dx, tx), (one[1], dw, tw)):
            off = (a - want).abs() > t + half(dtype) * (want.abs() + t) + tiny
            assert off[:, :used].double().mean() > 0.1

"""layer_norm, pack8 and label_loss read nothing of a workspace or an output
that they have not written: every tensor that they allocate holds 0xFF bytes
(a NaN in each floating type) before the call."""

import pytest
import torch

from metal_gauss_b200.activations import pack8, unpack8
from metal_gauss_b200.layernorm import layer_norm
from test_features import BF16, F16, F32, check_label, gen, label_case

pytestmark = pytest.mark.gpu


@pytest.fixture
def poisoned(monkeypatch):
    """torch.empty and torch.empty_like give memory full of NaN."""
    def fill(make):
        def run(*args, **kw):
            t = make(*args, **kw)
            if t.is_cuda and t.numel():
                t.view(-1).view(torch.uint8).fill_(255)
            return t
        return run

    monkeypatch.setattr(torch, "empty", fill(torch.empty))
    monkeypatch.setattr(torch, "empty_like", fill(torch.empty_like))
    assert torch.empty(3, device="cuda").isnan().all()


@pytest.mark.parametrize("n,d,v,dtype", [
    (36_000, 140, 1_280, F32),   # two pieces of several shares of the bias's gradient, the last short
    (36_000, 200, 1_900, F16),
    (36_000, 264, 1_900, BF16),
    (80_000, 264, 1_000, BF16),
    (2_600, 200, 20_000, F16),   # two pieces of one share
    (36_864, 140, 1_100, F32),   # one piece of two shares
    (700, 300, 90, F32),         # one piece of one share
    (300, 300, 40_000, F32),     # the classes in shares
    (40_000, 16, 200, F32),      # the logits' gradient stays on the SM
    (1_000, 100, 129, F32), (3, 20, 5_000, F16), (20_000, 24, 4_300, BF16), (257, 77, 513, BF16),
])
def test_label_loss_reads_what_it_wrote(cuda, poisoned, n, d, v, dtype):
    x, w, lab, bias, _ = label_case(n + 3 * d + v, n, d, v, dtype)
    check_label(x, w, lab, bias)


@pytest.mark.parametrize("saved", ["full", "int8"])
@pytest.mark.parametrize("n,d,dtype", [(1, 1, F32), (300, 77, F32), (5_000, 64, BF16), (40, 601, F16),
                                       (12_000, 1_025, F32), (300, 512, BF16), (9, 8_191, F16)])
def test_layer_norm_and_pack8_read_what_they_wrote(cuda, poisoned, n, d, dtype, saved):
    g = gen(n + d)
    x = torch.randn(n, d, generator=g, device=cuda).to(dtype).requires_grad_(True)
    w = torch.randn(d, generator=g, device=cuda).to(dtype).requires_grad_(True)
    y = layer_norm(x, w, w, saved=saved)
    grads = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert all(t.isfinite().all() for t in (y, *grads))
    codes, scales = pack8(x)
    assert scales.isfinite().all() and unpack8(codes, scales).isfinite().all()

"""layer_norm and label_loss called as a program calls them: whatever ran
before, at once on two streams, captured, on a padded batch."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent

ORDER = """
import hashlib, sys, torch
from metal_gauss_b200.layernorm import layer_norm
for d in map(int, sys.argv[1:]):
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(4000, d, generator=g, device="cuda", requires_grad=True)
    w = torch.randn(d, generator=g, device="cuda", requires_grad=True)
    y = layer_norm(x, w, w)
    out = [y.detach(), *torch.autograd.grad(y, (x, w), torch.ones_like(y))]
    print(d, *(hashlib.sha256(t.cpu().numpy().tobytes()).hexdigest() for t in out))
"""


def test_layer_norm_gives_the_same_bits_whatever_length_came_first(cuda):
    """Lengths that share a kernel, in two orders in two processes."""
    lengths = ["520", "1024", "516", "768", "33", "64", "40"]
    runs = [subprocess.run([sys.executable, "-c", ORDER, *order], cwd=ROOT, capture_output=True,
                           text=True, check=True).stdout.split("\n")
            for order in (lengths, lengths[::-1])]
    assert len(runs[0]) == len(lengths) + 1 and sorted(runs[0]) == sorted(runs[1])

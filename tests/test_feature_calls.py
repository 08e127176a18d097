"""layer_norm and label_loss called as a program calls them: whatever ran
before, at once on two streams, captured, on a padded batch."""

import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from metal_gauss_b200.activations import checkpoint8
from metal_gauss_b200.labels import label_loss
from metal_gauss_b200.layernorm import layer_norm
from test_features import BF16, F16, F32, check_label, gen, label_case

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


# features too wide for the logits' gradient to stay on the SM, and one that is not
WIDE = [(F32, 900, 200, 300), (BF16, 700, 300, 90), (F16, 1_500, 260, 700), (BF16, 3_000, 512, 1_000),
        (F32, 2_000, 64, 300)]


def loss_case(dtype, n, d, v):
    return label_case(n + d + v, n, d, v, dtype)[:4]


def loss_grads(x, w, lab, bias):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, bias)]
    loss = label_loss(leaves[0], leaves[1], lab, bias=leaves[2])
    return [loss.detach(), *torch.autograd.grad(loss, leaves)]


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b, strict=True))


@pytest.mark.parametrize("dtype,n,d,v", WIDE)
def test_equal_calls_give_equal_bits(cuda, dtype, n, d, v):
    args = loss_case(dtype, n, d, v)
    want = loss_grads(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = loss_grads(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert same(want, got) and same(want, loss_grads(*args))


def test_wide_calls_at_once_on_several_streams(cuda):
    cases = [loss_case(*c) for c in WIDE]
    want = [loss_grads(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(loss_grads(*c))
    torch.cuda.synchronize()
    assert all(same(g, want[i % len(cases)]) for i, g in enumerate(got))


def test_calls_at_once_from_several_threads(cuda):
    cases = [loss_case(*c) for c in WIDE]
    want = [loss_grads(*c) for c in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i].append(loss_grads(*cases[i]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(g) == 5 and all(same(q, w) for q in g) for g, w in zip(got, want))


def capture(make):
    """make() run once on a side stream, then captured."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        make()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = make()
    return graph, out


def test_wide_calls_captured_and_replayed_in_turn(cuda):
    captured = []
    for c in WIDE:
        x, w, lab, bias = loss_case(*c)
        leaves = [t.clone().requires_grad_(True) for t in (x, w, bias)]

        def make(leaves=leaves, lab=lab):
            loss = label_loss(leaves[0], leaves[1], lab, bias=leaves[2])
            return [loss.detach(), *torch.autograd.grad(loss, leaves)]

        captured.append((*capture(make), leaves, lab, (x, w, bias)))
    for rep in range(3):
        for graph, out, leaves, lab, first in captured:
            with torch.no_grad():
                for t, f in zip(leaves, first):
                    t.copy_(f * (1 + 0.1 * rep))
            graph.replay()
        for graph, out, leaves, lab, first in captured:
            assert same(out, loss_grads(leaves[0], leaves[1], lab, leaves[2]))


def test_checkpoint8_of_a_module_captured_and_replayed(cuda):
    x, c, lab, _ = loss_case(F32, 900, 24, 60)
    norm = torch.nn.Linear(24, 24, device=cuda)
    leaves = [x.clone().requires_grad_(True), c.clone().requires_grad_(True)]

    class Head(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = norm

        def forward(self, t, u):
            return label_loss(layer_norm(self.norm(t)), u, lab)

    head = Head()
    need = [*leaves, norm.weight, norm.bias]

    def make():
        loss = checkpoint8(head, *leaves)
        return [loss.detach(), *torch.autograd.grad(loss, need)]

    graph, out = capture(make)
    for rep in range(2):
        with torch.no_grad():
            leaves[0].copy_(x * (1 + 0.2 * rep))
        graph.replay()
        assert same(out, make())


@pytest.mark.parametrize("dtype,d", [(F32, 200), (BF16, 300), (F16, 260)])
def test_wide_calls_after_a_loss_of_nans(cuda, dtype, d):
    """NaN in every score, in G and in the products of an earlier call."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    bad = torch.full((sms * 128, d), math.nan, dtype=dtype, device=cuda).requires_grad_(True)
    wide = torch.randn(512, d, generator=gen(30), device=cuda).to(dtype).requires_grad_(True)
    zeros = torch.zeros(sms * 128, dtype=torch.int64, device=cuda)
    for v in (1, 5, 17, 33, 65, 130, 300):
        rows = label_loss(bad, wide, zeros, reduction="sum")
        assert all(t.isnan().any() for t in torch.autograd.grad(rows, (bad, wide)))
        x, w, lab, bias, _ = label_case(31 + v, 300, d, v, dtype)
        check_label(x, w, lab, bias)


def test_a_padded_batch_is_the_batch_without_its_padding(cuda):
    """Rows behind the last pixel are labelled with the ignored value and hold
    NaN: the loss and the gradients are the formula's without them, theirs is 0."""
    for c in WIDE:
        x, w, lab, bias = loss_case(*c)
        n = x.shape[0]
        x = torch.cat([x, torch.full((37, x.shape[1]), math.nan, dtype=x.dtype, device=cuda)])
        lab = torch.cat([lab, torch.full((37,), -100, device=cuda)])
        _, grads = check_label(x, w, lab, bias)
        assert not grads[0][n:].any()

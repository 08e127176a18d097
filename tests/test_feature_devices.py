"""Workspaces are sized for the device that the tensors are on. Two devices
with different numbers of SMs are played by a library and a current device of
the test's own."""

import contextlib

import pytest
import torch

from metal_gauss_b200 import _lib, labels, layernorm


class Devices:
    """`current` is what the C side would see."""

    def __init__(self, monkeypatch, sms):
        self.current, self.sms, self.asked = 0, sms, []
        monkeypatch.setattr(_lib, "load", lambda: self)
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: self.current, raising=False)
        monkeypatch.setattr(torch.cuda, "device", self.switch)

    @contextlib.contextmanager
    def switch(self, index):
        before, self.current = self.current, index
        yield
        self.current = before

    def mg_label_loss_scratch_bytes(self, *sizes):
        self.asked.append((self.current, sizes))
        return self.sms[self.current] * 256 + sum(sizes)

    mg_layer_norm_backward_scratch_bytes = mg_label_loss_scratch_bytes


@pytest.mark.parametrize("module,sizes", [(labels, (10, 8, 4, 0, 1)), (layernorm, (10, 8))])
def test_scratch_sizes_belong_to_a_device(monkeypatch, module, sizes):
    d = Devices(monkeypatch, sms=(148, 132))
    size = type(module._SCRATCH)(module._SCRATCH.name)     # one that knows no size yet
    for current in (0, 1):
        d.current = current
        for device in (1, 0, 1):
            assert size(device, *sizes) == d.sms[device] * 256 + sum(sizes)
            assert d.current == current
    assert sorted(d.asked) == [(0, sizes), (1, sizes)]     # asked once for each


def test_scratch_sizes_are_kept_for_a_bounded_number_of_shapes(monkeypatch):
    d = Devices(monkeypatch, sms=(148,))
    size = _lib.SizeOf("mg_layer_norm_backward_scratch_bytes")
    for n in range(1000):
        assert size(0, n, 8) == 148 * 256 + n + 8
    assert len(size.known) <= 256 and len(d.asked) == 1000

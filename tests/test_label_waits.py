"""The bounded waits of label_loss's tensor-core tiles, exercised without a
fault: mg_label_loss_wait_selftest runs the passes with tiles that are never
copied in, so that the waits for them run out. The kernels return promptly,
code 4 can be read, nothing that such a wait was for looks like a result, and
the calls after it are right."""

import time

import pytest
import torch

from metal_gauss_b200 import _lib, ext
from metal_gauss_b200._lib import ptr
from test_features import BF16, F16, F32, check_label, label_case

CODE = {F32: 0, BF16: 1, F16: 2}
ROUNDS = 32


def run(x, w, lab, units, rounds=ROUNDS):
    """Forward, and backward on the statistics of a whole forward pass."""
    lib = _lib.load()
    (n, d), v, code = x.shape, w.shape[0], CODE[x.dtype]
    loss, stats = torch.zeros(n, device="cuda"), torch.zeros(2 * n, device="cuda")
    unused = torch.zeros(2 * n, device="cuda")
    grad = torch.ones(n, device="cuda")
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(v, device="cuda")
    size = max(lib.mg_label_loss_scratch_bytes(n, d, v, code, back) for back in (0, 1))
    scratch = torch.zeros(size, dtype=torch.uint8, device="cuda")
    tail = (ptr(scratch), size, _lib.stream())
    _lib.call("mg_label_loss_forward", ptr(x), ptr(w), code, None, ptr(lab), 8, -100, n, d, v, 1.0,
              0, ptr(loss), ptr(stats), None, *tail)
    whole = loss.clone()
    args = (rounds, units, ptr(x), ptr(w), code, ptr(lab), n, d, v)
    _lib.call("mg_label_loss_wait_selftest", *args, ptr(loss), ptr(unused), None, None, None, None,
              *tail)
    forward_code = ext.device_error()
    _lib.call("mg_label_loss_wait_selftest", *args, None, ptr(stats), ptr(grad), ptr(dx), ptr(dw),
              ptr(db), *tail)
    return whole, loss, (dx, dw, db), forward_code, ext.device_error()


SHAPES = [(700, 24, 60, F32),       # classes resident, the logits' gradient on the SM
          (700, 100, 300, F32), (2_000, 64, 300, BF16), (500, 150, 700, F16),
          (3, 20, 5_000, F32),      # the classes in shares
          (700, 300, 90, BF16),     # the logits' gradient through scratch
          (300, 200, 700, F32), (900, 260, 400, F16)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v,dtype", SHAPES)
def test_waits_that_run_out_leave_nan_and_code_4(cuda, n, d, v, dtype):
    assert ext.device_error() == 0
    x, w, lab, bias, _ = label_case(n + d + v, n, d, v, dtype)
    lab[0] = 0
    t0 = time.perf_counter()
    whole, loss, grads, fcode, bcode = run(x, w, lab, 0)
    assert time.perf_counter() - t0 < 20.0
    assert fcode == 4 and bcode == 4
    live = lab != -100
    assert whole.isfinite().all()
    assert loss[live].isnan().all() and not loss[~live].any()
    assert all(g.isnan().all() for g in grads)
    # nothing of it reaches the next call
    check_label(x, w, lab, bias)
    assert ext.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d,v,dtype", [(24, 60, F32), (64, 300, BF16), (300, 90, BF16)])
def test_what_was_computed_before_a_wait_ran_out_is_right_or_nan(cuda, d, v, dtype):
    """One unit of each block gets its tiles, those after it none."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = 3 * sms * 128
    x, w, lab, bias, _ = label_case(d + v, n, d, v, dtype)
    whole, loss, (dx, _, _), fcode, bcode = run(x, w, lab, sms)
    assert fcode == 4 and bcode == 4
    bad = loss.isnan()
    assert bad.any() and torch.equal(loss[~bad], whole[~bad])
    xl = x.clone().requires_grad_(True)
    from metal_gauss_b200.labels import label_loss
    rows = label_loss(xl, w, lab, reduction="none")
    (want,) = torch.autograd.grad(rows, xl, torch.ones_like(rows))
    bad = dx.isnan()
    assert bad.any() and torch.equal(dx[~bad], want[~bad])
    assert ext.device_error() == 0


def test_the_selftest_refuses_limits_outside_its_range():
    """No CUDA call is made."""
    lib, one = _lib.load(), 256
    call = lambda **k: lib.mg_label_loss_wait_selftest(*{**dict(                # noqa: E731
        rounds=1, units=0, x=one, w=one, dtype=0, lab=one, rows=4, ch=8, v=3, loss=one, stats=one,
        g=None, dx=None, dw=None, db=None, scr=one, nb=1 << 30, st=None), **k}.values())
    assert [call(rounds=0), call(rounds=4097), call(units=-1), call(rows=0),
            call(rows=(1 << 20) + 1), call(ch=513), call(loss=None), call(stats=None),
            call(g=one), call(scr=None), call(nb=8), call(dtype=4)] == [1] * 12

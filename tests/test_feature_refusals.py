"""What layer_norm, pack8 / unpack8 / checkpoint8 and label_loss refuse, in
Python and at the C entry points. Needs no GPU: every refusal comes before
the first CUDA call."""

import pytest
import torch

from metal_gauss_b200 import _lib
from metal_gauss_b200.activations import checkpoint8, pack8, unpack8
from metal_gauss_b200.labels import label_loss
from metal_gauss_b200.layernorm import layer_norm


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused_not_moved():
    for call in (lambda: layer_norm(z(4, 8)), lambda: pack8(z(4, 8)),
                 lambda: unpack8(z(4, 8, dtype=torch.int8), z(4, 1)),
                 lambda: checkpoint8(lambda t: t, z(4, 8)),
                 lambda: label_loss(z(4, 8), z(3, 8), z(4, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("kw,err", [
    (dict(x=z(4, 8, dtype=torch.float64)), TypeError),
    (dict(x=z(4, 0)), ValueError),
    (dict(x=torch.tensor(1.0)), ValueError),
    (dict(x=z(2, 8193)), ValueError),
    (dict(x=z(4, 8), weight=z(7)), ValueError),
    (dict(x=z(4, 8), bias=z(1, 8)), ValueError),
    (dict(x=z(4, 8), weight=z(8, dtype=torch.float16)), TypeError),
    (dict(x=z(4, 8, dtype=torch.bfloat16), weight=z(8), bias=z(8, dtype=torch.bfloat16)), TypeError),
    (dict(x=z(4, 8), eps=-1.0), ValueError),
    (dict(x=z(4, 8), eps=float("nan")), ValueError),
    (dict(x=z(4, 8), saved="int4"), ValueError),
])
def test_layer_norm_refuses(kw, err):
    with pytest.raises(err):
        layer_norm(**kw)


@pytest.mark.parametrize("call,err", [
    (lambda: pack8(z(4, 8, dtype=torch.int32)), TypeError),
    (lambda: pack8(z(4, 0)), ValueError),
    (lambda: unpack8(z(4, 8), z(4, 1)), TypeError),
    (lambda: unpack8(z(4, 8, dtype=torch.int8), z(4, 1, dtype=torch.float16)), TypeError),
    (lambda: unpack8(z(4, 8, dtype=torch.int8), z(4, 2)), ValueError),
    (lambda: unpack8(z(4, 129, dtype=torch.int8), z(4, 1)), ValueError),
    (lambda: unpack8(z(4, 8, dtype=torch.int8), z(4, 1), dtype=torch.float64), TypeError),
    (lambda: checkpoint8(lambda t: t, z(4, 8, dtype=torch.float64)), TypeError),
])
def test_8_bit_form_refuses(call, err):
    with pytest.raises(err):
        call()


L = torch.int64


@pytest.mark.parametrize("args,kw,err", [
    ((z(4, 8, dtype=torch.float64), z(3, 8, dtype=torch.float64), z(4, dtype=L)), {}, TypeError),
    ((z(4, 8), z(3, 8, dtype=torch.bfloat16), z(4, dtype=L)), {}, TypeError),
    ((z(4, 8), z(3, 7), z(4, dtype=L)), {}, ValueError),
    ((z(4, 8), z(0, 8), z(4, dtype=L)), {}, ValueError),
    ((z(4, 8), z(8), z(4, dtype=L)), {}, ValueError),
    ((z(4, 513), z(3, 513), z(4, dtype=L)), {}, ValueError),
    ((z(4, 8), z(3, 8), z(5, dtype=L)), {}, ValueError),
    ((z(2, 2, 8), z(3, 8), z(4, dtype=L)), {}, ValueError),
    ((z(4, 8), z(3, 8), z(4, dtype=torch.int16)), {}, TypeError),
    ((z(4, 8), z(3, 8), z(4)), {}, TypeError),
    ((z(4, 8), z(3, 8), z(4, dtype=L)), dict(bias=z(4)), ValueError),
    ((z(4, 8), z(3, 8), z(4, dtype=L)), dict(bias=z(3, dtype=torch.float16)), TypeError),
    ((z(4, 8), z(3, 8), z(4, dtype=L)), dict(reduction="max"), ValueError),
])
def test_label_loss_refuses(args, kw, err):
    with pytest.raises(err):
        label_loss(*args, **kw)


def test_c_entry_points_refuse():
    """Statuses come back; nothing throws, aborts or touches a device."""
    L = _lib.load()
    one, f, s0 = 256, 0.0, None      # a non-null, 256-byte aligned address never dereferenced
    bad, cap = 1, 2
    ln = lambda **k: L.mg_layer_norm_forward(*{**dict(                         # noqa: E731
        x=one, dtype=0, w=one, b=one, pd=0, rows=4, ch=8, eps=1e-5, y=one, m=one, r=one, c=None,
        s=None, st=s0), **k}.values())
    assert [ln(dtype=3), ln(pd=-1), ln(rows=-1), ln(ch=0), ln(ch=8193), ln(eps=-1.0), ln(m=None),
            ln(s=one), ln(x=None), ln(c=257, s=one)] == [bad] * 10
    assert ln(rows=0) == 0
    lb = lambda **k: L.mg_layer_norm_backward(*{**dict(                        # noqa: E731
        dy=one, x=one, c=None, s=None, dtype=0, w=one, pd=0, m=one, r=one, rows=4, ch=8, dx=one,
        dw=one, db=one, scr=one, nb=1 << 20, st=s0), **k}.values())
    assert [lb(dtype=9), lb(ch=9000), lb(x=None), lb(c=one, s=one), lb(x=None, c=one), lb(dy=None),
            lb(m=None), lb(nb=16), lb(scr=None), lb(rows=-2)] == [bad] * 10
    assert L.mg_layer_norm_backward_scratch_bytes(0, 8) == 0
    assert L.mg_layer_norm_backward_scratch_bytes(10, 9000) == 0
    pk = lambda **k: L.mg_pack8(*{**dict(x=one, dtype=0, rows=4, ch=8, c=one, s=one,   # noqa: E731
                                         st=s0), **k}.values())
    assert [pk(dtype=7), pk(rows=-1), pk(ch=0), pk(x=None), pk(c=None), pk(s=None),
            pk(c=260)] == [bad] * 7
    assert pk(rows=1 << 40) == cap and pk(rows=0) == 0
    up = lambda **k: L.mg_unpack8(*{**dict(c=one, s=one, rows=4, ch=8, dtype=0, x=one,  # noqa: E731
                                           st=s0), **k}.values())
    assert [up(dtype=7), up(rows=-1), up(ch=0), up(x=None), up(c=None), up(c=260)] == [bad] * 6
    lf = lambda **k: L.mg_label_loss_forward(*{**dict(                         # noqa: E731
        x=one, w=one, dtype=0, b=None, lab=one, lb=8, ign=-100, rows=4, ch=8, v=3, sc=1.0, red=1,
        loss=one, stats=None, live=None, scr=one, nb=1 << 30, st=s0), **k}.values())
    assert [lf(dtype=5), lf(lb=2), lf(red=3), lf(rows=-1), lf(ch=0), lf(ch=513), lf(v=0),
            lf(v=(1 << 20) + 1), lf(x=None), lf(w=None), lf(lab=None), lf(loss=None), lf(scr=None),
            lf(scr=264), lf(nb=8)] == [bad] * 15
    assert lf(rows=(1 << 30) + 1) == cap
    gb = lambda **k: L.mg_label_loss_backward(*{**dict(                        # noqa: E731
        x=one, w=one, dtype=0, b=None, lab=one, lb=8, ign=-100, rows=4, ch=8, v=3, sc=1.0, red=1,
        g=one, stats=one, live=one, dx=one, dw=one, db=None, scr=one, nb=1 << 30, st=s0),
        **k}.values())
    assert [gb(dtype=5), gb(lb=3), gb(red=-1), gb(g=None), gb(stats=None), gb(live=None),
            gb(scr=None), gb(scr=128), gb(nb=8), gb(dx=264), gb(dw=264)] == [bad] * 11
    assert L.mg_label_loss_scratch_bytes(0, 8, 8, 0, 0) == 0
    assert L.mg_label_loss_scratch_bytes(8, 600, 8, 0, 0) == 0
    assert b"label_loss" in L.mg_last_error()

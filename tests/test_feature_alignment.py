"""The C entry points on feature maps refuse an address off its element's
boundary, which would fault on the device. No CUDA call is made."""

from metal_gauss_b200 import _lib

BAD = 1          # MG_ERR_INVALID_ARGUMENT
AT = 4096        # an address on every boundary, never dereferenced


def statuses(fn, base, off):
    return {k: fn(*{**base, k: AT + by}.values()) for k, by in off.items()}


def refused(fn, base, off):
    got = statuses(fn, base, off)
    assert got == dict.fromkeys(off, BAD), got
    assert b"boundary" in _lib.load().mg_last_error()


def test_addresses_off_their_elements_boundary_are_refused():
    lib = _lib.load()
    for dtype, by in ((0, 2), (1, 1), (2, 1)):
        refused(lib.mg_pack8, dict(x=AT, dtype=dtype, rows=4, ch=8, c=AT, s=AT, st=None),
                dict(x=by, s=2))
        refused(lib.mg_unpack8, dict(c=AT, s=AT, rows=4, ch=8, dtype=dtype, x=AT, st=None),
                dict(x=by, s=1))
        refused(lib.mg_layer_norm_forward,
                dict(x=AT, dtype=dtype, w=AT, b=AT, pd=dtype, rows=4, ch=8, eps=1e-5, y=AT, m=AT,
                     r=AT, c=AT, s=AT, st=None),
                dict(x=by, w=by, b=by, y=by, m=2, r=2, s=2))
        refused(lib.mg_layer_norm_backward,
                dict(dy=AT, x=AT, c=None, s=None, dtype=dtype, w=AT, pd=dtype, m=AT, r=AT, rows=4,
                     ch=8, dx=AT, dw=AT, db=AT, scr=AT, nb=1 << 20, st=None),
                dict(dy=by, x=by, w=by, m=2, r=2, dx=by, dw=by, db=by, scr=2))
        for size in (4, 8):
            refused(lib.mg_label_loss_forward,
                    dict(x=AT, w=AT, dtype=dtype, b=AT, lab=AT, lb=size, ign=-100, rows=4, ch=8,
                         v=3, sc=1.0, red=1, loss=AT, stats=AT, live=AT, scr=AT, nb=1 << 30,
                         st=None),
                    dict(x=by, w=by, b=2, lab=size // 2, loss=2, stats=2, live=2))
            refused(lib.mg_label_loss_backward,
                    dict(x=AT, w=AT, dtype=dtype, b=AT, lab=AT, lb=size, ign=-100, rows=4, ch=8,
                         v=3, sc=1.0, red=1, g=AT, stats=AT, live=AT, dx=AT, dw=AT, db=AT, scr=AT,
                         nb=1 << 30, st=None),
                    dict(x=by, w=by, b=2, lab=size // 2, g=2, stats=2, live=2, db=2))

"""layer_norm, the 8-bit activation checkpoints and label_loss against plain
64-bit implementations.

Tolerances are counted, not tuned. u = 2^-24 is half a step of fp32, h half a
step of the tensor's type (finfo.eps / 2). A sum of n products in any order is
off by at most (n + 2) u times the sum of their magnitudes; a result rounded to
its type by h times itself. Each bound below adds those terms up from 64-bit
magnitudes of the same case."""

import math

import pytest
import torch

from metal_gauss_b200 import _lib, ext
from metal_gauss_b200.activations import checkpoint8, pack8, unpack8
from metal_gauss_b200.cuda_backend import render
from metal_gauss_b200.labels import label_loss
from metal_gauss_b200.layernorm import layer_norm

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    off = (got - want).abs() - tol
    bad = ~(off <= 0) & ~(got.isnan() & want.isnan())
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of tolerance, worst " \
                          f"{float((got - want).abs().max()):.3e} against {float(tol.max()):.3e}"


# ------------------------------------------------------------------ layer norm

def norm64(x, w, b, eps, held, dy):
    """y, dx, dw, db in 64 bits and their bounds (fp32 work on a row of d)."""
    x, held, dy = x.double(), held.double(), dy.double()
    n, d = x.shape
    w64 = torch.ones(d, device=x.device).double() if w is None else w.double()
    b64 = torch.zeros(d, device=x.device).double() if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    y = h * w64 + b64
    hh = (held - mean) * rstd
    g = dy * w64
    dx = rstd * (g - g.mean(1, keepdim=True) - hh * (g * hh).mean(1, keepdim=True))
    # a row sum of d terms: (d + 2) u of the magnitudes; mean, then rstd, then h
    k = (d + 16) * U
    spread = x.abs().mean(1, keepdim=True) * rstd
    # the deviation's error carries the mean's: relative to the deviation
    a = k * (2 * spread + 2 * hh.abs().maximum(h.abs())) + k * spread * hh.abs()
    ty = a * w64.abs() + 4 * U * (h * w64).abs() + 2 * U * y.abs()
    gm, ghm = g.abs().mean(1, keepdim=True), (g * hh).abs().mean(1, keepdim=True)
    tdx = rstd * (k * (g.abs() + gm + hh.abs() * ghm) + a * ghm
                  + hh.abs() * (g.abs() * a).mean(1, keepdim=True) + 8 * U * (g.abs() + gm)) \
        + k * (1 + spread) * dx.abs()
    kn = (n + 8) * U
    tdw = kn * (dy * hh).abs().sum(0) + (dy.abs() * a).sum(0)
    tdb = kn * dy.abs().sum(0)
    return (y, dx, (dy * hh).sum(0), dy.sum(0)), (ty, tdx, tdw, tdb)


def held8(x):
    return unpack8(*pack8(x))


NORM = [(1, 1), (1, 512), (2, 3), (5, 7), (33, 16), (17, 64), (300, 77), (1000, 128), (65, 129),
        (64, 512), (31, 520), (9, 1000), (40, 1024), (7, 1025), (12, 1028), (5, 2048), (3, 4100),
        (3, 8192), (2, 8191), (5000, 32)]


@pytest.mark.parametrize("saved", ["full", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,d", NORM)
def test_layer_norm(cuda, n, d, dtype, saved):
    g = gen(n * 10007 + d)
    x = (torch.randn(n, d, generator=g, device=cuda) + 0.5).to(dtype).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(d, generator=g, device=cuda)).to(dtype).requires_grad_(True)
    b = torch.randn(d, generator=g, device=cuda).to(dtype).requires_grad_(True)
    dy = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    y = layer_norm(x, w, b, saved=saved)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    held = x.detach() if saved == "full" else held8(x)
    want, tol = norm64(x.detach(), w.detach(), b.detach(), 1e-5, held, dy)
    for got, ref, t, what in zip((y.detach(), *grads), want, tol, ("y", "dx", "dw", "db")):
        assert got.dtype == dtype
        # half a step of the smallest subnormal of fp16 besides the relative half step
        within(got, ref, t + half(dtype) * (ref.abs() + t) + 2.0 ** -25 * (dtype == F16), what)


@pytest.mark.parametrize("saved", ["full", "int8"])
@pytest.mark.parametrize("n,d,dtype", [(200_001, 19, F32), (60_000, 77, BF16), (30_001, 601, F16),
                                       (100_003, 64, F32), (20_000, 1000, BF16), (12_000, 1025, F32)])
def test_layer_norm_of_many_rows(cuda, n, d, dtype, saved):
    """Blocks that take several chunks or rounds of rows each."""
    test_layer_norm(cuda, n, d, dtype, saved)


@pytest.mark.parametrize("dtype,wdtype", [(BF16, F32), (F16, F32), (F32, F32)])
def test_layer_norm_parameter_types_and_absent_parameters(cuda, dtype, wdtype):
    g = gen(3)
    n, d = 50, 48
    x = torch.randn(n, d, generator=g, device=cuda).to(dtype).requires_grad_(True)
    dy = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    for has_w, has_b in ((1, 1), (1, 0), (0, 1), (0, 0)):
        w = torch.randn(d, generator=g, device=cuda).to(wdtype).requires_grad_(True) if has_w else None
        b = torch.randn(d, generator=g, device=cuda).to(wdtype).requires_grad_(True) if has_b else None
        y = layer_norm(x, w, b, eps=1e-3)
        leaves = [t for t in (x, w, b) if t is not None]
        grads = torch.autograd.grad(y, leaves, dy)
        want, tol = norm64(x.detach(), w and w.detach() if w is None else w.detach(),
                           None if b is None else b.detach(), 1e-3, x.detach(), dy)
        keep = [True, True, has_w, has_b]
        want = [v for v, k in zip(want, keep) if k]
        tol = [v for v, k in zip(tol, keep) if k]
        for got, ref, t in zip((y.detach(), *grads), want, tol):
            within(got, ref, t + half(got.dtype) * (ref.abs() + t) + 2.0 ** -25, "value")
        assert all(q.dtype == leaf.dtype for q, leaf in zip(grads, leaves))


def test_layer_norm_gradient_against_differences(cuda):
    """The 64-bit formula's derivative along a direction, by central
    differences of the 64-bit function (error O(step^2) and rounding), and
    the kernel's gradient along it."""
    g = gen(8)
    x = torch.randn(6, 40, generator=g, device=cuda)
    w, b = torch.randn(2, 40, generator=g, device=cuda).unbind(0)
    dy, dirn = torch.randn(2, 6, 40, generator=g, device=cuda).unbind(0)

    def f(t):
        t = t.double()
        c = t - t.mean(1, keepdim=True)
        return ((c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * w + b) * dy).sum()

    e = 1e-5
    slope = float((f(x.double() + e * dirn) - f(x.double() - e * dirn)) / (2 * e))
    xl = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(layer_norm(xl, w, b), xl, dy)
    got = float((dx.double() * dirn).sum())
    # third derivatives of order |dir|^3 / std^3 ~ 10^2 times step^2; fp32 work on 40 channels
    size = float((dx.double().abs() * dirn.abs()).sum())
    assert abs(got - slope) <= 1e-6 + 100 * U * size


def test_layer_norm_strides_offsets_and_empty(cuda):
    g = gen(4)
    base = torch.randn(40, 70, generator=g, device=cuda)
    w = torch.randn(33, generator=g, device=cuda)
    x = base[::2, 1:67:2]                       # strides 140 and 2, odd offset
    want = layer_norm(x.contiguous(), w)
    assert torch.equal(layer_norm(x, w), want)
    flat = torch.randn(10 * 64 + 1, generator=g, device=cuda)
    x = flat[1:].view(10, 64)                   # contiguous, 4 bytes off a 16-byte boundary
    ref, tol = norm64(x, None, None, 1e-5, x, x)
    within(layer_norm(x), ref[0], tol[0] + half(F32) * ref[0].abs(), "offset view")
    for shape in ((0, 16), (3, 0, 16)):
        e = torch.zeros(shape, device=cuda, requires_grad=True)
        w = torch.ones(16, device=cuda, requires_grad=True)
        for saved in ("full", "int8"):
            y = layer_norm(e, w, saved=saved)
            assert y.shape == shape
            gx, gw = torch.autograd.grad(y.sum(), (e, w))
            assert gx.shape == shape and torch.equal(gw, torch.zeros_like(gw))
    x = torch.randn(2, 3, 5, 24, generator=g, device=cuda)
    assert torch.equal(layer_norm(x).view(30, 24), layer_norm(x.view(30, 24)))
    # a gradient that is a broadcast (stride 0)
    x.requires_grad_(True)
    (a,) = torch.autograd.grad(layer_norm(x).sum(), x)
    (b,) = torch.autograd.grad(layer_norm(x), x, torch.ones_like(x))
    assert torch.equal(a, b)


def test_layer_norm_keeps_rows_apart_and_flat_rows_finite(cuda):
    """A NaN or infinite row spoils that row alone; a constant row has h = 0
    and y = b."""
    g = gen(5)
    x = torch.randn(64, 96, generator=g, device=cuda)
    b = torch.randn(96, generator=g, device=cuda)
    clean = layer_norm(x, None, b)
    y = x.clone()
    y[3, 5], y[10, 0], y[20] = math.nan, math.inf, 7.25
    out = layer_norm(y, None, b)
    keep = torch.ones(64, dtype=torch.bool, device=cuda)
    keep[[3, 10, 20]] = False
    assert torch.equal(out[keep], clean[keep])
    assert out[3].isnan().all() and out[10].isnan().all() and torch.equal(out[20], b)


# ------------------------------------------------------------------ 8 bits

PACK = [(1, 1), (3, 19), (50, 32), (7, 127), (7, 128), (7, 129), (5, 256), (4, 300), (2, 1000),
        (1000, 64), (257, 5), (1, 5000)]


def pack_plain(x):
    """The documented steps on the host, each one correctly rounded fp32."""
    x = x.float().cpu()
    n, d = x.shape
    codes, scales = [], []
    for c in range(0, d, 128):
        p = x[:, c:c + 128]
        a = p.abs().amax(1, keepdim=True)
        t = torch.full_like(a, 127.0)
        dead = a < 1e-30
        s = torch.where(dead, torch.zeros_like(a), a / t)
        q = torch.where(dead, torch.zeros_like(p), torch.round(p * (t / a)))
        codes.append(q)
        scales.append(s)
    return torch.cat(codes, 1), torch.cat(scales, 1)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,d", PACK)
def test_pack8_equals_its_definition(cuda, n, d, dtype):
    g = gen(n + 31 * d)
    x = torch.randn(n, d, generator=g, device=cuda) * torch.logspace(-3, 3, n, device=cuda)[:, None]
    x[0, :] = 0.0
    x = x.to(dtype)
    codes, scales = pack8(x)
    q, s = pack_plain(x)
    assert torch.equal(codes.cpu().float(), q) and torch.equal(scales.cpu(), s)
    for out in (F32, BF16, F16):
        got = unpack8(codes, scales, dtype=out)
        sc = s.repeat_interleave(128, 1)[:, :d]
        assert torch.equal(got.cpu(), (q * sc).to(out))
    # a value comes back within half a code's step
    off = (unpack8(codes, scales).double() - x.double()).abs().cpu()
    step = s.double().repeat_interleave(128, 1)[:, :d]
    assert (off <= step * (0.5 + 256 * U)).all()


@pytest.mark.parametrize("n,d,dtype", [(300_000, 19, F32), (40_000, 200, BF16), (20_000, 333, F32),
                                       (200_000, 64, F16)])
def test_pack8_of_many_rows(cuda, n, d, dtype):
    test_pack8_equals_its_definition(cuda, n, d, dtype)


def test_pack8_ties_non_finite_tiny_and_views(cuda):
    # a = 127 makes inv = 1: ties go to the even code
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -127.0, 126.5]], device=cuda)
    assert pack8(x)[0].tolist() == [[127, 0, 2, 2, 0, -2, -127, 126]]
    x = torch.ones(4, 200, device=cuda)
    x[0, 3], x[1, 130], x[2] = math.nan, -math.inf, 1e-31
    y = unpack8(*pack8(x))
    assert y[0, :128].isnan().all() and torch.equal(y[0, 128:], x[0, 128:])
    assert y[1, 128:].isnan().all() and torch.equal(y[1, :128], x[1, :128])
    assert torch.equal(y[2], torch.zeros_like(y[2])) and torch.equal(y[3], x[3])
    top = torch.finfo(F32).max
    z = unpack8(*pack8(torch.tensor([[top, -top, 0.0, top / 2]], device=cuda)))
    assert z.isfinite().all() and z[0, 2] == 0
    base = torch.randn(20, 41, generator=gen(1), device=cuda)
    v = base[1::3, 2:40:2]
    assert all(torch.equal(a, b) for a, b in zip(pack8(v), pack8(v.contiguous())))
    flat = torch.randn(161, generator=gen(2), device=cuda)
    v = flat[1:].view(5, 32)
    assert all(torch.equal(a, b) for a, b in zip(pack8(v), pack8(v.clone())))
    codes, scales = pack8(v)
    odd = torch.zeros(161, dtype=torch.int8, device=cuda)
    odd[1:] = codes.flatten()
    assert torch.equal(unpack8(odd[1:].view(5, 32), scales), unpack8(codes, scales))
    c, s = pack8(torch.zeros(0, 7, device=cuda))
    assert c.shape == (0, 7) and s.shape == (0, 1) and unpack8(c, s).shape == (0, 7)
    assert pack8(torch.ones(5, device=cuda))[1].shape == (1,)


def test_checkpoint8_is_the_segment_at_the_value_read_back(cuda):
    g = gen(6)
    x = torch.randn(70, 48, generator=g, device=cuda, requires_grad=True)
    w = torch.randn(48, generator=g, device=cuda, requires_grad=True)
    c = torch.randn(9, 48, generator=g, device=cuda, requires_grad=True)
    lab = torch.randint(0, 9, (70,), generator=g, device=cuda)

    def segment(x, w, c, k):
        return label_loss(layer_norm(x, w), c, lab, scale=k)

    loss = checkpoint8(segment, x, w, c, 0.5)
    assert torch.equal(loss, segment(x, w, c, 0.5))
    got = torch.autograd.grad(loss * 3, (x, w, c))
    xr = held8(x).requires_grad_(True)
    want = torch.autograd.grad(segment(xr, w, c, 0.5) * 3, (xr, w, c))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # only some inputs need a gradient; an unused one gets none
    (gw,) = torch.autograd.grad(checkpoint8(segment, x.detach(), w, c.detach(), 0.5) * 3, w)
    assert torch.equal(gw, want[1])
    gx, gu = torch.autograd.grad(checkpoint8(lambda t, u: t * 2, x, w).sum(), (x, w),
                                 allow_unused=True)
    assert torch.equal(gx, torch.full_like(x, 2)) and gu is None
    with torch.no_grad():
        assert torch.equal(checkpoint8(segment, x, w, c, 0.5), loss)
    with pytest.raises(TypeError, match="one tensor"):
        checkpoint8(lambda t: (t, t), x)


def test_layer_norm_int8_holds_a_quarter(cuda):
    x = torch.randn(4096, 256, device=cuda, requires_grad=True)
    w = torch.ones(256, device=cuda, requires_grad=True)

    def held(saved):
        y = layer_norm(x * 1.0, w, saved=saved)
        return sum(t.numel() * t.element_size() for t in y.grad_fn.saved_tensors if t is not None)

    full, packed = held("full"), held("int8")
    assert packed <= full / 4 + 4096 * 4 * 5


# ------------------------------------------------------------------ label loss

def label64(x, w, lab, bias, scale, ignored, reduction, grad):
    """loss, dx, dw, db in 64 bits and their bounds."""
    dtype = x.dtype
    n, d = x.shape
    v = w.shape[0]
    live = lab != ignored
    x64 = torch.where(live[:, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    w64 = w.double()
    b64 = torch.zeros(v, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    z = scale * (x64 @ w64.t()) + b64
    # fp32 products summed over d, times scale, plus bias; infinite bias is exact
    mag = abs(scale) * (x64.abs() @ w64.abs().t()) + torch.where(b64.isinf(), 0.0, b64.abs())
    tz = (d + 8) * U * mag
    lse = torch.logsumexp(z, 1)
    idx = torch.where(live, lab, 0).long()
    zl = z.gather(1, idx[:, None])[:, 0]
    loss = torch.where(live, lse - zl, torch.zeros_like(zl))
    tmax = tz.amax(1)
    # the loss is a function of differences of logits, each off by 2 tz; exp and log: few u of 1 + lse
    tl = torch.where(live, 2 * tmax + 16 * U * (1 + lse.abs()) + (v + 8) * U, torch.zeros_like(zl))
    count = live.sum().clamp_min(1).double()
    r = live.double()
    if reduction == "mean":
        r, total, ttotal = r / count, loss.sum() / count, tl.sum() / count
    elif reduction == "sum":
        total, ttotal = loss.sum(), tl.sum()
    else:
        r, total, ttotal = r * grad.double(), loss, tl
    if reduction != "none":
        r = r * float(grad)
        ttotal = ttotal + 2 * U * total.abs()
    p = torch.exp(z - lse[:, None])
    onehot = torch.zeros_like(p).scatter_(1, idx[:, None], 1.0)
    others = (p * (1 - onehot)).sum(1)
    G = torch.where(onehot > 0, -others[:, None], p) * r[:, None]
    # relative error of an entry of G: differences of logits, the log-sum's rounding, a sum of v
    rel = (4 * tmax + 16 * U * (1 + lse.abs()) + (v + 8) * U)[:, None]
    # the logits' gradient may be held in the features' type
    rel = rel + (half(dtype) if dtype != F32 else 2 * U)
    aG = torch.where(live[:, None], G.abs(), torch.zeros_like(G))
    dx = scale * (G @ w64)
    tdx = abs(scale) * ((aG * (rel + (v + 8) * U)) @ w64.abs())
    dw = scale * (G.t() @ x64)
    tdw = abs(scale) * ((aG * (rel + (n + 8) * U)).t() @ x64.abs())
    # the bias's gradient is fp32 and sums the unrounded entries
    relb = rel - (half(dtype) if dtype != F32 else 0.0)
    db = G.sum(0)
    tdb = (aG * (relb + (n + 8) * U)).sum(0)
    return (total, dx, dw, db), (ttotal, tdx, tdw, tdb)


def label_case(seed, n, d, v, dtype, ldtype=torch.int64, ignored=-100, share=0.2):
    g = gen(seed)
    w = (torch.randn(v, d, generator=g, device="cuda") * 2 / math.sqrt(d))
    lab = torch.randint(0, v, (n,), generator=g, device="cuda")
    x = torch.randn(n, d, generator=g, device="cuda") + w[lab]
    lab[torch.rand(n, generator=g, device="cuda") < share] = ignored
    bias = torch.randn(v, generator=g, device="cuda")
    return x.to(dtype), w.to(dtype), lab.to(ldtype), bias, g


def check_label(x, w, lab, bias, scale=1.0, ignored=-100, reduction="mean", grad=None):
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    bl = None if bias is None else bias.detach().requires_grad_(True)
    grad = torch.tensor(1.0, device=x.device) if grad is None else grad
    loss = label_loss(xl, wl, lab, bias=bl, scale=scale, ignore_index=ignored, reduction=reduction)
    assert loss.dtype == F32
    leaves = [xl, wl] + ([bl] if bl is not None else [])
    grads = torch.autograd.grad(loss, leaves, grad)
    want, tol = label64(x, w, lab.long(), bias, scale, ignored, reduction, grad)
    for got, ref, t, what in zip((loss.detach(), *grads), want, tol, ("loss", "dx", "dw", "db")):
        tiny = 2.0 ** -25 if got.dtype == F16 else 0.0
        within(got, ref, t + half(got.dtype) * (ref.abs() + t) + tiny, what)
    return loss.detach(), grads


LABELS = [(1, 1, 1), (1, 3, 2), (2, 16, 5), (63, 8, 64), (64, 16, 65), (65, 17, 63), (1, 64, 1000),
          (200, 13, 129), (129, 64, 257), (300, 65, 100), (128, 128, 128), (257, 77, 513),
          (90, 200, 300), (140, 512, 260), (1000, 16, 200), (33, 511, 33), (3, 20, 5000)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,d,v", LABELS)
def test_label_loss(cuda, n, d, v, dtype):
    x, w, lab, bias, _ = label_case(n + 7 * d + 31 * v, n, d, v, dtype)
    check_label(x, w, lab, bias)


@pytest.mark.parametrize("n,d,v,dtype", [
    (40_000, 16, 200, F32),      # classes that stay in shared memory, several row tiles to a block
    (40_000, 100, 129, F32),     # the same with two chunks of channels
    (20_000, 24, 4_300, BF16),   # more than one visit of the accumulator to memory
    (25_000, 140, 300, F32),     # wide features: the logits' gradient through scratch
    (5_000, 300, 16_500, BF16),  # in more than one piece
    (2_500, 200, 20_000, F16),
    (300, 300, 40_000, F32),     # few rows: the classes in shares
    (50_000, 128, 2_000, F32),   # two streamed tiles are all that fits
])
def test_label_loss_of_many(cuda, n, d, v, dtype):
    x, w, lab, bias, _ = label_case(n + d + v, n, d, v, dtype)
    check_label(x, w, lab, bias)


def test_label_loss_off_the_boundaries(cuda):
    """Contiguous tensors that start 2 or 4 bytes off a 16-byte boundary."""
    for dtype in (F32, BF16):
        x, w, lab, bias, g = label_case(22, 90, 32, 50, dtype)

        def off(t):
            flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)
            flat[1:] = t.flatten()
            return flat[1:].view(t.shape)

        a, ga = check_label(x, w, lab, bias)
        b, gb = check_label(off(x), off(w), off(lab), off(bias))
        assert torch.equal(a, b) and all(torch.equal(p, q) for p, q in zip(ga, gb))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["none", "sum"])
@pytest.mark.parametrize("n,d,v", [(130, 24, 70), (64, 100, 256)])
def test_label_loss_reductions_and_scale(cuda, n, d, v, reduction, dtype):
    x, w, lab, bias, g = label_case(n + d + v, n, d, v, dtype)
    grad = torch.randn(n, generator=g, device=cuda) if reduction == "none" else \
        torch.tensor(-0.75, device=cuda)
    check_label(x, w, lab, None, scale=2.5, reduction=reduction, grad=grad)
    check_label(x, w, lab, bias, scale=-0.5, reduction=reduction, grad=grad)


@pytest.mark.parametrize("ldtype,ignored", [(torch.uint8, 255), (torch.int32, -1),
                                            (torch.int64, 3), (torch.uint8, 3)])
def test_label_types_and_ignored_values(cuda, ldtype, ignored):
    x, w, lab, bias, _ = label_case(11, 150, 20, 40, F32, ldtype, ignored)
    check_label(x, w, lab, bias, ignored=ignored)


def test_label_loss_shapes_strides_and_bias_types(cuda):
    x, w, lab, bias, g = label_case(12, 120, 24, 40, BF16)
    base = torch.empty(120, 50, dtype=BF16, device=cuda)
    xs = base[:, 1:49:2]
    xs.copy_(x)
    ws = torch.empty(24, 40, dtype=BF16, device=cuda).t()
    ws.copy_(w)
    ls = torch.stack([lab, lab], 1)[:, 0]
    a, ga = check_label(xs, ws, ls, bias)
    b, gb = check_label(x, w, lab, bias)
    assert torch.equal(a, b) and all(torch.equal(p, q) for p, q in zip(ga, gb))
    img = label_loss(x.view(10, 12, 24), w, lab.view(10, 12), reduction="none")
    assert img.shape == (10, 12)
    assert torch.equal(img.flatten(), label_loss(x, w, lab, reduction="none"))
    one = label_loss(x[0], w, lab.clamp_min(0)[0], reduction="none")
    assert one.shape == ()
    bb = bias.to(BF16).requires_grad_(True)
    (g1,) = torch.autograd.grad(label_loss(x, w, lab, bias=bb), bb)
    assert g1.dtype == BF16
    # elements that autograd does not ask for are left out
    wl = w.clone().requires_grad_(True)
    (gw,) = torch.autograd.grad(label_loss(x, wl, lab, bias=bias), wl)
    assert torch.equal(gw, gb[1])


def test_label_loss_no_live_rows_and_no_rows(cuda):
    x, w, lab, bias, _ = label_case(13, 100, 20, 30, F32)
    x[:] = math.nan
    lab[:] = -100
    for red, want in (("mean", torch.zeros((), device=cuda)), ("sum", torch.zeros((), device=cuda)),
                      ("none", torch.zeros(100, device=cuda))):
        xl, wl, bl = (t.clone().requires_grad_(True) for t in (x, w, bias))
        loss = label_loss(xl, wl, lab, bias=bl, reduction=red)
        assert torch.equal(loss, want)
        for q in torch.autograd.grad(loss.sum(), (xl, wl, bl)):
            assert torch.equal(q, torch.zeros_like(q))
    for red in ("mean", "sum", "none"):
        xl, wl, bl = (t.clone().requires_grad_(True) for t in (x[:0], w, bias))
        loss = label_loss(xl, wl, lab[:0], bias=bl, reduction=red)
        assert loss.shape == ((0,) if red == "none" else ())
        gx, gw, gb = torch.autograd.grad(loss.sum(), (xl, wl, bl))
        assert gx.shape == (0, 20) and not gw.any() and not gb.any()


def test_label_loss_ignored_rows_hold_anything(cuda):
    """NaN, infinity and the type's lowest value in ignored rows change no bit
    of anything."""
    for dtype in (F32, BF16):
        x, w, lab, bias, _ = label_case(14, 200, 40, 50, dtype)
        a, ga = check_label(x, w, lab, bias)
        gone = (lab == -100).nonzero()[:, 0]
        assert gone.numel() > 10
        y = x.clone()
        y[gone[0::3]] = math.nan
        y[gone[1::3]] = math.inf
        y[gone[2::3]] = torch.finfo(dtype).min
        yl, wl, bl = (t.clone().requires_grad_(True) for t in (y, w, bias))
        b = label_loss(yl, wl, lab, bias=bl)
        gb = torch.autograd.grad(b, (yl, wl, bl))
        assert torch.equal(a, b) and all(torch.equal(p, q) for p, q in zip(ga, gb))
        assert not gb[0][gone].any()


def test_label_loss_classes_taken_out(cuda):
    """-infinity and the lowest float in the bias: those classes have
    probability 0 and gradient 0; a label on one has loss infinity (or the
    lowest float's size)."""
    x, w, lab, bias, _ = label_case(15, 150, 24, 140, F32, share=0.0)
    out = torch.arange(0, 140, 3, device=cuda)
    lab = torch.where(lab % 3 == 0, lab + 1, lab).clamp_max(139)
    lab = torch.where(lab % 3 == 0, lab - 1, lab)
    bias[out] = -math.inf
    _, (gx, gw, gb) = check_label(x, w, lab, bias)
    assert not gb[out].any() and not gw[out].any()
    bias[out] = torch.finfo(F32).min
    xl, wl, bl = (t.clone().requires_grad_(True) for t in (x, w, bias))
    g2 = torch.autograd.grad(label_loss(xl, wl, lab, bias=bl), (xl, wl, bl))
    assert all(torch.equal(p, q) for p, q in zip((gx, gw, gb), g2))
    bias[out] = -math.inf
    lab[7] = 3
    rows = label_loss(x, w, lab, bias=bias, reduction="none")
    assert rows[7] == math.inf and rows.isfinite().sum() == 149
    rows = label_loss(x, w, lab, bias=torch.full_like(bias, -math.inf), reduction="none")
    assert rows.isnan().all()


def test_label_loss_nan_features_spoil_their_row_alone(cuda):
    x, w, lab, bias, _ = label_case(16, 100, 24, 70, F32, share=0.0)
    clean = label_loss(x, w, lab, bias=bias, reduction="none")
    y = x.clone()
    y[9, 3] = math.nan
    yl = y.requires_grad_(True)
    rows = label_loss(yl, w, lab, bias=bias, reduction="none")
    (gx,) = torch.autograd.grad(rows, yl, torch.ones_like(rows))
    keep = torch.arange(100, device=cuda) != 9
    assert rows[9].isnan() and torch.equal(rows[keep].detach(), clean[keep])
    assert gx[9].isnan().all() and gx[keep].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_after_a_loss_of_nans(cuda, dtype):
    """What an earlier call left on the SMs (here NaN in every score) reaches
    no later one, whatever its number of classes."""
    bad = torch.full((148 * 128, 32), math.nan, dtype=dtype, device=cuda).requires_grad_(True)
    wide = torch.randn(512, 32, generator=gen(30), device=cuda).to(dtype)
    zeros = torch.zeros(148 * 128, dtype=torch.int64, device=cuda)
    for v in (1, 5, 8, 17, 33, 63, 65, 130):
        rows = label_loss(bad, wide, zeros, reduction="sum")
        assert torch.autograd.grad(rows, bad)[0].isnan().all()
        x, w, lab, bias, _ = label_case(31 + v, 300, 24, v, dtype)
        check_label(x, w, lab, bias)


def test_label_loss_confident_rows_keep_their_digits(cuda):
    """Rows whose class wins by 20 to 60: loss and gradient are e^-20 to e^-60
    and keep their relative precision (bounded by the logits' own)."""
    n, d = 40, 16
    w = torch.eye(d, device=cuda)[:8] * 4
    lab = torch.arange(n, device=cuda) % 8
    x = w[lab] * torch.linspace(1.3, 3.8, n, device=cuda)[:, None]
    xl = x.clone().requires_grad_(True)
    rows = label_loss(xl, w, lab, reduction="none")
    (gx,) = torch.autograd.grad(rows, xl, torch.ones_like(rows))
    z = (x.double() @ w.double().t())
    want = torch.log1p((z - z.gather(1, lab[:, None])).exp().scatter(1, lab[:, None], 0.0).sum(1))
    # exp of a difference of up to 61 with logits exact to 2^-23 of themselves
    rel = 4 * 61 * 2 * U + 16 * U
    within(rows.detach(), want, rel * want, "loss")
    p = torch.softmax(z, 1).scatter(1, lab[:, None], 0.0)
    G = p.scatter(1, lab[:, None], -p.sum(1, keepdim=True))
    within(gx, G @ w.double(), 2 * rel * (G.abs() @ w.double().abs()), "dx")


def test_label_outside_the_classes_is_reported(cuda):
    x, w, lab, bias, _ = label_case(17, 80, 16, 20, F32)
    assert ext.device_error() == 0
    for bad in (20, -1, 1 << 40, -(1 << 40)):
        lab2 = lab.clone()
        lab2[5] = bad
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        rows = label_loss(xl, wl, lab2, reduction="none")
        gx, gw = torch.autograd.grad(rows, (xl, wl), torch.ones_like(rows))
        assert rows[5].isnan() and rows.isnan().sum() == 1
        assert not gx[5].any() and gx.isfinite().all() and gw.isfinite().all()
        with pytest.raises(_lib.DeviceError, match="label"):
            _lib.check_device_error("test")
        assert label_loss(x, w, lab2).isnan()
        assert ext.device_error() == 3
    assert ext.device_error() == 0


def test_label_gradient_against_differences(cuda):
    g = gen(18)
    x, w, lab, bias, _ = label_case(18, 30, 12, 25, F32)
    dirs = [torch.randn(t.shape, generator=g, device=cuda) for t in (x, w, bias)]

    def f(e):
        z = (x.double() + e * dirs[0]) @ (w.double() + e * dirs[1]).t() + bias + e * dirs[2]
        return torch.nn.functional.cross_entropy(z, lab)

    e = 1e-5
    slope = float((f(e) - f(-e)) / (2 * e))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, bias)]
    grads = torch.autograd.grad(label_loss(leaves[0], leaves[1], lab, bias=leaves[2]), leaves)
    got = sum(float((q.double() * v).sum()) for q, v in zip(grads, dirs))
    size = sum(float((q.double().abs() * v.abs()).sum()) for q, v in zip(grads, dirs))
    # third derivatives of order |direction|^3 ~ 10^3 times step^2 = 10^-10; fp32 work
    assert abs(got - slope) <= 1e-6 + 200 * U * size


@pytest.mark.parametrize("d", [1030, 1032])
def test_more_than_2_to_the_32_elements(cuda, d):
    """Offsets past 32 bits: the last rows of a 8.6 GB map come out as they do
    alone."""
    n = 2 ** 32 // d + 3
    x = torch.zeros(n, d, dtype=BF16, device=cuda)
    tail = torch.randn(4, d, generator=gen(40), device=cuda).to(BF16)
    x[-4:] = tail
    codes, scales = pack8(x)
    one = pack8(tail)
    assert torch.equal(codes[-4:], one[0]) and torch.equal(scales[-4:], one[1])
    back = unpack8(codes, scales, dtype=BF16)
    assert torch.equal(back[-4:], unpack8(*one, dtype=BF16)) and not back[-8:-4].any()
    del codes, scales, back
    x.requires_grad_(True)
    w = torch.randn(d, generator=gen(41), device=cuda).to(BF16).requires_grad_(True)
    y = layer_norm(x, w, saved="int8")
    dy = torch.zeros_like(x)
    dy[-4:] = tail.flip(0)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    tl = tail.clone().requires_grad_(True)
    want = layer_norm(tl, w, saved="int8")
    wx, ww = torch.autograd.grad(want, (tl, w), tail.flip(0))
    assert torch.equal(y[-4:], want) and torch.equal(gx[-4:], wx)
    # the same four rows summed in another order
    assert float((gw - ww).abs().max()) <= 2 * half(BF16) * float(ww.abs().max())


def test_label_loss_past_2_to_the_32_elements(cuda):
    n, d = 2 ** 26 + 200, 64
    x = torch.zeros(n, d, dtype=BF16, device=cuda)
    xt, w, lab_t, _, _ = label_case(42, 150, d, 20, BF16)
    x[-150:] = xt
    lab = torch.full((n,), 255, dtype=torch.uint8, device=cuda)
    lab[-150:] = torch.where(lab_t == -100, 255, lab_t).to(torch.uint8)
    x.requires_grad_(True)
    loss = label_loss(x, w, lab, ignore_index=255, reduction="none")
    (gx,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
    tl = xt.clone().requires_grad_(True)
    want = label_loss(tl, w, lab[-150:], ignore_index=255, reduction="none")
    (wx,) = torch.autograd.grad(want, tl, torch.ones_like(want))
    assert torch.equal(loss[-150:], want) and not loss[:-150].any()
    assert torch.equal(gx[-150:], wx) and not gx[-1000:-150].any()


def test_second_derivatives_are_refused(cuda):
    """A first derivative may be part of a graph; asking for the second of
    these operators raises."""
    x, w, lab, bias, _ = label_case(21, 20, 8, 6, F32)
    for f in (lambda t: label_loss(t, w, lab), lambda t: layer_norm(t).square().sum(),
              lambda t: layer_norm(t, saved="int8").square().sum(),
              lambda t: checkpoint8(lambda u: label_loss(u, w, lab), t)):
        xl = x.clone().requires_grad_(True)
        (plain,) = torch.autograd.grad(f(xl), xl)
        (g,) = torch.autograd.grad(f(xl), xl, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), xl)


# ------------------------------------------------------------------ as a user's program runs them

def head(x, lw, lb, c, lab, cb):
    return label_loss(layer_norm(x, lw, lb, saved="int8"), c, lab, bias=cb)


def head_case(dtype=F32, n=900, d=24, v=60):
    x, w, lab, bias, g = label_case(19, n, d, v, dtype)
    lw = torch.randn(d, generator=g, device="cuda").to(dtype)
    lb = torch.randn(d, generator=g, device="cuda").to(dtype)
    return x, lw, lb, w, lab, bias


def head_grads(args):
    leaves = [t.detach().clone().requires_grad_(t.is_floating_point()) for t in args]
    loss = head(*leaves)
    return [loss.detach(), *torch.autograd.grad(loss, [t for t in leaves if t.requires_grad])]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_calls_give_equal_bits_on_any_stream(cuda, dtype):
    args = head_case(dtype)
    want = head_grads(args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = head_grads(args)
        got2 = head_grads(args)
    torch.cuda.current_stream().wait_stream(side)
    again = head_grads(args)
    for a, b, c, d in zip(want, got, got2, again):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


def test_two_calls_at_once_on_two_streams(cuda):
    cases = [head_case(F32, 5000, 24, 60), head_case(BF16, 7000, 64, 300)]
    want = [head_grads(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(head_grads(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_two_captured_graphs_replayed_with_new_inputs(cuda):
    """Forward and backward captured twice, replayed in turn with other
    inputs written into the captured ones."""
    shapes = [(F32, 900, 24, 60), (BF16, 700, 40, 300)]
    graphs = []
    for dt, n, d, v in shapes:
        args = head_case(dt, n, d, v)
        leaves = [t.detach().clone().requires_grad_(t.is_floating_point()) for t in args]
        need = [t for t in leaves if t.requires_grad]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(head(*leaves), need)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = head(*leaves)
            outs = [loss.detach(), *torch.autograd.grad(loss, need)]
        graphs.append((graph, leaves, outs, args))
    for rep in range(3):
        for graph, leaves, outs, args in graphs:
            new = [t * (1 + 0.1 * rep) if t.is_floating_point() else t for t in args]
            with torch.no_grad():
                for a, b in zip(leaves, new):
                    a.copy_(b)
            graph.replay()
        for graph, leaves, outs, args in graphs:
            want = head_grads([t.detach() for t in leaves])
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_rendered_features_through_the_head(cuda):
    """Six feature channels rendered as two explicit-colour passes, held in 8
    bits, normalised, compared with embeddings; the gradient reaches the
    Gaussians' features and equals the one of the same head in plain torch."""
    g = gen(20)
    n, W, H, v = 3000, 96, 64, 12
    means = torch.randn(n, 3, generator=g, device=cuda) * 0.6
    means[:, 2] += 4.0
    quats = torch.randn(n, 4, generator=g, device=cuda)
    scales = torch.rand(n, 3, generator=g, device=cuda) * 0.08 + 0.02
    opac = torch.rand(n, generator=g, device=cuda) * 0.7 + 0.15
    feats = torch.randn(n, 6, generator=g, device=cuda, requires_grad=True)
    K = torch.tensor([[77.0, 0, W / 2], [0, 77.0, H / 2], [0, 0, 1]])
    w = torch.randn(6, generator=g, device=cuda, requires_grad=True)
    c = torch.randn(v, 6, generator=g, device=cuda, requires_grad=True)
    lab = torch.randint(0, v, (H, W), generator=g, device=cuda, dtype=torch.int32).to(torch.uint8)
    lab[:10] = 255

    def feature_map():
        maps = [render(means, quats, scales, opac, None, K, torch.eye(4), W, H,
                       colors=feats[:, i:i + 3].contiguous())[0] for i in (0, 3)]
        return torch.cat(maps, 2)

    def segment(m, w, c):
        return label_loss(layer_norm(m, w, eps=1e-2), c, lab, ignore_index=255)

    fmap = feature_map()
    loss = checkpoint8(segment, fmap, w, c)
    df, dw, dc = torch.autograd.grad(loss, (feats, w, c))
    fmap = feature_map()
    held = fmap + (held8(fmap) - fmap).detach()
    y = torch.nn.functional.layer_norm(held.double(), (6,), w.double(), None, 1e-2)
    ref = torch.nn.functional.cross_entropy((y @ c.double().t()).view(-1, v), lab.view(-1).long(),
                                            ignore_index=255)
    rf, rw, rc = torch.autograd.grad(ref, (feats, w, c))
    for got, want in ((df, rf), (dw, rw), (dc, rc)):
        # the rasteriser's fp32 adjoint with float atomics: 1e-5 of the norm
        assert float((got.double() - want).norm()) <= 1e-5 * float(want.norm())
    assert ext.device_error() == 0

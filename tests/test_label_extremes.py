"""label_loss at the ends of the floating range."""

import math

import pytest
import torch

from metal_gauss_b200.labels import label_loss
from test_features import BF16, F16, F32, check_label, label_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v", [1, 40, 300])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_infinite_logit_gives_nan(cuda, dtype, v):
    """log sum exp(z) - z[label] is infinity - infinity where the label's logit
    is infinite: a NaN loss and gradient, as for another class's."""
    x, w, lab, bias, _ = label_case(50 + v, 60, 24, v, dtype, share=0.0)
    bias[0] = math.inf
    xl = x.clone().requires_grad_(True)
    rows = label_loss(xl, w, lab, bias=bias, reduction="none")
    (gx,) = torch.autograd.grad(rows, xl, torch.ones_like(rows))
    assert rows.isnan().all() and gx.isnan().all()
    # by a product that overflows, in its own row alone
    x, w, lab, bias, _ = label_case(51 + v, 60, 24, v, BF16, share=0.0)
    clean = label_loss(x, w, lab, bias=bias, reduction="none")
    w[:, 0] = 0.0
    w[lab[7], 0] = 3e38
    x[:, 0], x[7, 0] = 0.0, 3e38
    rows = label_loss(x, w, lab, bias=bias, reduction="none")
    keep = torch.arange(60, device=cuda) != 7
    assert rows[7].isnan() and rows[keep].isfinite().all() and clean.isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,d,v", [(70, 24, 50), (60, 150, 70), (40, 300, 50)])
def test_the_types_ends_where_the_other_side_is_zero(cuda, n, d, v, dtype):
    """The largest and the lowest finite value in an embedding or a feature
    whose partner is 0: products of 0, and gradients that large."""
    ends = torch.finfo(dtype)
    x, w, lab, bias, _ = label_case(n + d + v, n, d, v, dtype)
    x[:, 0] = 0.0
    w[3, 0], w[5, 0] = ends.min, ends.max
    w[:, d - 1] = 0.0
    live = (lab != -100).nonzero()[:, 0]
    x[live[2], d - 1], x[live[4], d - 1] = ends.max, ends.min
    check_label(x, w, lab, bias)

"""Gradients of the loss without scores where its own gradient is not a number: nothing of it may vanish, and rows that
it does not reach keep their gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def setup(rows, dtype, classes=1000):
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randn(rows, 64, generator=g, device="cuda").to(dtype)
    w = (torch.randn(64, classes, generator=g, device="cuda") / 8).to(dtype)
    b = torch.randn(classes, generator=g, device="cuda")
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return x, w, b, t


def finite(x):
    return bool(torch.isfinite(x).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("rows,others", [(1, 0.0), (40, 0.0), (40, 1.0), (1500, 0.5)])
def test_row_without_reduction(dtype, value, rows, others):
    """One row's gradient is not finite; the others' are zeros or not."""
    from flashlight_b200 import _lib as L
    from flashlight_b200 import functions as F
    x, w, b, t = setup(rows, dtype)
    loss, state, lse = F.linear_cross_entropy(x, w, b, t, L.REDUCE_NONE)
    go = torch.full((rows,), others, device="cuda")
    clean = F.linear_cross_entropy_backward(x, w, b, lse, go, state)
    at = rows // 2
    go[at] = value
    gx, gw, gb = F.linear_cross_entropy_backward(x, w, b, lse, go, state)
    assert not bool(torch.isfinite(gx[at]).any())
    assert not bool(torch.isfinite(gw).any()) and not bool(torch.isfinite(gb).any())
    rest = [r for r in range(rows) if r != at]
    assert finite(gx[rest]) and torch.equal(gx[rest], clean[0][rest])
    t[at] = -1  # a row that does not count: no trace of its gradient
    loss, state, lse = F.linear_cross_entropy(x, w, b, t, L.REDUCE_NONE)
    assert all(finite(got) for got in F.linear_cross_entropy_backward(x, w, b, lse, go, state))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("reduction", ["REDUCE_MEAN", "REDUCE_SUM"])
def test_reduced(value, reduction):
    from flashlight_b200 import _lib as L
    from flashlight_b200 import functions as F
    x, w, b, t = setup(40, torch.bfloat16)
    t[7] = -1
    loss, state, lse = F.linear_cross_entropy(x, w, b, t, getattr(L, reduction))
    gx, gw, gb = F.linear_cross_entropy_backward(x, w, b, lse, torch.full((1,), value, device="cuda"), state)
    rest = [r for r in range(40) if r != 7]
    for got in (gx[rest], gw, gb):
        assert not bool(torch.isfinite(got).any())
    assert bool((gx[7] == 0).all())  # it does not count


@pytest.mark.parametrize("reduction", ["REDUCE_MEAN", "REDUCE_SUM", "REDUCE_NONE"])
def test_rows_that_do_not_count(reduction):
    """The gradients against 64 bits where ignored rows' x is NaN (grad_x and grad_bias) and where it is large (all).
    Tolerances: G and each gradient are rounded to bf16 once, 2^-9 each of the terms: 2^-8 of the norm holds both;
    grad_bias is a sum of fp32 numbers that are right to 2e-5."""
    from flashlight_b200 import _lib as L
    from flashlight_b200 import functions as F
    x, w, b, t = setup(70, torch.bfloat16)
    t[3], t[44], t[60] = -1, 1000, -7
    out = torch.tensor([3, 44, 60], device="cuda")
    kept = torch.ones(70, dtype=torch.bool, device="cuda")
    kept[out] = False
    go = torch.randn(70 if reduction == "REDUCE_NONE" else 1, generator=torch.Generator("cuda").manual_seed(1),
                     device="cuda")
    for value in (float("nan"), 1e4):
        x[out] = value
        loss, state, lse = F.linear_cross_entropy(x, w, b, t, getattr(L, reduction))
        gx, gw, gb = F.linear_cross_entropy_backward(x, w, b, lse, go, state)
        xd, wd = x[kept].double(), w.double()
        G = torch.softmax(xd @ wd + b.double(), 1)
        G[torch.arange(67, device="cuda"), t[kept].long()] -= 1
        G *= go[kept, None].double() if len(go) > 1 else go.double() / (67 if reduction == "REDUCE_MEAN" else 1)
        near = lambda got, want, rel: float((got.double() - want).norm()) <= rel * float(want.norm())  # noqa: E731
        assert bool((gx[out] == 0).all()) and near(gx[kept], G @ wd.t(), 2.0 ** -8)
        assert near(gb, G.sum(0), 2e-5)
        if value == 1e4:
            assert near(gw, xd.t() @ G, 2.0 ** -8)

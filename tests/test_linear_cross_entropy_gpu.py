"""The loss without scores against its definition in 64 bits from the same 16-bit tensors.

Tolerances.  Scores are fp32 sums of exact products, off by at most 2^-22 of the sum of the products'
magnitudes (K up to 1000: tensor memory truncates what it carries); with |z| up to about 10 that is 2e-5 of
a row's loss at most.  G is rounded once to its type (2^-9 or 2^-12 of each entry), and each gradient once
more to its own: relative to the gradient's norm 2^-8 and 2^-11 hold both with room."""
import pytest
import torch

pytestmark = pytest.mark.gpu
REL = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def definition(x, w, b, t, gl, reduction, ignore):
    x, w = x.double().requires_grad_(), w.double().requires_grad_()
    b = b.double().requires_grad_() if b is not None else None
    z = x @ w + (b if b is not None else 0)
    kept = (t != ignore) & (t >= 0) & (t < z.shape[1])
    at = torch.where(kept, t, torch.zeros_like(t)).long()
    loss = (torch.logsumexp(z, 1) - z.gather(1, at[:, None])[:, 0])
    loss = torch.where(kept, loss, torch.zeros_like(loss))
    if reduction == "mean":
        loss = loss.sum().reshape(1) / kept.sum()
    elif reduction == "sum":
        loss = loss.sum().reshape(1)
    (loss * gl.double()).sum().backward()
    return loss.detach(), x.grad, w.grad, b.grad if b is not None else None


def near(got, want, rel):
    want = want.double()
    off = float((got.double() - want).norm())
    assert bool(torch.isfinite(got).all()) and off <= rel * float(want.norm()) + 1e-30, (off, float(want.norm()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,dim,classes,reduction,bias", [
    (1, 64, 500, "mean", True), (3, 8, 40, "none", True), (61, 512, 8000, "mean", True), (128, 72, 256, "sum", False),
    (129, 1000, 2049, "mean", True), (257, 67, 1031, "none", False), (300, 256, 33, "sum", True),
    (1000, 136, 5003, "mean", False), (37, 64, 1, "sum", True), (1500, 320, 12800, "none", True)])
def test_loss_and_gradients(dtype, rows, dim, classes, reduction, bias):
    from flashlight_b200 import _lib as L
    from flashlight_b200 import autograd as A
    g = torch.Generator("cuda").manual_seed(rows + classes)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    w = (torch.randn(dim, classes, generator=g, device="cuda") * 2 / dim ** 0.5).to(dtype)
    b = torch.randn(classes, generator=g, device="cuda") if bias else None
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    t[0] = classes - 1
    if rows > 3:
        t[1], t[3] = -1, 0  # one row is ignored
    red = {"mean": L.REDUCE_MEAN, "sum": L.REDUCE_SUM, "none": L.REDUCE_NONE}[reduction]
    gl = torch.randn(rows if reduction == "none" else 1, generator=g, device="cuda")
    want = definition(x, w, b, t, gl, reduction, -1)
    xv, wv = A.Variable(x, True), A.Variable(w, True)
    bv = A.Variable(b, True) if bias else None
    before = L.lib.flb200_tc_kernel_launches()
    loss = A.linear_cross_entropy(xv, wv, bv, t, red, -1)
    assert L.lib.flb200_tc_kernel_launches() > before
    loss.backward(gl)
    assert loss.tensor.shape == want[0].shape
    near(loss.tensor, want[0], 2e-5)
    if classes > 1:  # (of one class every probability is one)
        near(xv.grad, want[1], REL[dtype])
        near(wv.grad, want[2], REL[dtype])
        if bias:
            near(bv.grad, want[3], 2e-5)
    else:
        assert float(xv.grad.abs().max()) <= 1e-5 and float(wv.grad.abs().max()) <= 1e-4


def test_views_off_alignment_and_wide_weights():
    """Tensors whose rows TMA cannot address, and the fp32 gradient of master weights."""
    from flashlight_b200 import autograd as A
    from flashlight_b200.autograd import Variable
    g = torch.Generator("cuda").manual_seed(9)
    flat = torch.randn(40 * 64 + 1, generator=g, device="cuda").bfloat16()
    master = torch.randn(64, 700, generator=g, device="cuda") / 8
    x, t = flat[1:].view(40, 64), torch.arange(40, device="cuda", dtype=torch.int32)
    xv, mv = Variable(x, True), Variable(master, True)
    wv = A.cast(mv, torch.bfloat16)
    w = wv.tensor
    loss = A.linear_cross_entropy(xv, wv, None, t)
    loss.backward()
    want = definition(x, w, None, t, torch.ones(1, device="cuda"), "mean", -1)
    near(loss.tensor, want[0], 2e-5)
    near(xv.grad, want[1], 2.0 ** -8)
    assert mv.grad.dtype == torch.float32
    near(mv.grad, want[2], 2.0 ** -8)


def test_pieces_of_the_vocabulary(monkeypatch):
    """Enough rows for several pieces and for a last one that is short: 40000 rows take pieces of 2048 columns (128 MB
    of scores' gradient hold 1600).  Compared with the operators one by one on samples in 64 bits."""
    from flashlight_b200 import autograd as A
    from flashlight_b200.autograd import Variable
    g = torch.Generator("cuda").manual_seed(11)
    rows, dim, classes = 40000, 64, 4500
    x = torch.randn(rows, dim, generator=g, device="cuda").bfloat16()
    w = (torch.randn(dim, classes, generator=g, device="cuda") / 4).bfloat16()
    b = torch.randn(classes, generator=g, device="cuda")
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    want = definition(x, w, b, t, torch.ones(1, device="cuda"), "mean", -1)
    xv, wv, bv = Variable(x, True), Variable(w, True), Variable(b, True)
    loss = A.linear_cross_entropy(xv, wv, bv, t)
    loss.backward()
    near(loss.tensor, want[0], 2e-5)
    near(xv.grad, want[1], 2.0 ** -8)
    near(wv.grad, want[2], 2.0 ** -8)
    near(bv.grad, want[3], 2e-5)


def test_special_rows():
    """Classes of -inf, targets out of range and ignored, rows of NaN or infinity that are ignored or not."""
    from flashlight_b200 import _lib as L
    from flashlight_b200 import functions as F
    g = torch.Generator("cuda").manual_seed(13)
    rows, dim, classes = 70, 64, 300
    x = torch.randn(rows, dim, generator=g, device="cuda").bfloat16()
    w = torch.randn(dim, classes, generator=g, device="cuda").bfloat16()
    b = torch.zeros(classes, device="cuda")
    b[:256] = float("-inf")  # whole tiles of classes that nobody can have
    t = torch.full((rows,), 270, dtype=torch.int32, device="cuda")
    x[3], t[3] = float("nan"), -1       # ignored: no trace of it
    x[4, 0] = float("inf")              # counts: its loss is not a number
    t[5], t[6] = classes, -7            # out of range
    t[7] = 10                           # a class of -inf: an infinite loss
    loss, state, lse = F.linear_cross_entropy(x, w, b, t, L.REDUCE_NONE)
    assert int(state.count[1]) == 1 and bool((loss[[3, 5, 6]] == 0).all())
    assert not bool(torch.isfinite(loss[4])) and float(loss[7]) == float("inf")
    with pytest.raises(ValueError):
        F.check_targets(state)
    rest = [r for r in range(rows) if r not in (3, 4, 5, 6, 7)]
    z = x[rest].double() @ w.double() + b.double()
    near(loss[rest], torch.logsumexp(z, 1) - z[:, 270], 2e-5)
    t[4] = t[7] = -1
    loss, state, lse = F.linear_cross_entropy(x, w, b, t, L.REDUCE_SUM)
    gx, gw, gb = F.linear_cross_entropy_backward(x, w, b, lse, torch.ones(1, device="cuda"), state)
    for gr in (gx[rest], gb):
        assert bool(torch.isfinite(gr).all())
    assert bool((gb[:256] == 0).all())


def test_all_rows_ignored():
    from flashlight_b200 import _lib as L
    from flashlight_b200 import functions as F
    x, w = torch.ones(5, 64, device="cuda").bfloat16(), torch.ones(64, 100, device="cuda").bfloat16()
    t = torch.full((5,), 3, dtype=torch.int32, device="cuda")
    for red in (L.REDUCE_MEAN, L.REDUCE_SUM):
        loss, state, lse = F.linear_cross_entropy(x, w, None, t, red, ignore_index=3)
        assert int(state.count[0]) == 0
        gx, gw, gb = F.linear_cross_entropy_backward(x, w, None, lse, torch.ones(1, device="cuda"), state)
        assert gb is None and bool((gx == 0).all()) and bool((gw == 0).all())


def test_gradient_is_the_differences():
    """(loss(x + e d) - loss(x - e d)) / 2e along d in the weights, which 64 bits of the operator's own loss allow
    to about 1 %: e moves every weight by two steps of its type."""
    from flashlight_b200 import autograd as A
    from flashlight_b200.autograd import Variable
    g = torch.Generator("cuda").manual_seed(17)
    x = torch.randn(200, 128, generator=g, device="cuda").half()
    w = (torch.randn(128, 1000, generator=g, device="cuda") / 8).half()
    t = torch.randint(0, 1000, (200,), generator=g, device="cuda", dtype=torch.int32)
    wv = Variable(w, True)
    A.linear_cross_entropy(Variable(x, False), wv, None, t).backward()
    e = torch.sign(wv.grad.float()) * 2.0 ** -6
    up, down = (w.float() + e).half(), (w.float() - e).half()
    f = lambda p: float(A.linear_cross_entropy(Variable(x, False), Variable(p, False), None, t).tensor)  # noqa: E731
    along = float((wv.grad.double() * (up.double() - down.double())).sum())
    assert abs(f(up) - f(down) - along) <= 0.02 * abs(along)


def test_refusals_and_the_chain():
    from flashlight_b200 import autograd as A
    from flashlight_b200 import functions as F
    from flashlight_b200.autograd import Variable
    x, w = torch.ones(4, 64, device="cuda").bfloat16(), torch.ones(64, 2048, device="cuda").bfloat16()
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (lambda: F.linear_cross_entropy(x, w, None, t[:3]),
                lambda: F.linear_cross_entropy(x, w[:32], None, t),
                lambda: F.linear_cross_entropy(x, w.half(), None, t),
                lambda: F.linear_cross_entropy(x, w, torch.ones(7, device="cuda"), t),
                lambda: F.linear_cross_entropy(x, w, torch.ones(2048, device="cuda").half(), t),
                lambda: F.linear_cross_entropy(x[:0], w, None, t[:0]),
                lambda: F.linear_cross_entropy(x, w, None, t, 7)):
        with pytest.raises(ValueError):
            bad()
    loss, state, lse = F.linear_cross_entropy(x, w, None, t)
    with pytest.raises(ValueError):
        F.linear_cross_entropy_backward(x, w, None, lse, torch.ones(4, device="cuda"), state)
    # fp32 tensors: the operators one by one
    assert F.linear_cross_entropy(x.float(), w.float(), None, t) is None
    xv = Variable(x.float(), True)
    loss = A.linear_cross_entropy(xv, Variable(w.float(), True), None, t)
    loss.backward()
    assert abs(float(loss.tensor) - 7.6246) < 1e-3 and xv.grad is not None

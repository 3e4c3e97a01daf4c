"""AdamW over many tensors against its definition in 64 bits.

Tolerances.  fp32 arithmetic with an approximate square root and quotient (2^-22 each) on a step of a few
roundings: the step is right to 2^-19 of its length, a moment to 2^-22, and the parameter to a rounding of its
own type.  An 8-bit state is right to half a step of e4m3: 2^-4 of the value, or 2^-10 of the scale below
2^-6 of it (2^-9 where a root is lifted to the least code)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.1)
EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}


def definition(p, g, m, v, step, grad_scale=1.0, lr=0., beta1=0., beta2=0., eps=0., weight_decay=0.):
    g = g * grad_scale
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    length = m / (1 - beta1 ** step) / ((v / (1 - beta2 ** step)).sqrt() + eps)
    return p - lr * (length + weight_decay * p), m, v, lr * length.abs()


def blocks_of(x):
    return torch.nn.functional.pad(x, (0, -len(x) % 256)).view(-1, 256)


def check_code(codes, scales, value, least):
    """codes * scales against the value in 64 bits."""
    got, want = blocks_of(codes.float().double()) * scales.double()[:, None], blocks_of(value)
    scale = want.abs().amax(1, keepdim=True) / 448
    assert torch.allclose(scales.double()[:, None], scale.clamp(min=1e-30 / 448), rtol=1e-5, atol=0)
    off = (got - want).abs()
    assert bool((off <= 1.001 * torch.maximum(want.abs() * 2.0 ** -4, scale * least)).all())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad", [("float32", "float32"), ("float32", "bfloat16"), ("float32", "float16"),
                                        ("bfloat16", "bfloat16"), ("float16", "float16")])
def test_one_step(param, grad, bits):
    from flashlight_b200 import functions as F
    pt, gt = getattr(torch, param), getattr(torch, grad)
    g = torch.Generator("cuda").manual_seed(3)
    randn = lambda n, dt=torch.float32: torch.randn(n, generator=g, device="cuda").to(dt)  # noqa: E731
    # lengths around a lane's, a block's and a chunk's, an empty tensor, and views off every alignment
    sizes = [1, 7, 8, 9, 255, 256, 257, 0, 2047, 2048, 2049, 70001]
    ps, gs = [randn(n, pt) for n in sizes], [randn(n, gt) for n in sizes]
    ps.append(randn(5003, pt)[3:])
    gs.append(randn(5001, gt)[1:])
    ms, vs, s1, s2 = [], [], None, None
    if bits == 8:
        s1, s2 = [], []
    for p in ps:
        m, r = randn(len(p)) * 0.1, randn(len(p)).abs() * 0.5
        if len(m) > 1:
            m[::5], r[::3] = 0, 0
        if bits == 8:
            m, r = m.to(torch.float8_e4m3fn), r.to(torch.float8_e4m3fn)
            n = (len(p) + 255) // 256
            s1.append(torch.rand(n, generator=g, device="cuda") + 0.5)
            s2.append(torch.rand(n, generator=g, device="cuda") + 0.5)
            ms.append(m)
            vs.append(r)
        else:
            ms.append(m)
            vs.append(r * r)
    want = []
    for i, (p, gr) in enumerate(zip(ps, gs)):
        m, v = ms[i].double(), vs[i].double()
        if bits == 8:
            m = (blocks_of(m) * s1[i].double()[:, None]).view(-1)[:len(p)]
            v = (blocks_of(v) * s2[i].double()[:, None]).view(-1)[:len(p)] ** 2
        want.append(definition(p.double(), gr.double(), m, v, 7, 0.5, **HYPER))
    F.adamw_step(ps, gs, ms, vs, step=7, grad_scale=0.5, first_scales=s1, second_scales=s2, **HYPER)
    for i, (p, m, v, length) in enumerate(want):
        if not len(p):
            continue
        off = (ps[i].double() - p).abs()
        assert bool((off <= p.abs() * EPS[pt] + 2.0 ** -19 * length + 1e-7).all())
        if bits == 32:
            assert torch.allclose(ms[i].double(), m, rtol=2.0 ** -21, atol=2.0 ** -24)
            assert torch.allclose(vs[i].double(), v, rtol=2.0 ** -21, atol=2.0 ** -40)
        else:
            check_code(ms[i], s1[i], m, 2.0 ** -10)
            check_code(vs[i], s2[i], v.sqrt(), 2.0 ** -9)
            assert bool((vs[i].float()[v > 0] > 0).all())


def test_hundreds_of_tensors_and_missing_gradients():
    """More tensors than a launch takes, some without a gradient, and what lies between them untouched."""
    from flashlight_b200 import _lib as L
    from flashlight_b200 import functions as F
    n, count = 300, 1100
    arena = torch.ones(count * (n + 20), device="cuda")
    ps = [arena[i * (n + 20):i * (n + 20) + n] for i in range(count)]
    gs = [None if i % 7 == 3 else torch.full((n,), float(i + 1), device="cuda") for i in range(count)]
    ms, vs = ([torch.zeros(n, device="cuda") for _ in range(count)] for _ in range(2))
    before = L.kernel_launches()
    F.adamw_step(ps, gs, ms, vs, step=1, lr=0.5, eps=0.0)
    assert L.kernel_launches() - before == math.ceil(sum(g is not None for g in gs) / 480)
    for i in range(count):  # the first step's length is lr wherever the gradient is not zero
        want = 1.0 if gs[i] is None else 0.5
        assert bool((ps[i] - want).abs().max() < 1e-5)
        assert bool((arena[i * (n + 20) + n:(i + 1) * (n + 20)] == 1).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_optimiser_over_steps(bits):
    """AdamWOptimizer on the tape's Variables; a 2-d parameter, and a gradient in another memory order."""
    from flashlight_b200.autograd import Variable
    from flashlight_b200.optim import AdamWOptimizer
    g = torch.Generator("cuda").manual_seed(5)
    variables = [Variable(torch.randn(s, generator=g, device="cuda"), True) for s in ((33, 17), (1000,), (3,))]
    opt = AdamWOptimizer(variables, 1e-2, 0.8, 0.9, 1e-8, 0.01, state_bits=bits)
    exact = [(v.tensor.double(), torch.zeros_like(v.tensor).double(), torch.zeros_like(v.tensor).double())
             for v in variables]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for step in range(1, 5):
            opt.zeroGrad()
            for i, v in enumerate(variables[:2]):
                grad = torch.randn(v.tensor.shape[::-1], generator=g, device="cuda").mT if i == 0 else torch.randn(
                    v.tensor.shape, generator=g, device="cuda")
                v.addGrad(grad)
                p, m, s, _ = definition(exact[i][0], grad.double(), exact[i][1], exact[i][2], step, lr=1e-2,
                                        beta1=0.8, beta2=0.9, eps=1e-8, weight_decay=0.01)
                exact[i] = (p, m, s)
            opt.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(variables[2].tensor.double(), exact[2][0])  # it had no gradient
    for v, (p, _, _) in zip(variables, exact):
        # in 8 bits each of the three steps behind the first has moments off by up to 2^-4, so up to an
        # eighth of a step of 0.01 * 2 (m / sqrt(v) is at most 2 here)
        tol = 1e-6 if bits == 32 else 3 * 0.02 / 8
        assert float((v.tensor.double() - p).abs().max()) <= tol


def test_not_finite_gradients():
    """NaN stays where it is, an infinity takes its block of 8-bit states with it, others are untouched."""
    from flashlight_b200 import functions as F
    n = 600
    for bits in (32, 8):
        p, grad = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
        grad[5], grad[300] = math.nan, math.inf
        if bits == 32:
            m, v, s1, s2 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), None, None
        else:
            m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
            s1, s2 = [torch.zeros(3, device="cuda")], [torch.zeros(3, device="cuda")]
        F.adamw_step([p], [grad], [m], [v], step=1, lr=0.1, first_scales=s1, second_scales=s2)
        bad = torch.isnan(p)
        assert bool(bad[5]) and bool(bad[300]) and int(bad.sum()) == 2
        state = m.float() if bits == 32 else blocks_of(m.float()).mul(s1[0][:, None]).view(-1)[:n]
        finite = torch.isfinite(state)
        assert not bool(finite[5]) and not bool(finite[300])
        assert bool(finite[512:].all()) and bool(finite[:256].sum() == 255)
        assert int(finite[256:512].sum()) == (255 if bits == 32 else 0)


def test_refusals():
    from flashlight_b200 import functions as F
    from flashlight_b200.autograd import Variable
    from flashlight_b200.optim import AdamWOptimizer
    x = lambda n=8, dt=torch.float32: torch.zeros(n, device="cuda", dtype=dt)  # noqa: E731
    f8 = x(8, torch.uint8).view(torch.float8_e4m3fn)
    bad = [
        (([x()], [x(7)], [x()], [x()]), dict(step=1)),                            # another shape
        (([x()], [x()], [x(7)], [x()]), dict(step=1)),                            # a short moment
        (([x()], [x()], [x(8, torch.bfloat16)], [x()]), dict(step=1)),            # a moment in 16 bits
        (([x()], [x()], [f8], [f8]), dict(step=1)),                               # codes without scales
        (([x()], [x()], [f8], [f8]), dict(step=1, first_scales=[x(1)])),          # one of two
        (([x()], [x()], [f8], [f8]), dict(step=1, first_scales=[x(2)], second_scales=[x(1)])),
        (([x()], [], [x()], [x()]), dict(step=1)),                                # lists of two lengths
        (([x()], [x()], [x()], [x()]), dict(step=0)),
        (([x()], [x()], [x()], [x()]), dict(step=1, beta1=1.0)),
        (([x()], [x()], [x()], [x()]), dict(step=1, eps=-1.0)),
        (([x(16)[::2]], [x()], [x()], [x()]), dict(step=1)),                      # a strided parameter
        (([x().cpu()], [x().cpu()], [x().cpu()], [x().cpu()]), dict(step=1)),
        (([x(8, torch.float64)], [x(8, torch.float64)], [x()], [x()]), dict(step=1)),
    ]
    for lists, more in bad:
        with pytest.raises(ValueError):
            F.adamw_step(*lists, lr=0.1, **more)
    with pytest.raises(RuntimeError):  # 16-bit parameters with gradients of another type
        F.adamw_step([x(8, torch.float16)], [x()], [x()], [x()], step=1, lr=0.1)
    with pytest.raises(ValueError):
        AdamWOptimizer([Variable(x(), True)], 0.1, state_bits=4)
    with pytest.raises(ValueError):
        AdamWOptimizer([Variable(x(16)[::2], True)], 0.1)
    F.adamw_step([], [], [], [], step=1, lr=0.1)

"""A step that AdamW refuses has changed nothing, whichever of its tensors was the reason."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("wrong", ["type", "shape", "step"])
def test_nothing_changes(wrong, bits):
    from flashlight_b200 import functions as F
    rand = lambda n, dt=torch.float32: torch.rand(n, device="cuda").to(dt)  # noqa: E731
    params = [rand(300), rand(300, torch.bfloat16), rand(300, torch.float16)]
    grads = [rand(300), rand(300, torch.bfloat16), rand(300, torch.float16)]
    state = torch.float32 if bits == 32 else torch.float8_e4m3fn
    first, second = [rand(300, state) for _ in params], [rand(300, state) for _ in params]
    scales = [[rand(2) for _ in params] if bits == 8 else None for _ in range(2)]
    if wrong == "type":
        grads[2] = rand(300)  # a 16-bit parameter with a gradient of another type
    elif wrong == "shape":
        grads[2] = rand(299, torch.float16)
    everything = params + grads + first + second + (scales[0] + scales[1] if bits == 8 else [])
    before = [t.clone().view(torch.uint8) for t in everything]
    with pytest.raises(RuntimeError if wrong == "type" else ValueError):
        F.adamw_step(params, grads, first, second, step=0 if wrong == "step" else 1, lr=0.1, first_scales=scales[0],
                     second_scales=scales[1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(before, everything))


def test_refused_steps_do_not_count():
    from flashlight_b200.autograd import Variable
    from flashlight_b200.optim import AdamWOptimizer
    a, b = Variable(torch.ones(40, device="cuda"), True), Variable(torch.ones(40, device="cuda").half(), True)
    a.addGrad(torch.ones(40, device="cuda"))
    b.addGrad(torch.ones(40, device="cuda").half())
    b._grad = torch.ones(40, device="cuda")
    optimiser = AdamWOptimizer([a, b], 0.1)
    with pytest.raises(RuntimeError):
        optimiser.step()
    assert optimiser.steps == 0 and bool((a.tensor == 1).all()) and bool((optimiser.first == 0).all())
    b._grad = torch.ones(40, device="cuda").half()
    optimiser.step()
    assert optimiser.steps == 1
    assert bool(((a.tensor - 0.9).abs() < 1e-6).all()) and bool(((b.tensor.float() - 0.9).abs() < 1e-3).all())

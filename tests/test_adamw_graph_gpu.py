"""A step of AdamW captured in a CUDA graph: the step's number, the rate and the tensors' addresses are of the capture, so
a replay is that step again, on what the parameters and states have become and the gradients now are."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_replay_is_the_captured_step(bits):
    from flashlight_b200 import functions as F
    from flashlight_b200.autograd import Variable
    from flashlight_b200.optim import AdamWOptimizer
    g = torch.Generator("cuda").manual_seed(bits)
    randn = lambda n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    params = [Variable(randn(n), True) for n in (5, 300, 4099)]
    optimiser = AdamWOptimizer(params, 1e-2, 0.9, 0.99, 1e-6, 0.1, state_bits=bits)
    for p in params:
        p.addGrad(randn(p.tensor.numel()))
    optimiser.step()
    optimiser.step()
    same = lambda ts: None if ts is None else [t.clone() for t in ts]  # noqa: E731
    mine = [same(x) for x in ([p.tensor for p in params], optimiser.firsts, optimiser.seconds, optimiser.first_scales,
                              optimiser.second_scales)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optimiser.step()
    assert optimiser.steps == 3
    for _ in range(3):  # new gradients in the captured buffers
        for p in params:
            p.grad.copy_(randn(p.tensor.numel()))
        graph.replay()
        F.adamw_step(mine[0], [p.grad for p in params], mine[1], mine[2], step=3, lr=1e-2, beta1=0.9, beta2=0.99,
                     eps=1e-6, weight_decay=0.1, first_scales=mine[3], second_scales=mine[4])
        torch.cuda.synchronize()
        for a, b in zip(mine, ([p.tensor for p in params], optimiser.firsts, optimiser.seconds, optimiser.first_scales,
                               optimiser.second_scales)):
            assert a is None or all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
    assert optimiser.steps == 3

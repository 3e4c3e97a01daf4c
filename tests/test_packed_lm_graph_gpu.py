"""A training step on packed rows, forward and gradient, captured as one CUDA graph on a stream of its own, and the same
step on two streams at once: the same bits as the step by itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def model_and_batch(seed):
    from flashlight_b200.packed_lm import packed_batch
    from flashlight_b200.workloads import TransformerLM
    m = TransformerLM(1000, 128, 2, 256, 2, seed=seed, compute_dtype=torch.bfloat16, packed=True, kv_heads=1, softcap=30.0,
                      distance_bias=True)
    return m, [t.cuda() for t in packed_batch(2, 300, 1000, 70, torch.Generator().manual_seed(seed))]


def step(model, batch):
    model.zeroGrad()
    loss = model.loss(*batch)
    value = loss.tensor
    loss.backward()
    return value


def test_replays_bit_for_bit():
    model, batch = model_and_batch(3)
    other = model_and_batch(4)[1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step(model, batch).clone()
    torch.cuda.current_stream().wait_stream(side)
    grads = [p.grad.clone() for p in model.parameters()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(model, batch)
    captured = [p.grad for p in model.parameters()]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert all(torch.equal(a, b) for a, b in zip(captured, grads))
    for into, new in zip(batch, other):  # new inputs in the captured buffers
        into.copy_(new)
    graph.replay()
    replayed = [g.clone() for g in captured]
    fresh = step(model, batch)
    torch.cuda.synchronize()
    assert torch.equal(got, fresh)
    assert all(torch.equal(a, p.grad) for a, p in zip(replayed, model.parameters()))


def test_two_streams_at_once():
    pairs = [model_and_batch(seed) for seed in (5, 6)]
    want = []
    for model, batch in pairs:
        value = step(model, batch).clone()
        want.append((value, [p.grad.clone() for p in model.parameters()]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pairs]
    for _ in range(3):
        got = []
        for stream, (model, batch) in zip(streams, pairs):
            with torch.cuda.stream(stream):
                got.append(step(model, batch))
        torch.cuda.synchronize()
        for value, (model, _), (loss, grads) in zip(got, pairs, want):
            assert torch.equal(value, loss)
            assert all(torch.equal(p.grad, g) for p, g in zip(model.parameters(), grads))

"""The three operators together: the language model on packed rows against itself on each document alone, and a training
run of it.

Tolerances.  Both ways compute in bf16 and round alike but for the attention's probabilities and the loss's gradient: per
layer a few roundings of 2^-9 of activations of order one.  A mean loss near log(vocabulary) then agrees to 1e-3, a
parameter's gradient to 3 % of its norm (twice what two layers of independent roundings leave)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
VOCAB, D, HEADS, FFN, LAYERS = 2000, 128, 2, 256, 2


def model(**more):
    from flashlight_b200.workloads import TransformerLM
    return TransformerLM(VOCAB, D, HEADS, FFN, LAYERS, seed=3, compute_dtype=torch.bfloat16, **more)


def test_packed_rows_equal_documents_alone():
    g = torch.Generator().manual_seed(7)
    lengths = [[128, 70, 50], [200, 48]]  # of 256 positions: the first row ends in padding of 8
    T = 256
    ids = torch.randint(VOCAB, (2, T), generator=g, dtype=torch.int32)
    targets, documents = torch.full((2, T), -1, dtype=torch.int32), torch.full((2, T), -1, dtype=torch.int32)
    spans = []
    for row, ns in enumerate(lengths):
        at = 0
        for k, n in enumerate(ns):
            documents[row, at:at + n] = 10 + k
            targets[row, at:at + n] = torch.randint(VOCAB, (n,), generator=g, dtype=torch.int32)
            spans.append((row, at, n))
            at += n
    packed, alone = model(packed=True), model()
    loss = packed.loss(ids.cuda(), targets.view(-1).cuda(), documents.cuda())
    value = float(loss.tensor)
    loss.backward()
    total = sum(n for _, _, n in spans)
    mean = 0.0
    for row, at, n in spans:
        one = alone.loss(ids[row:row + 1, at:at + n].contiguous().cuda(), targets[row, at:at + n].contiguous().cuda())
        mean += float(one.tensor) * n / total
        one.backward(torch.full_like(one.tensor, n / total))
    assert abs(value - mean) < 1e-3
    for a, b in zip(packed.parameters(), alone.parameters()):
        norm = float(b.grad.double().norm())
        assert float((a.grad.double() - b.grad.double()).norm()) <= 0.03 * norm + 1e-6


@pytest.mark.parametrize("bits,more", [(32, []), (8, ["--kv-heads", "1", "--softcap", "20", "--distance-bias"])])
def test_training_learns(bits, more):
    from flashlight_b200 import packed_lm
    args = ["--batch", "4", "--length", "256", "--document", "60", "--vocab", "64", "--layers", "2", "--width", "128",
            "--heads", "2", "--lr", "2e-3", "--state-bits", str(bits)] + more
    first = packed_lm.main(args + ["--steps", "1"])
    last = packed_lm.main(args + ["--steps", "60"])
    # (tokens are uniform: what is learnt is the patterns, through the attention)
    assert last < 0.8 * first


def test_refusals():
    for more in (dict(softcap=5.0), dict(kv_heads=1), dict(distance_bias=True)):
        with pytest.raises(ValueError):
            model(**more)
    from flashlight_b200.workloads import TransformerLM
    with pytest.raises(ValueError):
        TransformerLM(VOCAB, D, HEADS, FFN, LAYERS, packed=True)
    ids = torch.zeros(1, 16, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        model().loss(ids, ids.view(-1), documents=ids)

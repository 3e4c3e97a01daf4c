"""Masked attention where a visible key is not a number: nothing of it may vanish, wherever the key stands in its block."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("bias", [False, True])
def test_visible_key(dtype, D, softcap, bias):
    """A row of the batch for each key of a block that all queries see whole.  One head has the NaN, in its k; the other
    head's results have the bits that they have without it."""
    from flashlight_b200 import functions as F
    B, Tq, Tk, H = 128, 128, 256, 2
    g = torch.Generator("cuda").manual_seed(D)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v, go = randn(B, Tq, H, D), randn(B, Tk, H, D), randn(B, Tk, H, D), randn(B, Tq, H, D)
    slopes = torch.tensor([0.02, 0.01], device="cuda") if bias else None
    mask, scale = F.attention_mask(B, Tq, Tk), 1 / math.sqrt(D)

    def both(k):
        out, lse, rest = F.masked_attention(q, k, v, mask, scale, softcap, slopes)
        return (out, lse.transpose(1, 2)) + tuple(
            F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, scale, softcap, slopes))

    clean = both(k)
    bad = k.clone()
    at = torch.arange(B, device="cuda")
    bad[at, at, 1] = float("nan")
    for name, got, want in zip(("out", "lse", "dq", "dk", "dv"), both(bad), clean):
        assert bool(torch.isfinite(want).all()), name
        assert torch.equal(got[:, :, 0], want[:, :, 0]), name
        assert bool(torch.isnan(got[:, :, 1]).all()), name


@pytest.mark.parametrize("D", [64, 128])
def test_visible_key_of_one_query(D):
    """The same where the keys of a single query are shared out among CTAs and joined."""
    from flashlight_b200 import functions as F
    T, H, dtype = 4096, 2, torch.bfloat16
    g = torch.Generator("cuda").manual_seed(D)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v = randn(1, 1, H, D), randn(1, T, H, D), randn(1, T, H, D)
    mask = F.attention_mask(1, 1, T)
    clean = F.masked_attention(q, k, v, mask, 0.125)
    for at in range(512, 640):
        bad = k.clone()
        bad[:, at, 1] = float("nan")
        got = F.masked_attention(q, bad, v, mask, 0.125)
        for a, b in zip(got[:2], clean[:2]):
            a, b = a.reshape(H, -1), b.reshape(H, -1)
            assert torch.equal(a[0], b[0]) and bool(torch.isnan(a[1]).all()), at

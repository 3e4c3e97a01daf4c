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


def test_behind_the_mask_in_the_gradient():
    """Padding of a whole block and more: nothing of its q, k, v and of its output's gradient reaches another row.  In
    blocks that are partly seen, a key behind the mask may have any score."""
    from flashlight_b200 import functions as F
    B, T, H, D = 2, 600, 2, 64
    g = torch.Generator("cuda").manual_seed(4)
    q, k, v, go = (torch.randn(B, T, H, D, generator=g, device="cuda").bfloat16() for _ in range(4))
    ids = torch.zeros(B, T, dtype=torch.int32)
    ids[:, 130:] = 1
    ids[:, 384:] = -1
    mask = F.attention_mask(B, T, documents=ids.cuda())

    def both(q, k, v, go):
        out, lse, rest = F.masked_attention(q, k, v, mask, 0.125)
        return (out,) + tuple(F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, 0.125))

    clean = both(q, k, v, go)
    bad = [t.clone() for t in (q, k, v, go)]
    for t, value in zip(bad, ("nan", "nan", "inf", "inf")):
        t[:, 384:] = float(value)
    for name, got, want in zip(("out", "dq", "dk", "dv"), both(*bad), clean):
        assert torch.equal(got, want), name
        assert bool((got[:, 384:] == 0).all()) and bool(torch.isfinite(got).all()), name
    # the first document's end is inside a block: behind it the second document's queries see nothing of the first
    far = k.clone()
    far[:, 128:130] = float("nan")
    out, lse, _ = F.masked_attention(q, far, v, mask, 0.125)
    assert torch.equal(out[:, 130:384], clean[0][:, 130:384]) and bool(torch.isnan(out[:, 129]).all())
    assert torch.equal(out[:, :128], clean[0][:, :128])

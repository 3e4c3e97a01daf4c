"""Gradients of masked attention in f16 where the output's gradient is small, as it is in training without a loss scale.

Tolerance.  dS is kept with 11 bits relative to the largest that its row (dQ) or the call (dK) can have, so dq and dk are
right to the 8 u of the tests at gradients of order one (u = 2^-12), and each result is rounded once more to f16,
which below 2^-14 has steps of 2^-24: at most 2^-25 an element, sqrt(elements) of that in the norm.  (dS rounded in
steps of 2^-24 itself: 1.7 times that bound with 750 keys and a dO of 1e-5, 3.3 times with 5000.)"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def definition(q, k, v, go, scale, softcap):
    q, k, v = (t.double().requires_grad_() for t in (q, k, v))
    rep, T = q.shape[2] // k.shape[2], q.shape[1]
    kk, vv = k.repeat_interleave(rep, 2), v.repeat_interleave(rep, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, kk) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    s = s.masked_fill(torch.triu(torch.ones(T, T, dtype=torch.bool, device="cuda"), 1), -math.inf)
    (torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), vv) * go.double()).sum().backward()
    return q.grad, k.grad, v.grad


def gradients(q, k, v, go, scale, softcap):
    from flashlight_b200 import functions as F
    mask = F.attention_mask(q.shape[0], q.shape[1])
    out, lse, rest = F.masked_attention(q, k, v, mask, scale, softcap)
    return F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, scale, softcap)


def close(got, want, name):
    off = float((got.double() - want).norm())
    assert off <= 8 * 2.0 ** -12 * float(want.norm()) + math.sqrt(want.numel()) * 2.0 ** -25, (
        name, off, float(want.norm()), math.sqrt(want.numel()) * 2.0 ** -25)


@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("T,H,Hk,D,softcap", [(750, 2, 2, 64, 0.0), (1500, 4, 1, 128, 30.0), (333, 3, 3, 40, 0.0),
                                              (5000, 1, 1, 64, 0.0)])
def test_small(T, H, Hk, D, softcap, size):
    g = torch.Generator("cuda").manual_seed(T)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v = randn(1, T, H, D).half(), randn(1, T, Hk, D).half(), randn(1, T, Hk, D).half()
    go = (randn(1, T, H, D) * size).half()
    got, want = gradients(q, k, v, go, 1.5 / math.sqrt(D), softcap), definition(q, k, v, go, 1.5 / math.sqrt(D), softcap)
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        close(a, b, name)


def test_rows_of_different_sizes():
    """Each row's dq by its own size, whatever the others'; a row that is not finite changes no other row's dq."""
    T, H, D = 600, 2, 64
    g = torch.Generator("cuda").manual_seed(7)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v = (randn(1, T, H, D).half() for _ in range(3))
    go = randn(1, T, H, D)
    go[:, ::2] *= 1e-4
    go[:, ::10] = 0
    go = go.half()
    got, want = gradients(q, k, v, go, 0.125, 0.0), definition(q, k, v, go, 0.125, 0.0)
    for rows in (slice(0, None, 2), slice(1, None, 2)):
        close(got[0][:, rows], want[0][:, rows], "dq")
    assert bool((got[0][:, ::10] == 0).all())
    close(got[1], want[1], "dk")
    close(got[2], want[2], "dv")
    small = (randn(1, T, H, D) * 1e-4).half()
    alone = gradients(q, k, v, small, 0.125, 0.0)
    small[:, T - 1] = float("inf")
    dq, dk, dv = gradients(q, k, v, small, 0.125, 0.0)
    assert torch.equal(dq[:, :T - 1], alone[0][:, :T - 1]) and not bool(torch.isfinite(dq[:, T - 1]).any())
    assert not bool(torch.isfinite(dk).any()) and not bool(torch.isfinite(dv).any())


def test_large():
    """Gradients far above one are not scaled: what fitted fits."""
    T, H, D = 256, 2, 64
    g = torch.Generator("cuda").manual_seed(9)
    q, k, v, go = (torch.randn(1, T, H, D, generator=g, device="cuda") for _ in range(4))
    q, k, v, go = q.half(), k.half(), v.half(), (go * 200).half()
    for name, a, b in zip(("dq", "dk", "dv"), gradients(q, k, v, go, 0.125, 0.0), definition(q, k, v, go, 0.125, 0.0)):
        close(a, b, name)

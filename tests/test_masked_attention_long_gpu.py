"""Masked attention and its gradient over many blocks: rows longer than 4096 (at 64 dimensions another kernel's ring,
which goes round several times on either side) and query heads that share one key head.

Against the definition in 64 bits from the same 16-bit tensors.  P and dS are rounded once to the tensors' type
before their products and each result once more; relative to a result's norm each is at most u = 2^-9 (bf16) or
2^-12 (f16) of terms that add up at random or better: 4 u holds the output and dv, 8 u dq and dk, whose terms are
differences, on the norm per head."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Tq,Tk,H,Hk,D,causal,docs,prefix,softcap,bias", [
    (4500, 4500, 2, 1, 64, True, False, 0, 0.0, False),
    (4500, 4500, 2, 2, 64, True, True, 700, 0.0, True),
    (4200, 4200, 1, 1, 40, False, True, 0, 25.0, False),
    (1000, 5000, 2, 1, 64, True, False, 0, 20.0, True),     # the last queries of a longer row
    (1700, 1700, 8, 1, 64, True, False, 0, 0.0, False),
    (1700, 1700, 6, 2, 128, True, False, 300, 30.0, False),
    (2200, 2200, 4, 1, 128, True, True, 0, 0.0, True),
    (900, 900, 12, 1, 72, False, False, 0, 0.0, False),
])
def test_output_and_gradients(Tq, Tk, H, Hk, D, causal, docs, prefix, softcap, bias, dtype):
    from flashlight_b200 import functions as F
    g = torch.Generator("cuda").manual_seed(Tk + H)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v, go = randn(1, Tq, H, D), randn(1, Tk, Hk, D), randn(1, Tk, Hk, D), randn(1, Tq, H, D)
    scale, rep = 1.5 / math.sqrt(D), H // Hk
    at = torch.arange(Tk, device="cuda")
    ids = torch.zeros(Tk, dtype=torch.int32, device="cuda")
    if docs:
        ids[300:] = 1
        ids[Tk // 2 + 7:] = 2
        ids[Tk - 130:] = -1
    pre = torch.tensor([prefix], dtype=torch.int32, device="cuda") if prefix else None
    slopes = torch.tensor([2.0 ** -(2 + h) for h in range(H)], device="cuda") if bias else None
    mask = F.attention_mask(1, Tq, Tk, causal=causal, documents=ids[None].contiguous() if docs else None, prefix=pre)
    out, lse, rest = F.masked_attention(q, k, v, mask, scale, softcap, slopes)
    grads = F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, scale, softcap, slopes)

    i, mine = at[Tk - Tq:, None], ids[Tk - Tq:, None]
    seen = (ids[None] == mine) & (mine >= 0)
    if causal:
        seen &= (at[None] <= i) | (at[None] < prefix)
    u = UNIT[dtype]

    def near(got, want, name, h, much):
        off = float((got.double() - want).norm())
        assert off <= much * u * float(want.norm()) + 1e-6, (name, h, off, float(want.norm()))

    dk, dv = torch.zeros(Tk, Hk, D, dtype=torch.float64, device="cuda"), torch.zeros(Tk, Hk, D, dtype=torch.float64,
                                                                                  device="cuda")
    for h in range(H):
        qd, kd, vd, gd = (t[0, :, x].double() for t, x in ((q, h), (k, h // rep), (v, h // rep), (go, h)))
        z, flat = qd @ kd.t() * scale, 1.0
        if softcap:
            z = torch.tanh(z / softcap)
            flat = 1 - z * z
            z = z * softcap
        if bias:
            z = z - float(slopes[h]) * (i - at[None]).abs()
        want = torch.logsumexp(z.masked_fill(~seen, -math.inf), 1)
        p = torch.where(seen, torch.exp(z - want.nan_to_num(neginf=0.0)[:, None]), 0.0)
        del z
        o = p @ vd
        live = torch.isfinite(want)
        assert torch.equal(lse[0, h] == -math.inf, ~live)
        assert bool(((lse[0, h].double() - want)[live].abs() <= 2e-5 * (1 + want[live].abs())).all())
        near(out[0, :, h], o, "out", h, 4)
        ds = p * (gd @ vd.t() - (gd * o).sum(1, keepdim=True)) * flat * scale
        near(grads[0][0, :, h], ds @ kd, "dq", h, 8)
        dk[:, h // rep] += ds.t() @ qd
        dv[:, h // rep] += p.t() @ gd
    for h in range(Hk):
        near(grads[1][0, :, h], dk[:, h], "dk", h, 8)
        near(grads[2][0, :, h], dv[:, h], "dv", h, 4)
    again = F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, scale, softcap, slopes)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))

"""Masked attention against its definition in 64 bits from the same 16-bit tensors.

Tolerances.  Scores, statistics and sums are fp32 (2^-21 and below).  P and dS are rounded once to the tensors' type
before their products and the result once more: relative to a result's norm each rounding is at most u = 2^-9
(bf16) or 2^-12 (f16) of the products' terms, which add up at random or better.  4 u holds the gradients and the
output with room, tested on the norm per head; the lse to 2e-5."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


def visible(B, Tq, Tk, causal, documents=None, prefix=None):
    """By the definition, a position at a time."""
    seen = torch.zeros(B, Tq, Tk, dtype=torch.bool)
    for b in range(B):
        ids = documents[b].tolist() if documents is not None else [0] * Tk
        run = [0]
        for p in range(1, Tk):
            run.append(run[-1] + (ids[p] != ids[p - 1]))
        run = torch.tensor(run)
        j = torch.arange(Tk)
        for i in range(Tq):
            p = i + Tk - Tq
            if ids[p] < 0:
                continue
            ok = run == run[p]
            if causal:
                ok &= (j <= p) | (j < (int(prefix[b]) if prefix is not None else 0))
            seen[b, i] = ok
    return seen


def definition(q, k, v, go, seen, scale, softcap, slopes):
    q, k, v = (t.double().requires_grad_() for t in (q, k, v))
    B, Tq, H, D = q.shape
    Tk, rep = k.shape[1], H // k.shape[2]
    kk, vv = k.repeat_interleave(rep, 2), v.repeat_interleave(rep, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, kk) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        far = (torch.arange(Tq, device=q.device)[:, None] + Tk - Tq - torch.arange(Tk, device=q.device)).abs()
        s = s - slopes.double()[:, None, None] * far
    s = s.masked_fill(~seen.to(q.device)[:, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen.to(q.device)[:, None], torch.exp(s - lse.nan_to_num(neginf=0.0)[..., None]), 0.0)
    o = torch.einsum("bhij,bjhd->bihd", p, vv)
    (o * go.double()).sum().backward()
    return o.detach(), lse.detach(), q.grad, k.grad, v.grad


def near(got, want, unit, name):
    for h in range(want.shape[2]):  # a head at a time
        off = float((got[:, :, h].double() - want[:, :, h]).norm())
        assert off <= 4 * unit * float(want[:, :, h].norm()) + 1e-6, (name, h, off, float(want[:, :, h].norm()))


def packed(B, T, mean, seed, pad=True):
    r = random.Random(seed)
    rows = []
    for _ in range(B):
        row, doc = [], 5
        while len(row) < T:
            row += [doc] * (1 + int(r.expovariate(1.0 / mean)))
            doc += 1
        row = row[:T]
        n = r.randrange(1 + T // 4) if pad else 0
        rows.append(row[:T - n] + [-1] * n)
    return torch.tensor(rows, dtype=torch.int32)


CASES = [
    # B, Tq, Tk, H, Hk, D, causal, documents, prefix, softcap, bias
    (1, 1, 1, 1, 1, 64, True, 0, False, 0.0, False),
    (2, 5, 5, 2, 1, 8, True, 0, False, 0.0, False),
    (1, 77, 77, 3, 3, 64, True, 0, True, 0.0, False),
    (2, 128, 128, 2, 2, 64, False, 0, False, 0.0, False),
    (1, 129, 129, 2, 2, 128, True, 0, False, 0.0, False),
    (2, 255, 255, 4, 2, 72, True, 40, False, 0.0, True),
    (2, 300, 300, 2, 2, 64, False, 100, False, 20.0, False),
    (1, 512, 512, 4, 1, 128, True, 0, False, 30.0, False),
    (3, 400, 400, 2, 2, 64, True, 60, True, 5.0, True),
    (1, 700, 700, 2, 1, 80, True, 3, False, 0.0, True),
    (2, 1, 500, 4, 2, 64, True, 0, False, 0.0, False),      # a single token behind a long context
    (1, 1, 1000, 2, 2, 128, True, 150, False, 10.0, True),
    (1, 130, 515, 2, 2, 64, True, 0, False, 0.0, True),
    (1, 33, 513, 2, 2, 40, False, 200, False, 0.0, False),
    (1, 1100, 1100, 1, 1, 64, True, 0, False, 0.0, False),
    (1, 1, 5000, 4, 2, 64, True, 0, False, 0.0, False),     # keys shared out among CTAs and joined
    (2, 3, 3000, 2, 1, 128, True, 700, False, 15.0, True),  # (some have no key of the query's document)
    (1, 140, 2000, 1, 1, 72, False, 900, False, 0.0, False),
    (1, 2, 1030, 1, 1, 16, True, 0, True, 0.0, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_output_and_gradients(case, dtype):
    from flashlight_b200 import autograd as A
    from flashlight_b200 import functions as F
    B, Tq, Tk, H, Hk, D, causal, docs, prefix, softcap, bias = case
    g = torch.Generator("cuda").manual_seed(Tk + H)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v, go = randn(B, Tq, H, D), randn(B, Tk, Hk, D), randn(B, Tk, Hk, D), randn(B, Tq, H, D)
    documents = packed(B, Tk, docs, Tk) if docs else None
    pre = torch.tensor([Tk // 2 - 3 * b for b in range(B)], dtype=torch.int32) if prefix else None
    slopes = torch.tensor([2.0 ** -(1 + h) for h in range(H)], device="cuda") if bias else None
    scale = 1.5 / math.sqrt(D)
    seen = visible(B, Tq, Tk, causal, documents, pre)
    want = definition(q, k, v, go, seen, scale, softcap, slopes)
    mask = F.attention_mask(B, Tq, Tk, causal=causal, documents=documents.cuda() if docs else None,
                            prefix=pre.cuda() if prefix else None, device="cuda")
    qv, kv, vv = A.Variable(q, True), A.Variable(k, True), A.Variable(v, True)
    out = A.masked_attention(qv, kv, vv, mask, scale, softcap, slopes)
    lse = F.masked_attention(q, k, v, mask, scale, softcap, slopes)[1]
    result = out.tensor
    out.backward(go)
    empty = ~seen.any(-1).cuda()
    assert bool((result[empty] == 0).all()) and bool((qv.grad[empty] == 0).all())
    assert torch.equal(torch.isinf(lse).transpose(1, 2), empty[..., None].expand(-1, -1, H))
    finite = torch.isfinite(lse)
    assert bool(((lse - want[1])[finite].abs() <= 2e-5 * (1 + want[1][finite].abs())).all())
    u = UNIT[dtype]
    near(result, want[0], u, "out")
    near(vv.grad, want[4], u, "dv")
    if int(seen.sum(-1).max()) > 1:
        # dS of a row of few keys is a difference of nearly equal numbers: of the size of its terms
        near(qv.grad, want[2], 2 * u, "dq")
        near(kv.grad, want[3], 2 * u, "dk")


def test_mask_tables():
    """The intervals of every query, over long rows with runs across the scan's chunks."""
    from flashlight_b200 import functions as F
    T = 9001
    ids = torch.zeros(3, T, dtype=torch.int32)
    ids[0, 4095:] = 1          # a run that begins at a chunk's last position
    ids[0, 4097:8200] = 2
    ids[1] = -1
    ids[1, 10:8193] = 7
    ids[2, ::2] = 1            # runs of one
    pre = torch.tensor([5000, 8000, 3], dtype=torch.int32)
    for causal, prefix in ((True, None), (True, pre), (False, None)):
        m = F.attention_mask(3, T, causal=causal, documents=ids.cuda(), prefix=prefix.cuda() if prefix is not None else None)
        nq = (T + 127) // 128
        tables = 3 * nq * 16 + (3 * nq * 8 + 15) // 16 * 16
        rows = m.data[tables:].view(torch.int32).view(3, T, 2).cpu()
        for b in range(3):
            change = torch.cat([torch.tensor([True]), ids[b, 1:] != ids[b, :-1]])
            begin = torch.where(change, torch.arange(T), 0).cummax(0)[0]
            end = torch.tensor(T) - torch.where(torch.cat([change[1:], torch.tensor([True])]),
                                                T - 1 - torch.arange(T), 0).flip(0).cummax(0)[0].flip(0)
            hi = torch.arange(T) + 1 if causal else end
            if prefix is not None:
                hi = torch.minimum(end, torch.maximum(hi, prefix[b]))
            lo = torch.where(ids[b] < 0, 0, begin)
            hi = torch.where(ids[b] < 0, 0, hi)
            assert torch.equal(rows[b, :, 1], hi.int()) or bool((rows[b, :, 1] <= rows[b, :, 0])[ids[b] < 0].all())
            live = ids[b] >= 0
            assert torch.equal(rows[b, live, 0], lo[live].int()) and torch.equal(rows[b, live, 1], hi[live].int())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strides_and_packed(dtype):
    """Views of a packed projection, heads before positions, a batch that is broadcast, rows off alignment."""
    from flashlight_b200 import autograd as A
    from flashlight_b200 import functions as F
    B, T, H, Hk, D = 2, 200, 4, 2, 64
    g = torch.Generator("cuda").manual_seed(2)
    qkv = torch.randn(B * T, (H + 2 * Hk) * D, generator=g, device="cuda").to(dtype)
    go = torch.randn(B * T, H * D, generator=g, device="cuda").to(dtype)
    mask = F.attention_mask(B, T)
    x = A.Variable(qkv, True)
    out = A.masked_attention_packed(x, H, mask, 0.1, kv_heads=Hk)
    result = out.tensor
    out.backward(go)
    t = qkv.view(B, T, H + 2 * Hk, D)
    parts = [t[:, :, :H], t[:, :, H:H + Hk], t[:, :, H + Hk:]]
    same = [A.Variable(p.contiguous(), True) for p in parts]
    o2 = A.masked_attention(*same, mask, 0.1)
    r2 = o2.tensor
    o2.backward(go.view(B, T, H, D))
    assert torch.equal(result.view(B, T, H, D), r2)
    assert torch.equal(x.grad.view(t.shape), torch.cat([s.grad for s in same], 2))
    # other orders of the same values, and values that are no 16-byte rows
    heads_first = [p.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for p in parts]
    odd = [torch.empty(p.numel() + 1, dtype=dtype, device="cuda")[1:].view(p.shape).copy_(p) for p in parts]
    last = [p.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2) for p in parts]
    for other in (heads_first, odd, last):
        vs = [A.Variable(p, True) for p in other]
        o3 = A.masked_attention(*vs, mask, 0.1)
        assert torch.equal(o3.tensor, r2)
        o3.backward(go.view(B, T, H, D))
        for a, b in zip(vs, same):
            assert torch.equal(a.grad, b.grad)
    one = parts[1][:1].expand(B, T, Hk, D)
    o4 = F.masked_attention(parts[0], one, one, mask, 0.1)[0]
    o5 = F.masked_attention(parts[0], one.contiguous(), one.contiguous(), mask, 0.1)[0]
    assert torch.equal(o4, o5)


def test_values_behind_the_mask():
    """What no query of a block sees may be anything; a masked key's infinite score leaves no trace."""
    from flashlight_b200 import functions as F
    B, T, H, D = 1, 300, 2, 64
    g = torch.Generator("cuda").manual_seed(4)
    q, k, v, go = (torch.randn(B, T, H, D, generator=g, device="cuda").bfloat16() for _ in range(4))
    ids = torch.zeros(B, T, dtype=torch.int32)
    ids[:, 128:] = 1
    ids[:, 256:] = -1          # padding: a whole block that nobody sees
    mask = F.attention_mask(B, T, documents=ids.cuda())
    clean = F.masked_attention(q, k, v, mask, 0.125)
    bad = [t.clone() for t in (q, k, v)]
    bad[1][:, 256:] = float("nan")
    bad[2][:, 256:] = float("inf")
    bad[0][:, 256:] = float("nan")
    dirty = F.masked_attention(*bad, mask, 0.125)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    # keys whose scores overflow, seen by nobody of the rows that come before them
    k2 = k.clone()
    k2[:, 100:128] = 1e38
    got = F.masked_attention(q, k2, v, mask, 0.125)[0]
    assert torch.equal(got[:, :100], clean[0][:, :100])
    # gradients of the rows that count, with the padding's dO infinite in the rows that do not exist for the mask
    grads = F.masked_attention_backward(q, k, v, clean[0], clean[2], go, clean[1], mask, 0.125)
    assert all(bool(torch.isfinite(x).all()) for x in grads)
    assert bool((grads[1][:, 256:] == 0).all()) and bool((grads[2][:, 256:] == 0).all())
    assert bool((grads[0][:, 256:] == 0).all())


def test_large_scores_and_equal_bits():
    """Scores far beyond exp's range, maxima that rise from block to block; the same bits twice."""
    from flashlight_b200 import functions as F
    B, T, H, D = 1, 700, 2, 64
    g = torch.Generator("cuda").manual_seed(6)
    q, k, v, go = (torch.randn(B, T, H, D, generator=g, device="cuda") for _ in range(4))
    k = k * torch.linspace(0.1, 40, T, device="cuda")[None, :, None, None]  # spread of hundreds
    q, k, v, go = (t.bfloat16() for t in (q, k, v, go))
    seen = visible(B, T, T, True)
    want = definition(q, k, v, go, seen, 1.0, 0.0, None)
    mask = F.attention_mask(B, T)
    out, lse, rest = F.masked_attention(q, k, v, mask, 1.0)
    near(out, want[0], UNIT[torch.bfloat16], "out")
    a = F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, 1.0)
    b = F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, 1.0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for got, w, name in zip(a, want[2:], ("dq", "dk", "dv")):
        near(got, w, 4 * UNIT[torch.bfloat16], name)


def test_gradient_is_the_differences():
    from flashlight_b200 import functions as F
    B, T, H, D = 1, 150, 2, 32
    g = torch.Generator("cuda").manual_seed(8)
    q, k, v, go = (torch.randn(B, T, H, D, generator=g, device="cuda").half() for _ in range(4))
    mask = F.attention_mask(B, T)
    slopes = torch.tensor([0.1, 0.3], device="cuda")
    out, lse, rest = F.masked_attention(q, k, v, mask, 0.3, 4.0, slopes)
    grads = F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, 0.3, 4.0, slopes)
    f = lambda a, b, c: float((F.masked_attention(a, b, c, mask, 0.3, 4.0, slopes)[0].double() * go.double()).sum())  # noqa: E731
    for i in range(3):
        e = torch.sign(grads[i].float()) * 2.0 ** -6
        up, down = [[q, k, v] for _ in range(2)]
        up[i], down[i] = (up[i].float() + e).half(), (down[i].float() - e).half()
        along = float((grads[i].double() * (up[i].double() - down[i].double())).sum())
        assert abs(f(*up) - f(*down) - along) <= 0.02 * abs(along)


def test_refusals():
    from flashlight_b200 import autograd as A
    from flashlight_b200 import functions as F
    t = lambda *s, dt=torch.bfloat16: torch.zeros(s, device="cuda", dtype=dt)  # noqa: E731
    mask = F.attention_mask(1, 16)
    q = t(1, 16, 4, 64)
    ids = torch.zeros(1, 16, dtype=torch.int32, device="cuda")
    for bad in (lambda: F.attention_mask(0, 4), lambda: F.attention_mask(1, 5, 4),
                lambda: F.attention_mask(1, 16, documents=ids.long()),
                lambda: F.attention_mask(2, 16, documents=ids),
                lambda: F.attention_mask(1, 16, documents=ids.cpu()),
                lambda: F.attention_mask(1, 16, causal=False, prefix=ids[0, :1]),
                lambda: F.masked_attention(q, t(1, 16, 3, 64), t(1, 16, 3, 64), mask, 1.0),
                lambda: F.masked_attention(q, q, t(1, 16, 2, 64), mask, 1.0),
                lambda: F.masked_attention(q, q.half(), q.half(), mask, 1.0),
                lambda: F.masked_attention(t(1, 15, 4, 64), q, q, mask, 1.0),
                lambda: F.masked_attention(q, q, q, mask, 0.0),
                lambda: F.masked_attention(q, q, q, mask, 1.0, -1.0),
                lambda: F.masked_attention(q, q, q, mask, 1.0, 0.0, torch.zeros(3, device="cuda")),
                lambda: F.masked_attention(q[0], q[0], q[0], mask, 1.0),
                lambda: A.masked_attention_packed(A.Variable(t(16, 100), True), 4, mask, 1.0)):
        with pytest.raises(ValueError):
            bad()
    for x in (t(1, 16, 4, 65), t(1, 16, 4, 136), t(1, 16, 4, 64, dt=torch.float32)):
        with pytest.raises(RuntimeError):
            F.masked_attention(x, x, x, mask, 1.0)

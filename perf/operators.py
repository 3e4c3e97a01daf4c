"""What a training step of a language model over packed documents is measured on beyond cases.py: its
attention, its loss and its optimiser, each called as the step calls it.

  attention  softmax(cap(scale q k^T) - slope |i - j|) v over the keys that a query sees, mask included:
             forward, or forward and gradient
  loss       cross entropy of x W + b over a vocabulary: forward, or forward and gradient
  adamw      one AdamW step over all parameters, states of 32 bits or 8

With `own` the calls are the framework's; without, the same in elementary torch operations in 32 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 256         # elements of an 8-bit state that share a scale
E4M3_MAX = 448.0
ADAMW = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


def listed():
    return [
        # a prompt scored in evaluation mode, its first 20 positions seen by all: one sequence, latency
        dict(name="attention_prompt_t77", op="attention", train=False, batch=1, q_len=77, k_len=77, heads=12,
             kv_heads=12, head_dim=64, dtype="bf16", causal=True, documents=0, prefix=20, softcap=0.0, bias=False),
        # the Transformer workload's own attention (8 x 512, 12 heads of 64), rows packed with documents
        dict(name="attention_packed_train_t512", op="attention", train=True, batch=8, q_len=512, k_len=512,
             heads=12, kv_heads=12, head_dim=64, dtype="bf16", causal=True, documents=150, prefix=0, softcap=0.0,
             bias=False),
        # capped scores, four query heads to a key head of 128, a length off the tiles, f16
        dict(name="attention_capped_train_t1500", op="attention", train=True, batch=2, q_len=1500, k_len=1500,
             heads=16, kv_heads=4, head_dim=128, dtype="f16", causal=True, documents=0, prefix=0, softcap=30.0,
             bias=False),
        # long rows of few long documents with a distance bias
        dict(name="attention_long_train_t8192", op="attention", train=True, batch=1, q_len=8192, k_len=8192,
             heads=12, kv_heads=12, head_dim=64, dtype="bf16", causal=True, documents=3000, prefix=0, softcap=0.0,
             bias=True),
        # the perplexity of a short text: few rows against a small vocabulary
        dict(name="loss_eval_r61", op="loss", train=False, rows=61, dim=512, vocab=8000, dtype="bf16", bias=True,
             ignored=0.0),
        # the Transformer workload's head: 8 x 512 tokens, 768 features, 32000 classes
        dict(name="loss_train_r4096_v32000", op="loss", train=True, rows=4096, dim=768, vocab=32000, dtype="bf16",
             bias=True, ignored=0.0),
        # rows and vocabulary off every tile, a tenth of the targets ignored, f16
        dict(name="loss_train_r2055_v50001", op="loss", train=True, rows=2055, dim=1000, vocab=50001, dtype="f16",
             bias=False, ignored=0.1),
        # a large head
        dict(name="loss_train_r8192_v128000", op="loss", train=True, rows=8192, dim=2048, vocab=128000,
             dtype="bf16", bias=False, ignored=0.0),
        # norms and biases only: a hundred short tensors, latency
        dict(name="adamw_100_short", op="adamw", tensors=100, elements=60_000, sizes=1, param="f32", grad="f32",
             bits=32),
        # the Transformer workload's parameters and their fp32 gradients
        dict(name="adamw_lm_134m", op="adamw", tensors=148, elements=134_000_000, sizes=2, param="f32", grad="f32",
             bits=32),
        # fp32 master weights with bf16 gradients and states in 8 bits, odd sizes
        dict(name="adamw_8bit_30m", op="adamw", tensors=64, elements=30_000_001, sizes=3, param="f32", grad="bf16",
             bits=8),
        # a large model all in 16 and 8 bits
        dict(name="adamw_8bit_1g", op="adamw", tensors=200, elements=1_000_000_000, sizes=4, param="bf16",
             grad="bf16", bits=8),
    ]


def _log(rng, low, high, step=1):
    """A size between low and high, spread over its logarithm, in whole steps (no feed-forward width of the
    Transformer workload by chance: it stands for itself elsewhere)."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step
    n = min(max(n, low), high)
    return n + step if n == 3072 else n


def draw(rng):
    op = rng.choice(["attention", "loss", "adamw"])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        train = rng.random() < 0.7
        k_len = _log(rng, 8 if train else 1, 6000)  # (of one visible key the scores' gradient is zero)
        batch = max(1, min(_log(rng, 1, 16), int(6e8 / (heads * k_len * k_len + 1))))
        q_len = k_len if rng.random() < 0.8 else _log(rng, 1, k_len) if k_len > 1 else 1
        causal = rng.random() < 0.8
        return dict(op=op, train=train, batch=batch, q_len=q_len, k_len=k_len, heads=heads,
                    kv_heads=kv_heads, head_dim=rng.choice([32, 64, 64, 80, 128]),
                    dtype=rng.choice(["bf16", "f16"]), causal=causal,
                    documents=_log(rng, 3, 4000) if rng.random() < 0.5 else 0,
                    prefix=_log(rng, 1, k_len) if causal and k_len > 1 and rng.random() < 0.3 else 0,
                    softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.4)
    if op == "loss":
        dim, vocab = _log(rng, 64, 2048, 8), _log(rng, 500, 128000)
        rows = _log(rng, 1, max(2, min(8192, int(1.2e12 / (dim * vocab)))))
        return dict(op=op, train=rng.random() < 0.8, rows=rows, dim=dim, vocab=vocab,
                    dtype=rng.choice(["bf16", "f16"]), bias=rng.random() < 0.5,
                    ignored=rng.choice([0.0, 0.0, 0.2]))
    elements = _log(rng, 5_000, 600_000_000)
    param = rng.choice(["f32", "f32", "bf16", "f16"])
    return dict(op=op, tensors=_log(rng, 1, 200), elements=elements, sizes=rng.randrange(1 << 20), param=param,
                grad=rng.choice(["f32", "bf16", "f16"]) if param == "f32" else param, bits=rng.choice([32, 8]))


# ---------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def prepare(case, seed):
    return {"attention": _prepare_attention, "loss": _prepare_loss, "adamw": _prepare_adamw}[case["op"]](case, seed)


def _prepare_attention(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "head_dim"))
    s = dict(case=case, q=_randn(g, b, tq, h, d, dtype=dt), k=_randn(g, b, tk, hk, d, dtype=dt),
             v=_randn(g, b, tk, hk, d, dtype=dt), documents=None, prefix=None, slopes=None,
             scale=1.0 / math.sqrt(d))
    if case["softcap"]:  # trained scores reach the cap
        s["q"] *= 3
    if case["train"]:
        s["grad"] = _randn(g, b, tq, h, d, dtype=dt)
    if case["documents"]:
        # ends of documents of that mean length; what is behind a row's last document is padding (-1)
        r = random.Random(seed)
        ids = []
        for _ in range(b):
            row, doc = [], 0
            while len(row) < tk:
                row += [doc] * min(tk, 1 + int(r.expovariate(1.0 / case["documents"])))
                doc += 1
            pad = r.randrange(1 + min(tk - 1, tk // 16))
            ids.append(row[:tk - pad] + [-1] * pad)
        s["documents"] = torch.tensor(ids, dtype=torch.int32).cuda()
    if case["prefix"]:
        r = random.Random(seed + 1)
        s["prefix"] = torch.tensor([r.randint(case["prefix"] // 2, case["prefix"]) for _ in range(b)],
                                   dtype=torch.int32).cuda()
    if case["bias"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)]).cuda()
    return s


def _prepare_loss(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    r, d, v = case["rows"], case["dim"], case["vocab"]
    s = dict(case=case, x=_randn(g, r, d, dtype=dt), w=_randn(g, d, v, dtype=dt).mul_(1.5 / math.sqrt(d)),
             b=_randn(g, v).mul_(0.1) if case["bias"] else None,
             targets=torch.randint(0, v, (r,), generator=g, device="cuda", dtype=torch.int32))
    if case["ignored"]:
        s["targets"][torch.rand(r, generator=g, device="cuda") < case["ignored"]] = -1
    s["targets"][0] = v - 1
    return s


def _sizes(case):
    """Lengths of the case's tensors: a few long ones hold most of the elements."""
    r, n, total = random.Random(case["sizes"]), case["tensors"], case["elements"]
    n = min(n, total)
    weights = [math.exp(r.uniform(0.0, 6.0)) for _ in range(n)]
    sizes = [max(1, int(total * w / sum(weights))) for w in weights]
    sizes[-1] = max(1, sizes[-1] + total - sum(sizes))
    return sizes


def _prepare_adamw(case, seed):
    g, sizes = _generator(seed), _sizes(case)
    starts, at = [], 0
    for n in sizes:  # tensors of one arena, each on a block of its own; what is between them stays zero
        starts.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    views = lambda arena: [arena[a:a + n] for a, n in zip(starts, sizes)]  # noqa: E731

    def filled(dtype, scale, spread):
        arena = torch.zeros(at, device="cuda", dtype=dtype)
        for k, v in enumerate(views(arena)):
            v.normal_(0.0, scale * 10.0 ** (spread * ((k * 7) % 5 - 2)), generator=g)
        return arena

    s = dict(case=case, param=filled(DTYPES[case["param"]], 0.02, 0.0),
             grad=filled(DTYPES[case["grad"]], 1e-3, 0.5), step=20)
    first, second = filled(torch.float32, 3e-4, 0.5), filled(torch.float32, 1e-3, 0.5).abs_()
    if case["bits"] == 8:
        s["first"], s["first_scale"] = _to_8bit(first, False)
        s["second"], s["second_scale"] = _to_8bit(second, True)
    else:
        s["first"], s["second"] = first, second.square_()
    for k in ("param", "grad", "first", "second"):
        s[k + "s"] = views(s[k])
    for k in ("first_scale", "second_scale"):
        s[k + "s"] = [s[k][a // BLOCK:(a + n + BLOCK - 1) // BLOCK] for a, n in zip(starts, sizes)] if k in s else None
    return s


# ---------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "loss": _own_loss, "adamw": _own_adamw}[op](state)
    return {"attention": _plain_attention, "loss": _plain_loss, "adamw": _plain_adamw}[op](state)


def _own_attention(s):
    from flashlight_b200 import autograd as A
    from flashlight_b200 import functions as F
    c, train = s["case"], s["case"]["train"]
    mask = F.attention_mask(c["batch"], c["q_len"], c["k_len"], causal=c["causal"], documents=s["documents"],
                            prefix=s["prefix"], device=s["q"].device)
    q, k, v = (A.Variable(s[n], train) for n in "qkv")
    out = A.masked_attention(q, k, v, mask, s["scale"], softcap=c["softcap"], slopes=s["slopes"])
    if not train:
        return out.tensor
    result = out.tensor
    out.backward(s["grad"])
    return result, q.grad, k.grad, v.grad


def _own_loss(s):
    from flashlight_b200 import autograd as A
    train = s["case"]["train"]
    x, w = A.Variable(s["x"], train), A.Variable(s["w"], train)
    b = A.Variable(s["b"], train) if s["b"] is not None else None
    loss = A.linear_cross_entropy(x, w, b, s["targets"])
    if not train:
        return loss.tensor
    result = loss.tensor
    loss.backward()
    return (result, x.grad, w.grad) + ((b.grad,) if b is not None else ())


def _own_adamw(s):
    from flashlight_b200 import functions as F
    s["step"] += 1
    F.adamw_step(s["params"], s["grads"], s["firsts"], s["seconds"], first_scales=s["first_scales"],
                 second_scales=s["second_scales"], step=s["step"], **ADAMW)
    return _adamw_outputs(s)


# ---------------------------------------------------------------------------------------- plain forms
def _plain_attention(s):
    c = s["case"]
    b, tq, tk, h, hk, d = (c[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "head_dim"))
    rep = h // hk
    q = s["q"].float().permute(0, 2, 1, 3).reshape(b, hk, rep * tq, d)
    k, v = (s[n].float().permute(0, 2, 1, 3) for n in "kv")
    i = torch.arange(tk - tq, tk, device="cuda")[:, None]
    j = torch.arange(tk, device="cuda")[None, :]
    seen = torch.ones(1, tq, tk, dtype=torch.bool, device="cuda")
    if c["causal"]:
        seen = (j <= i)[None]
        if s["prefix"] is not None:
            seen = seen | (j[None] < s["prefix"][:, None, None])
    if s["documents"] is not None:
        ids = s["documents"]
        run_of = torch.nn.functional.pad((ids[:, 1:] != ids[:, :-1]).int(), (1, 0)).cumsum(1)
        seen = seen & (run_of[:, tk - tq:, None] == run_of[:, None, :]) & (ids[:, tk - tq:, None] >= 0)
    seen = seen[:, None, None]                                             # (b, 1, 1, tq, tk)
    z = (q @ k.transpose(2, 3)).view(b, hk, rep, tq, tk).mul_(s["scale"])
    tanh = None
    if c["softcap"]:
        tanh = torch.tanh(z.div_(c["softcap"]))
        z = tanh * c["softcap"]
    if s["slopes"] is not None:
        z = z - s["slopes"].view(1, hk, rep, 1, 1) * (i - j).abs().float()
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True).clamp_(min=-3e38)
    p = (z - top).exp_()
    del z
    p = p / p.sum(-1, keepdim=True).clamp_(min=1e-38)
    o = (p.view(b, hk, rep * tq, tk) @ v).view(b, hk, rep, tq, d)
    heads_first = lambda t, n: t.reshape(b, n, -1, d).permute(0, 2, 1, 3).contiguous()  # noqa: E731
    out = heads_first(o, h).to(s["q"].dtype)
    if not c["train"]:
        return out
    go = s["grad"].float().permute(0, 2, 1, 3).reshape(b, hk, rep * tq, d)
    gv = p.view(b, hk, rep * tq, tk).transpose(2, 3) @ go
    gp = (go @ v.transpose(2, 3)).view(b, hk, rep, tq, tk)
    gz = gp.sub_((go.view(b, hk, rep, tq, d) * o).sum(-1, keepdim=True)).mul_(p)
    del p
    if tanh is not None:
        gz = gz * (1 - tanh * tanh)
    gz = gz.mul_(s["scale"]).view(b, hk, rep * tq, tk)
    gq, gk = gz @ k, gz.transpose(2, 3) @ q
    return (out, heads_first(gq, h).to(out.dtype), heads_first(gk, hk).to(out.dtype),
            heads_first(gv, hk).to(out.dtype))


def _plain_loss(s):
    x, w, t = s["x"].float(), s["w"].float(), s["targets"].long()
    z = x @ w
    if s["b"] is not None:
        z += s["b"]
    kept = t >= 0
    at = t.clamp(min=0)[:, None]
    top = z.amax(1, keepdim=True)
    total = (z - top).exp_().sum(1, keepdim=True)
    lse = top + total.log()
    count = kept.sum()
    loss = (torch.where(kept[:, None], lse - z.gather(1, at), torch.zeros_like(lse)).sum() / count).reshape(1)
    if not s["case"]["train"]:
        return loss
    z.sub_(lse).exp_()
    z.scatter_add_(1, at, -torch.ones_like(lse))
    z *= (kept / count)[:, None]
    gx, gw = (z @ w.t()).to(s["x"].dtype), (x.t() @ z).to(s["w"].dtype)
    return (loss, gx, gw) + ((z.sum(0),) if s["b"] is not None else ())


def _to_8bit(values, positive):
    """Blocks of 256 as e4m3 of their largest magnitude: (codes, scales).  positive: values above zero keep a
    code above zero, because they divide."""
    blocks = values.view(-1, BLOCK)
    top = blocks.abs().amax(1, keepdim=True).clamp_(min=1e-30)
    scaled = blocks * (E4M3_MAX / top)
    if positive:
        scaled = torch.where(blocks > 0, scaled.clamp(min=2.0 ** -9), scaled)
    return scaled.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(-1), (top / E4M3_MAX).view(-1)


def _of_8bit(codes, scales):
    return (codes.view(-1, BLOCK).float() * scales[:, None]).view(-1)


def _plain_adamw(s):
    eight, a = s["case"]["bits"] == 8, ADAMW
    s["step"] += 1
    g = s["grad"].float()
    m = _of_8bit(s["first"], s["first_scale"]) if eight else s["first"]
    v = _of_8bit(s["second"], s["second_scale"]).square_() if eight else s["second"]
    m = m * a["beta1"] + g * (1 - a["beta1"])
    v = v * a["beta2"] + g * g * (1 - a["beta2"])  # (g may be the gradient itself)
    del g
    root = v.sqrt()
    update = m / (1 - a["beta1"] ** s["step"]) / (root / math.sqrt(1 - a["beta2"] ** s["step"]) + a["eps"])
    p = s["param"].float()
    s["param"].copy_(p - a["lr"] * (update + a["weight_decay"] * p))
    del p, update
    if eight:
        for name, value, positive in (("first", m, False), ("second", root, True)):
            codes, scales = _to_8bit(value, positive)
            s[name].view(torch.uint8).copy_(codes.view(torch.uint8))
            s[name + "_scale"].copy_(scales)
    else:
        s["first"].copy_(m)
        s["second"].copy_(v)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {k: s[k] for k in ("param", "first", "second", "first_scale", "second_scale") if k in s}


# ---------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "loss": _exact_loss, "adamw": _exact_adamw}[case["op"]](s)


def _exact_attention(s):
    """By the definition, one head of one sequence at a time."""
    c = s["case"]
    b, tq, tk, h, hk = (c[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads"))
    if 2e-11 * b * h * tq * tk * c["head_dim"] > 15:
        return None
    out, gq = (torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") for _ in "ab")
    gk, gv = (torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in "ab")
    where = torch.arange(tk, device="cuda")
    mine = where[tk - tq:]
    for n in range(b):
        hidden = torch.zeros(tq, tk, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden |= where[None, :] > mine[:, None]
            if s["prefix"] is not None:
                hidden[:, :int(s["prefix"][n])] = False
        if s["documents"] is not None:
            ids = s["documents"][n].tolist()
            first, begin = [], 0
            for p, doc in enumerate(ids):
                begin = p if p and doc != ids[p - 1] else begin
                first.append(begin)
            first = torch.tensor(first, device="cuda")
            hidden |= first[None, :] != first[mine][:, None]
            hidden |= s["documents"][n][mine][:, None] < 0
        for m in range(h):
            q, k, v = s["q"][n, :, m].double(), s["k"][n, :, m * hk // h].double(), s["v"][n, :, m * hk // h].double()
            raw = s["scale"] * (q @ k.T)
            slope = torch.ones_like(raw)
            if c["softcap"]:
                capped = c["softcap"] * torch.tanh(raw / c["softcap"])
                slope, raw = 1 - (capped / c["softcap"]) ** 2, capped
            if s["slopes"] is not None:
                raw = raw - float(s["slopes"][m]) * (mine[:, None] - where[None, :]).abs()
            weight = torch.softmax(raw.masked_fill(hidden, -math.inf), 1).nan_to_num(0.0)
            del raw
            out[n, :, m] = weight @ v
            if c["train"]:
                go = s["grad"][n, :, m].double()
                gv[n, :, m * hk // h] += weight.T @ go
                gs = go @ v.T
                gs = weight * (gs - (weight * gs).sum(1, keepdim=True)) * slope * s["scale"]
                gq[n, :, m] = gs @ k
                gk[n, :, m * hk // h] += gs.T @ q
    return (out, gq, gk, gv) if c["train"] else out


def _exact_loss(s):
    """By the definition, some rows at a time."""
    c = s["case"]
    if 8e-13 * c["rows"] * c["dim"] * c["vocab"] > 15:
        return None
    w, n = s["w"].double(), int((s["targets"] >= 0).sum())
    loss = torch.zeros(1, dtype=torch.float64, device="cuda")
    gx = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    gw, gb = torch.zeros_like(w), torch.zeros(c["vocab"], dtype=torch.float64, device="cuda")
    for a in range(0, c["rows"], 1024):
        x, t = s["x"][a:a + 1024].double(), s["targets"][a:a + 1024].long()
        x, t, rows = x[t >= 0], t[t >= 0], torch.arange(a, a + len(t), device="cuda")[t >= 0]
        logp = x @ w if s["b"] is None else torch.addmm(s["b"].double(), x, w)
        logp = torch.log_softmax(logp, 1)
        pick = torch.arange(len(t), device="cuda"), t
        loss -= logp[pick].sum() / n
        if c["train"]:
            g = logp.exp_()
            g[pick] -= 1
            g /= n
            gx[rows] = g @ w.T
            gw += x.T @ g
            gb += g.sum(0)
    if not c["train"]:
        return loss
    return (loss, gx, gw) + ((gb,) if s["b"] is not None else ())


def _exact_adamw(s):
    """By the definition, some blocks at a time."""
    eight, a, t = s["case"]["bits"] == 8, ADAMW, s["step"] + 1
    names = ("param", "first", "second") + (("first_scale", "second_scale") if eight else ())
    out = {k: torch.empty(s[k].shape, dtype=torch.float64, device="cuda") for k in names}

    def e4m3(x):
        unit = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(x / unit) * unit

    piece = BLOCK << 17
    for lo in range(0, s["param"].numel(), piece):
        part = slice(lo, lo + piece)
        blocks = slice(lo // BLOCK, (lo + piece) // BLOCK)
        p, g, m, v = (s[k][part].double() for k in ("param", "grad", "first", "second"))
        if eight:
            m = (m.view(-1, BLOCK) * s["first_scale"][blocks].double()[:, None]).view(-1)
            v = (v.view(-1, BLOCK) * s["second_scale"][blocks].double()[:, None]).view(-1) ** 2
        m = a["beta1"] * m + (1 - a["beta1"]) * g
        v = a["beta2"] * v + (1 - a["beta2"]) * g * g
        hat_m, hat_v = m / (1 - a["beta1"] ** t), v / (1 - a["beta2"] ** t)
        out["param"][part] = p - a["lr"] * (hat_m / (hat_v.sqrt() + a["eps"]) + a["weight_decay"] * p)
        if eight:
            for k, x in (("first", m), ("second", v.sqrt())):
                x = x.view(-1, BLOCK)
                scale = x.abs().amax(1, keepdim=True).clamp(min=1e-30) / E4M3_MAX
                code = e4m3(x / scale)
                if k == "second":
                    code = torch.where(x > 0, code.clamp(min=2.0 ** -9), code)
                out[k][part], out[k + "_scale"][blocks] = code.view(-1), scale.view(-1)
        else:
            out["first"][part], out["second"][part] = m, v
    return out


# ---------------------------------------------------------------------------------------- work
def work(case):
    """Each input read and each output written once; of the products those that the result needs, the gradient's
    recomputed scores among them (they are not kept), over the pairs that a mask of the case's kind leaves."""
    if case["op"] == "attention":
        b, tq, tk, h, hk, d = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "head_dim"))
        e = BYTES[case["dtype"]]
        mean = min(tk, case["documents"]) if case["documents"] else tk
        pairs = tq * min(tk, mean * (1.0 if not case["causal"] else 0.5) + (0 if mean < tk else (tk - tq) * 0.5))
        pairs = max(pairs, tq)
        forward = 4.0 * b * h * d * pairs
        io = b * d * (2 * tq * h + 2 * tk * hk) * e
        return dict(bytes=io * (1 if not case["train"] else 3), flops=forward * (1 if not case["train"] else 3.5))
    if case["op"] == "loss":
        r, d, v, e = case["rows"], case["dim"], case["vocab"], BYTES[case["dtype"]]
        once = (r * d + d * v) * e
        return dict(bytes=once * (3 if case["train"] else 1) + 4 * r,
                    flops=2.0 * r * d * v * (4 if case["train"] else 1))
    n, state = case["elements"], 8 if case["bits"] == 32 else 2 + 8 / BLOCK
    return dict(bytes=n * (2 * BYTES[case["param"]] + BYTES[case["grad"]] + 2 * state), flops=16.0 * n)

"""What four further language-model operators of ``ad_b200.ops`` are measured on.

The ends and the middle of a language model's training step, and what happens to its gradients
before the update:

* ``embed``            scaled rows of an embedding table for given tokens, and the table's gradient,
                       summed by token
* ``feed_forward``     a gated feed-forward block, y = (act(x Wg^T) * (x Wu^T)) Wd^T, with its gradients
* ``linear_logprobs``  log probabilities of given tokens under softmax(scale x W^T) over a large
                       vocabulary, whose logits are not kept, with its gradients
* ``clip_norm``        the norm of all gradients of a model and their scaling down to a largest norm

Where ``own`` is false ``run`` computes them from elementary torch operations in 32 bits, rounded
once at the end; where it is true it calls the framework.  ``exact`` computes them in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one new token for each of 32 sequences: launch latency counts
        dict(name="embed decode", op="embed", rows=32, vocab=32000, width=512, dtype="bf16", grad="bf16", scale=22.0,
             skew=False, train=False),
        # an fp32 training step of 32 sequences of 509 tokens; the odd vocabulary is a tokenizer's
        dict(name="embed train fp32", op="embed", rows=32 * 509, vocab=50001, width=1024, dtype="f32", grad="f32",
             scale=32.0, skew=True, train=True),
        # a large bf16 step whose table's gradient is held in fp32; frequent tokens come up thousands of times
        dict(name="embed train large", op="embed", rows=131072, vocab=131072, width=2048, dtype="bf16", grad="f32",
             scale=1.0, skew=True, train=True),
        # a few tokens being generated
        dict(name="feed-forward decode", op="feed_forward", rows=4, width=1024, hidden=4096, dtype="bf16", act="silu",
             train=False),
        # one training step of a small encoder, a row short of 32 sequences of 128
        dict(name="feed-forward train small", op="feed_forward", rows=4095, width=512, hidden=2048, dtype="f16",
             act="gelu", train=True),
        # sizes that no tile divides and whose rows are not aligned
        dict(name="feed-forward train odd", op="feed_forward", rows=3001, width=1001, hidden=2731, dtype="bf16",
             act="gelu_tanh", train=True),
        # a large training step
        dict(name="feed-forward train large", op="feed_forward", rows=16384, width=2048, hidden=8192, dtype="bf16",
             act="silu", train=True),
        # scoring the last positions of a few sequences
        dict(name="linear logprobs score", op="linear_logprobs", rows=64, width=512, vocab=32000, dtype="bf16",
             scale=1.25, train=False, ignored=False),
        # a training step in fp16 with an odd vocabulary and an odd number of positions
        dict(name="linear logprobs train", op="linear_logprobs", rows=2047, width=1024, vocab=50001, dtype="f16",
             scale=1.0, train=True, ignored=True),
        # the loss of a large bf16 step
        dict(name="linear logprobs train large", op="linear_logprobs", rows=8192, width=2048, vocab=65537, dtype="bf16",
             scale=1.0, train=True, ignored=True),
        # the gradients of one small encoder layer, fp32
        dict(name="clip small", op="clip_norm", layers=1, width=512, hidden=2048, vocab=0, dtype="f32", norms="f32",
             max_norm=1.0),
        # those of eight layers and their embedding, bf16 matrices and fp32 norm weights
        dict(name="clip large", op="clip_norm", layers=8, width=2048, hidden=8192, vocab=65537, dtype="bf16",
             norms="f32", max_norm=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("embed", "feed_forward", "linear_logprobs", "clip_norm"))
    if op == "embed":
        dtype = rng.choice(("f32", "bf16", "f16"))
        vocab, width = _log_int(rng, 100, 131072), rng.choice((64, 256, 500, 512, 1001, 1024, 2048, 4096))
        while vocab * width > 131072 * 2048 // 2:
            vocab //= 2
        most = 131072 * 2048 // (width * (2 if dtype == "f32" else 1))
        return dict(op=op, rows=_log_int(rng, 1, min(most, 262144)), vocab=vocab, width=width, dtype=dtype,
                    grad=rng.choice(("f32", dtype)), scale=rng.choice((1.0, 22.625, 0.125)), skew=rng.random() < 0.6,
                    train=rng.random() < 0.75)
    if op == "feed_forward":
        width, hidden = _log_int(rng, 64, 4096), _log_int(rng, 64, 16384)
        if rng.random() < 0.6:
            width, hidden = (width + 63) // 64 * 64, (hidden + 63) // 64 * 64
        train = rng.random() < 0.6
        most = 16384 * 2048 * 8192 // (width * hidden)
        rows = rng.randint(1, 16) if not train and rng.random() < 0.5 else _log_int(rng, 1, max(2, min(most, 32768)))
        return dict(op=op, rows=rows, width=width, hidden=hidden, dtype=rng.choice(("bf16", "f16")),
                    act=rng.choice(("silu", "gelu", "gelu_tanh", "relu")), train=train)
    if op == "linear_logprobs":
        width, vocab = _log_int(rng, 64, 4096), _log_int(rng, 1000, 131072)
        if rng.random() < 0.6:
            width = (width + 63) // 64 * 64
        most = min(8192 * 2048 * 65537 // (width * vocab), 8192 * 65537 // vocab)
        return dict(op=op, rows=_log_int(rng, 1, max(2, min(most, 16384))), width=width, vocab=vocab,
                    dtype=rng.choice(("bf16", "f16")), scale=rng.choice((1.0, 0.7, 1.25)), train=rng.random() < 0.7,
                    ignored=rng.random() < 0.5)
    dtype = rng.choice(("f32", "bf16", "f16"))
    return dict(op=op, layers=_log_int(rng, 1, 4 if dtype == "f32" else 8),
                width=rng.choice((64, 200, 512, 1001, 1024, 2048)), hidden=_log_int(rng, 64, 8192),
                vocab=rng.choice((0, 1000, 20000, 32000)), dtype=dtype, norms=rng.choice(("f32", "bf16")),
                max_norm=rng.choice((1.0, 0.1, 1e6)))


# ------------------------------------------------------------------ inputs

def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return torch.empty(shape, device="cuda").normal_(mean, std, generator=gen).to(DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return dict(globals()["_prepare_" + case["op"]](case, gen), case=case)


def _prepare_embed(c, gen):
    rows, vocab, width = c["rows"], c["vocab"], c["width"]
    u = torch.rand((rows,), device="cuda", generator=gen, dtype=torch.float64)
    if c["skew"]:  # the r-th most frequent token about as often as 1 / r, in no order of their numbers
        tokens = (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(max=vocab - 1)
        tokens = torch.randperm(vocab, device="cuda", generator=gen)[tokens]
    else:
        tokens = (u * vocab).long().clamp(max=vocab - 1)
    if rows > 16:
        tokens[::17] = -1  # padding
    return dict(tokens=tokens, table=_normal(gen, (vocab, width), c["dtype"], 0.5),
                dy=_normal(gen, (rows, width), c["dtype"], 0.1) if c["train"] else None)


def _prepare_feed_forward(c, gen):
    rows, width, hidden, dt = c["rows"], c["width"], c["hidden"], c["dtype"]
    return dict(x=_normal(gen, (rows, width), dt), gate=_normal(gen, (hidden, width), dt, width ** -0.5),
                up=_normal(gen, (hidden, width), dt, width ** -0.5),
                down=_normal(gen, (width, hidden), dt, hidden ** -0.5),
                dy=_normal(gen, (rows, width), dt, 0.3) if c["train"] else None)


def _prepare_linear_logprobs(c, gen):
    rows, width, vocab, dt = c["rows"], c["width"], c["vocab"], c["dtype"]
    weight = _normal(gen, (vocab, width), dt, 2.5 * width ** -0.5)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    # the model has learnt something: hidden states lean towards their tokens, some more, some less
    lean = torch.empty((rows, 1), device="cuda").normal_(1.0, 0.4, generator=gen)
    x = torch.empty((rows, width), device="cuda").normal_(0.0, 1.0, generator=gen) + lean * weight[tokens].float()
    if c["ignored"] and rows > 16:
        tokens[::16] = -1  # positions without a target
    return dict(x=x.to(DTYPES[dt]), weight=weight, tokens=tokens,
                g_logp=torch.empty((rows,), device="cuda").normal_(-1.0, 0.3, generator=gen),
                g_lse=torch.empty((rows,), device="cuda").normal_(0.01, 0.002, generator=gen))


def _prepare_clip_norm(c, gen):
    w, h = c["width"], c["hidden"]
    layer = [((3 * w, w), "dtype"), ((w, w), "dtype"), ((h, w), "dtype"), ((w, h), "dtype"), ((w,), "norms"),
             ((w,), "norms"), ((h,), "norms")]
    shapes = layer * c["layers"] + ([((c["vocab"], w), "dtype")] if c["vocab"] else [])
    grads = [_normal(gen, s, c[t], 0.01) for s, t in shapes]
    # what the optimiser reads: the gradients themselves stay as the backward pass left them
    return dict(grads=grads, out=[torch.empty_like(g) for g in grads])


# ------------------------------------------------------------------ one pass

def run(state):
    c = state["case"]
    return globals()[("_own_" if own else "_plain_") + c["op"]](c, state)


def _own_embed(c, s):
    from ad_b200 import ops
    y = ops.embed(s["tokens"], s["table"], scale=c["scale"])
    if not c["train"]:
        return y
    out = None if c["grad"] == c["dtype"] else torch.empty_like(s["table"], dtype=DTYPES[c["grad"]])
    return y, ops.embed_grad(s["dy"], s["tokens"], c["vocab"], scale=c["scale"], out=out)


def _own_feed_forward(c, s):
    from ad_b200 import ops
    r = ops.feed_forward(s["x"], s["gate"], s["up"], s["down"], act=c["act"], keep=c["train"])
    if not c["train"]:
        return r.y
    g = ops.feed_forward_grad(s["dy"], s["x"], s["gate"], s["up"], s["down"], r.gate, r.up, act=c["act"])
    return r.y, g.x, g.w_gate, g.w_up, g.w_down


def _own_linear_logprobs(c, s):
    from ad_b200 import ops
    r = ops.linear_logprobs(s["x"], s["weight"], s["tokens"], scale=c["scale"])
    if not c["train"]:
        return r.logp, r.lse
    g = ops.linear_logprobs_grad(s["x"], s["weight"], s["tokens"], r.stats, s["g_logp"], s["g_lse"], scale=c["scale"])
    return r.logp, r.lse, g.x, g.weight


def _own_clip_norm(c, s):
    from ad_b200 import ops
    return [ops.clip_norm(s["grads"], c["max_norm"], out=s["out"])] + s["out"]


def _plain_embed(c, s):
    table, tokens = s["table"], s["tokens"]
    has = tokens >= 0
    y = torch.where(has[:, None], table[tokens.clamp(min=0)].float() * c["scale"], 0.0).to(table.dtype)
    if not c["train"]:
        return y
    # rows without a token go to a row behind the table
    grad = torch.zeros((c["vocab"] + 1, c["width"]), device="cuda")
    grad.index_add_(0, torch.where(has, tokens, c["vocab"]), s["dy"].float())
    return y, (grad[:-1] * c["scale"]).to(DTYPES[c["grad"]])


def _act(z, act):
    """The activation and its slope."""
    if act == "relu":
        return z.clamp(min=0.0), (z > 0).to(z.dtype)
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    k = (2 / math.pi) ** 0.5
    t = torch.tanh(k * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


def _plain_feed_forward(c, s):
    dt = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "gate", "up", "down"))
    g, u = x @ wg.T, x @ wu.T
    a, slope = _act(g, c["act"])
    h = a * u
    y = (h @ wd.T).to(dt)
    if not c["train"]:
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    du, dg = dh * a, dh * u * slope
    return y, (dg @ wg + du @ wu).to(dt), (dg.T @ x).to(dt), (du.T @ x).to(dt), (dy.T @ h).to(dt)


def _plain_linear_logprobs(c, s):
    x, w, tokens = s["x"].float(), s["weight"].float(), s["tokens"]
    z = x @ w.T
    z *= c["scale"]
    top = z.amax(-1, keepdim=True)
    has, at = tokens >= 0, tokens.clamp(min=0)[:, None]
    target = z.gather(1, at) - top
    p = z.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    logp = torch.where(has, (target - torch.log(total))[:, 0], 0.0)
    lse = (top + torch.log(total))[:, 0]
    if not c["train"]:
        return logp, lse
    g = torch.where(has, s["g_logp"], 0.0)[:, None]
    d = p.mul_((s["g_lse"][:, None] - g) / total)
    d.scatter_add_(1, at, g)
    d *= c["scale"]
    return logp, lse, (d @ w).to(s["x"].dtype), (d.T @ x).to(s["weight"].dtype)


def _plain_clip_norm(c, s):
    norm = torch.stack([g.float().square().sum().double() for g in s["grads"]]).sum().sqrt()
    factor = (c["max_norm"] / norm).clamp(max=1.0).float()
    return [norm.float()[None]] + [(g.float() * factor).to(g.dtype) for g in s["grads"]]


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    if case["op"] == "embed" and case["rows"] * case["width"] > 131072 * 2048:
        return None
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"]](case, s)


def _exact_embed(c, s):
    tokens = s["tokens"]
    rows = torch.nonzero(tokens >= 0)[:, 0]
    y = torch.zeros((c["rows"], c["width"]), dtype=torch.float64, device="cuda")
    y[rows] = c["scale"] * s["table"].double().index_select(0, tokens[rows])
    if not c["train"]:
        return y
    # occurrences side by side: sums over runs are differences of running sums, a slice of columns at a time
    order = rows[torch.sort(tokens[rows], stable=True).indices]
    ids, counts = torch.unique_consecutive(tokens[order], return_counts=True)
    ends = counts.cumsum(0)
    grad = torch.zeros((c["vocab"], c["width"]), dtype=torch.float64, device="cuda")
    for col in range(0, c["width"], 256):
        run = s["dy"][:, col:col + 256].double()[order].cumsum(0)
        total = run[ends - 1]
        total[1:] -= run[ends[:-1] - 1]
        grad[ids, col:col + 256] = c["scale"] * total
    return y, grad


def _exact_feed_forward(c, s):
    x, wg, wu, wd = (s[k].double() for k in ("x", "gate", "up", "down"))
    dy = s["dy"].double() if c["train"] else None
    y, dx, grads = [], [], [0.0, 0.0, 0.0]
    for r in range(0, c["rows"], 4096):
        xr = x[r:r + 4096]
        z, u = (torch.einsum("td,fd->tf", xr, w) for w in (wg, wu))
        if c["act"] == "silu":
            a = z / (1.0 + torch.exp(-z))
            slope = (1.0 + torch.exp(-z) * (1.0 + z)) / (1.0 + torch.exp(-z)) ** 2
        elif c["act"] == "relu":
            a, slope = torch.maximum(z, torch.zeros_like(z)), torch.heaviside(z, torch.zeros_like(z))
        elif c["act"] == "gelu":
            cdf = torch.special.ndtr(z)
            a, slope = z * cdf, cdf + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
        else:  # z times the logistic function of twice the argument of tanh
            k = math.sqrt(8 / math.pi)
            q = 1.0 / (1.0 + torch.exp(-k * (z + 0.044715 * z ** 3)))
            a, slope = z * q, q + z * q * (1.0 - q) * k * (1.0 + 0.134145 * z ** 2)
        y.append(torch.einsum("tf,df->td", a * u, wd))
        if c["train"]:
            dyr = dy[r:r + 4096]
            dh = torch.einsum("td,df->tf", dyr, wd)
            dz, du = dh * u * slope, dh * a
            dx.append(torch.einsum("tf,fd->td", dz, wg) + torch.einsum("tf,fd->td", du, wu))
            for i, (p, q) in enumerate(((dz, xr), (du, xr), (dyr, a * u))):
                grads[i] = grads[i] + torch.einsum("ti,tj->ij", p, q)
    if not c["train"]:
        return torch.cat(y)
    return (torch.cat(y), torch.cat(dx), *grads)


def _exact_linear_logprobs(c, s):
    x, w, tokens = s["x"].double(), s["weight"].double(), s["tokens"]
    logp, lse, dx, dw = [], [], [], 0.0
    for r in range(0, c["rows"], 2048):
        xr, t = x[r:r + 2048], tokens[r:r + 2048]
        z = c["scale"] * torch.einsum("td,vd->tv", xr, w)
        total = torch.logsumexp(z, -1)
        index, has = torch.arange(len(t), device=t.device), (t >= 0).double()
        lse.append(total)
        logp.append(has * (z[index, t.clamp(min=0)] - total))
        if c["train"]:
            g, e = s["g_logp"][r:r + 2048].double() * has, s["g_lse"][r:r + 2048].double()
            d = torch.softmax(z, -1) * (e - g)[:, None]
            d[index, t.clamp(min=0)] += g
            d = d * c["scale"]
            dx.append(torch.einsum("tv,vd->td", d, w))
            dw = dw + torch.einsum("tv,td->vd", d, xr)
    if not c["train"]:
        return torch.cat(logp), torch.cat(lse)
    return torch.cat(logp), torch.cat(lse), torch.cat(dx), dw


def _exact_clip_norm(c, s):
    parts = [torch.linalg.vector_norm(g.double()) for g in s["grads"]]
    norm = torch.linalg.vector_norm(torch.stack(parts))
    return [norm[None]] + [g.double() * min(1.0, c["max_norm"] / float(norm)) for g in s["grads"]]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    return globals()["_work_" + case["op"]](case)


def _work_embed(c):
    values, s = c["rows"] * c["width"], SIZE[c["dtype"]]
    # rows of the table that come up at all
    r = np.arange(1, c["vocab"] + 1)
    chance = np.log1p(1 / r) / math.log(c["vocab"] + 1) if c["skew"] else np.full(c["vocab"], 1 / c["vocab"])
    seen = int((1 - (1 - np.minimum(chance, 1.0)) ** c["rows"]).sum())
    size = 8 * c["rows"] + s * (values + seen * c["width"])
    if c["train"]:  # the tokens once more, the results' gradient, and the table's
        size += 8 * c["rows"] + s * values + SIZE[c["grad"]] * c["vocab"] * c["width"]
    return {"bytes": size, "flops": values * (2 if c["train"] else 1)}


def _work_feed_forward(c):
    x, w, f = c["rows"] * c["width"], c["width"] * c["hidden"], c["rows"] * c["hidden"]
    size, flops = 2 * (2 * x + 3 * w), 6 * x * c["hidden"] + 8 * f
    if c["train"]:  # x, dy and the weights -> dx and the weights' gradients; what lies between is kept or made again
        size += 2 * (3 * x + 6 * w + 4 * f)
        flops += 12 * x * c["hidden"] + 16 * f
    return {"bytes": size, "flops": flops}


def _work_linear_logprobs(c):
    x, w = c["rows"] * c["width"], c["vocab"] * c["width"]
    size, flops = 2 * (x + w) + 16 * c["rows"], 2 * x * c["vocab"] + 4 * c["rows"] * c["vocab"]
    if c["train"]:  # both once more, and their gradients; the logits have to be made twice, or kept
        size += 4 * (x + w) + 24 * c["rows"]
        flops += 4 * x * c["vocab"] + 4 * c["rows"] * c["vocab"]
    return {"bytes": size, "flops": flops}


def _work_clip_norm(c):
    w, h = c["width"], c["hidden"]
    matrices, vectors = c["layers"] * (4 * w * w + 2 * h * w) + c["vocab"] * w, c["layers"] * (2 * w + h)
    return {"bytes": 2 * (matrices * SIZE[c["dtype"]] + vectors * SIZE[c["norms"]]), "flops": 3 * (matrices + vectors)}

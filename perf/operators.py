"""What the language-model operators of ``ad_b200.ops`` are measured on.

Four operators that stand between the matrix products of a language model's
training step:

* ``rotary``         rotary positions of queries and keys (and, inverted, of their gradients)
* ``block_norm``     a norm after a block, its gate, the scaled residual sum and the norm before
                     the next block, with the gradients of all of them
* ``token_logprobs`` log probabilities of given tokens, entropy and the best alternatives of each
                     row of logits, with the gradient
* ``orthogonalize``  Newton-Schulz orthogonalisation of a matrix update

Where ``own`` is false ``run`` computes them from elementary torch operations in 32 bits, rounded
once at the end; where it is true it calls the framework.  ``exact`` computes them in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# One step of the Newton-Schulz iteration is x -> a x + b x^3 + c x^5 on every singular value.
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one new token for each of 32 sequences of different lengths: launch latency counts
        dict(name="rotary decode", op="rotary", batch=32, tokens=1, q_heads=8, k_heads=8, dim=64,
             rotary=64, layout="half", dtype="bf16", inverse=False, heads_first=False, table=4096),
        # queries and keys of an fp32 training step, heads outermost in memory as the per-head
        # projections leave them; an odd number of tokens
        dict(name="rotary train fp32", op="rotary", batch=32, tokens=509, q_heads=16, k_heads=16, dim=64,
             rotary=64, layout="half", dtype="f32", inverse=False, heads_first=True, table=512),
        # gradients (inverse rotation) of long sequences, shared key heads, half of each head
        # rotated in neighbouring pairs
        dict(name="rotary long gradient", op="rotary", batch=4, tokens=16384, q_heads=32, k_heads=8, dim=128,
             rotary=64, layout="interleaved", dtype="bf16", inverse=True, heads_first=False, table=16384),
        # a handful of tokens being generated: forward alone
        dict(name="norm decode", op="block_norm", rows=8, width=512, dtype="bf16", weights="f32", kind="rms",
             gate="row", sigmoid=True, scale=1.0, train=False),
        # fp32 training step of 32 sequences of 512, LayerNorm, a gate for each sequence
        dict(name="norm train fp32", op="block_norm", rows=16384, width=1024, dtype="f32", weights="f32",
             kind="layer", gate="group", groups=32, sigmoid=False, scale=0.5, train=True),
        # a large bf16 training step, a sigmoid gate for each value, weights in bf16 too
        dict(name="norm train large", op="block_norm", rows=65535, width=2048, dtype="bf16", weights="bf16",
             kind="rms", gate="row", sigmoid=True, scale=1.0, train=True),
        # sampling: four rows over a large vocabulary with the twenty best alternatives
        dict(name="logprobs decode", op="token_logprobs", rows=4, vocab=131072, dtype="bf16", top=20,
             scale=1.25, train=False, masked=True),
        # scoring and training in fp32, an odd vocabulary, four alternatives for the log
        dict(name="logprobs train fp32", op="token_logprobs", rows=2048, vocab=50001, dtype="f32", top=4,
             scale=1.0, train=True, masked=False),
        # the loss of a large bf16 step; the odd vocabulary leaves rows unaligned
        dict(name="logprobs train large", op="token_logprobs", rows=8191, vocab=65537, dtype="bf16", top=0,
             scale=1.0, train=True, masked=True),
        # the update of one attention projection
        dict(name="orthogonalize one", op="orthogonalize", count=1, rows=512, cols=512, dtype="f32"),
        # twelve layers' up-projections at once
        dict(name="orthogonalize stack", op="orthogonalize", count=12, rows=4096, cols=1024, dtype="f32"),
        # three tall odd-sized matrices whose update is held in bf16
        dict(name="orthogonalize odd", op="orthogonalize", count=3, rows=2049, cols=1001, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "block_norm", "token_logprobs", "orthogonalize"))
    if op == "rotary":
        dim = rng.choice((32, 64, 80, 96, 128, 256))
        k_heads = rng.choice((1, 2, 4, 8, 16))
        q_heads = k_heads * rng.choice((1, 2, 4))
        batch = _log_int(rng, 1, 64)
        # at most as many values as the largest listed case has
        most = 4 * 16384 * 40 * 128 // (batch * (q_heads + k_heads) * dim)
        tokens = 1 if rng.random() < 0.25 else _log_int(rng, 1, max(2, min(16384, most)))
        rotary = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        dtype = rng.choice(("f32", "bf16", "f16"))
        if dtype == "f32":
            tokens = max(1, tokens // 2)
        return dict(op=op, batch=batch, tokens=tokens, q_heads=q_heads, k_heads=k_heads, dim=dim, rotary=rotary,
                    layout=rng.choice(("half", "interleaved")), dtype=dtype, inverse=rng.random() < 0.4,
                    heads_first=rng.random() < 0.4, table=max(tokens, _log_int(rng, 64, 32768)))
    if op == "block_norm":
        dtype = rng.choice(("f32", "bf16", "f16"))
        width = rng.choice((256, 512, 1000, 1023, 1024, 2048, 4096, 5000))
        gate = rng.choice(("none", "row", "group", "one"))
        groups = rng.choice((1, 3, 8, 32)) if gate == "group" else 1
        per = max(1, _log_int(rng, 1, 65535 * 2048 // (width * (2 if dtype == "f32" else 1))) // groups)
        return dict(op=op, rows=per * groups, width=width, dtype=dtype, weights=rng.choice(("f32", dtype)),
                    kind=rng.choice(("rms", "layer")), gate=gate, groups=groups, sigmoid=rng.random() < 0.5,
                    scale=rng.choice((1.0, 0.5)), train=rng.random() < 0.7)
    if op == "token_logprobs":
        dtype = rng.choice(("f32", "bf16", "f16"))
        vocab = _log_int(rng, 1000, 131072)
        top = rng.choice((0, 0, 1, 5, 20))
        # the alternatives' plain form sorts keys of 64 bits: fewer rows where they are asked for
        most = 8191 * 65537 // (vocab * (2 if dtype == "f32" else 1) * (3 if top else 1))
        return dict(op=op, rows=_log_int(rng, 1, max(2, most)), vocab=vocab, dtype=dtype, top=top,
                    scale=rng.choice((1.0, 0.7, 1.25)), train=rng.random() < 0.6, masked=rng.random() < 0.5)
    rows, cols = _log_int(rng, 64, 4096), _log_int(rng, 64, 4096)
    lo, hi = min(rows, cols), max(rows, cols)
    most = int(12 * 1024 * 1024 * 4096 * 3.25 // (lo * lo * (3 * hi + lo)))
    count = _log_int(rng, 1, max(1, min(16, most)))
    while lo * lo * (3 * hi + lo) * count > 12 * 1024 * 1024 * (3 * 4096 + 1024):
        rows, cols = max(1, rows * 3 // 4), max(1, cols * 3 // 4)
        lo, hi = min(rows, cols), max(rows, cols)
    return dict(op=op, count=count, rows=rows, cols=cols, dtype=rng.choice(("f32", "bf16")))


# ------------------------------------------------------------------ inputs

def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return torch.empty(shape, device="cuda").normal_(mean, std, generator=gen).to(DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return dict(globals()["_prepare_" + case["op"]](case, gen), case=case)


def _prepare_rotary(c, gen):
    b, t, d, half = c["batch"], c["tokens"], c["dim"], c["rotary"] // 2
    # the table is the plan that a program keeps: cosines and sines of position * frequency
    angle = torch.arange(c["table"], device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        10000.0, torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 / c["rotary"]))
    first = torch.randint(0, c["table"] - t + 1, (b, 1), device="cuda", generator=gen)
    s = dict(cos=angle.cos().float(), sin=angle.sin().float(),
             positions=first + torch.arange(t, device="cuda"))
    for name, heads in (("q", c["q_heads"]), ("k", c["k_heads"])):
        shape = (b, heads, t, d) if c["heads_first"] else (b, t, heads, d)
        x = _normal(gen, shape, c["dtype"])
        s[name] = x.transpose(1, 2) if c["heads_first"] else x
    return s


def _prepare_block_norm(c, gen):
    rows, width, dt, wt = c["rows"], c["width"], c["dtype"], c["weights"]
    layer = c["kind"] == "layer"
    gate = {"none": None, "row": (rows, width), "group": (c.get("groups", 1), width), "one": (1, width)}[c["gate"]]
    return dict(
        x=_normal(gen, (rows, width), dt, 2.0), z=_normal(gen, (rows, width), dt, 0.7, 0.1),
        gate=None if gate is None else _normal(gen, gate, dt, 1.0, 0.5),
        after=_normal(gen, (width,), wt, 0.2, 1.0), before=_normal(gen, (width,), wt, 0.2, 1.0),
        after_bias=_normal(gen, (width,), wt, 0.1) if layer else None,
        before_bias=_normal(gen, (width,), wt, 0.1) if layer else None,
        dh=_normal(gen, (rows, width), dt, 0.1) if c["train"] else None,
        dy=_normal(gen, (rows, width), dt, 0.1) if c["train"] else None)


def _prepare_token_logprobs(c, gen):
    rows, vocab = c["rows"], c["vocab"]
    logits = torch.empty((rows, vocab), device="cuda", dtype=DTYPES[c["dtype"]])
    at = max(1, (1 << 28) // vocab)
    for r in range(0, rows, at):  # a common part and each row's own, with a few tokens far ahead
        n = min(at, rows - r)
        x = torch.empty((n, vocab), device="cuda").normal_(0.0, 2.5, generator=gen)
        peak = torch.randint(0, vocab, (n, 8), device="cuda", generator=gen)
        x.scatter_add_(1, peak, torch.empty((n, 8), device="cuda").normal_(8.0, 3.0, generator=gen))
        logits[r:r + n] = x
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    if c["masked"]:  # tokens that a grammar or the padding of the vocabulary rules out
        low = max(1, vocab - vocab // 16)
        logits[:, low:] = -math.inf
        tokens %= low
        if rows > 16:
            tokens[::16] = -1  # positions without a target
    return dict(logits=logits, tokens=tokens,
                g_logp=torch.empty((rows,), device="cuda").normal_(-1.0, 0.3, generator=gen),
                g_entropy=torch.empty((rows,), device="cuda").normal_(0.01, 0.002, generator=gen))


def _prepare_orthogonalize(c, gen):
    # a momentum: a decaying spectrum of shared directions and noise over it
    n, rows, cols = c["count"], c["rows"], c["cols"]
    rank = max(1, min(rows, cols) // 8)
    left = torch.empty((n, rows, rank), device="cuda").normal_(generator=gen)
    right = torch.empty((n, rank, cols), device="cuda").normal_(generator=gen)
    left /= torch.arange(1, rank + 1, device="cuda").float().sqrt()
    g = torch.empty((n, rows, cols), device="cuda").normal_(0.0, 0.5, generator=gen)
    return dict(g=(1e-3 * (g + torch.bmm(left, right))).to(DTYPES[c["dtype"]]))


# ------------------------------------------------------------------ one pass

def run(state):
    c = state["case"]
    return globals()[("_own_" if own else "_plain_") + c["op"]](c, state)


def _own_rotary(c, s):
    from ad_b200 import ops
    return ops.rotary(s["q"], s["k"], s["cos"], s["sin"], s["positions"], layout=c["layout"], inverse=c["inverse"])


def _own_block_norm(c, s):
    from ad_b200 import ops
    opts = dict(gate=s["gate"], after_bias=s["after_bias"], before_bias=s["before_bias"], kind=c["kind"],
                gate_sigmoid=c["sigmoid"], residual_scale=c["scale"], eps=1e-5)
    h, y, stats = ops.block_norm(s["x"], s["z"], s["after"], s["before"], **opts)
    if not c["train"]:
        return h, y
    g = ops.block_norm_grad(s["dh"], s["dy"], s["x"], s["z"], s["after"], s["before"], stats, **opts)
    return [h, y] + [v for v in g if v is not None]


def _own_token_logprobs(c, s):
    from ad_b200 import ops
    r = ops.token_logprobs(s["logits"], s["tokens"], top=c["top"], scale=c["scale"])
    out = [r.logp, r.entropy] + ([r.top_logp, r.top_index] if c["top"] else [])
    if c["train"]:
        out.append(ops.token_logprobs_grad(s["logits"], s["tokens"], r.stats, s["g_logp"], s["g_entropy"],
                                           scale=c["scale"]))
    return out


def _own_orthogonalize(c, s):
    from ad_b200 import ops
    return ops.orthogonalize(s["g"], steps=NS_STEPS, coefficients=NS_COEFFICIENTS, eps=NS_EPS)


def _rotate(x, cos, sin, rotary, layout):
    """x [batch, tokens, heads, dim]; cos, sin [batch, tokens, 1, rotary / 2]."""
    half = rotary // 2
    y = x[..., :rotary]
    if layout == "half":
        u, v = y[..., :half], y[..., half:]
    else:
        u, v = y[..., 0::2], y[..., 1::2]
    u, v = u * cos - v * sin, v * cos + u * sin
    y = torch.cat((u, v), -1) if layout == "half" else torch.stack((u, v), -1).flatten(-2)
    return torch.cat((y, x[..., rotary:]), -1)


def _plain_rotary(c, s):
    cos, sin = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
    if c["inverse"]:
        sin = -sin
    return tuple(_rotate(s[n].float(), cos, sin, c["rotary"], c["layout"]).to(s[n].dtype) for n in ("q", "k"))


def _normed(v, weight, bias, kind):
    """The norm of each row: (result, normalised row, reciprocal of the deviation)."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5)
    n = v * r
    y = n * weight
    return (y if bias is None else y + bias), n, r


def _norm_grad(dn, n, r, kind):
    """The gradient of the norm's input from that of the normalised row."""
    d = dn - n * (dn * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - dn.mean(-1, keepdim=True)
    return d * r


def _plain_block_norm(c, s):
    f = {k: None if v is None else v.float() for k, v in s.items() if k != "case"}
    return [t.to(d) for t, d in _block_norm(c, s, f)]


def _block_norm(c, s, f):
    """(value, type) of each output, in the precision of `f`."""
    kind, dt, wt = c["kind"], DTYPES[c["dtype"]], DTYPES[c["weights"]]
    rows, width = f["x"].shape
    u, nz, rz = _normed(f["z"], f["after"], f["after_bias"], kind)
    gate = per = act = None
    if f["gate"] is not None:
        gate, per = f["gate"], rows // f["gate"].shape[0]
        act = torch.sigmoid(gate) if c["sigmoid"] else gate
        wide = act if per == 1 else act.repeat_interleave(per, 0)
    h = f["x"] * c["scale"] + (u if gate is None else wide * u)
    y, nh, rh = _normed(h, f["before"], f["before_bias"], kind)
    out = [(h, dt), (y, dt)]
    if not c["train"]:
        return out
    dy = f["dy"]
    dh = f["dh"] + _norm_grad(dy * f["before"], nh, rh, kind)
    du = dh if gate is None else dh * wide
    out += [(dh * c["scale"], dt), (_norm_grad(du * f["after"], nz, rz, kind), dt)]
    if gate is not None:
        dg = (dh * u).reshape(-1, per, width).sum(1)
        out.append((dg * act * (1 - act) if c["sigmoid"] else dg, dt))
    out += [((du * nz).sum(0), wt), ((dy * nh).sum(0), wt)]
    if kind == "layer":
        out += [(du.sum(0), wt), (dy.sum(0), wt)]
    return out


def _plain_token_logprobs(c, s):
    x, tokens = s["logits"].float() * c["scale"], s["tokens"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lp = (x - top) - torch.log(total)
    p = e / total
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    has = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    out = [torch.where(has, lp.gather(1, at)[:, 0], 0.0), entropy]
    if c["top"]:
        # keys that order as the logits do, the lower index first among equal ones
        bits = (s["logits"].float() + 0.0).view(torch.int32)
        bits = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() << 32
        bits += c["vocab"] - 1 - torch.arange(c["vocab"], device=bits.device)
        index = c["vocab"] - 1 - (torch.topk(bits, c["top"]).values & 0xFFFFFFFF)
        out += [lp.gather(1, index), index]
    if c["train"]:
        g = torch.where(has, s["g_logp"], 0.0)[:, None]
        d = torch.where(p > 0, -p * (g + s["g_entropy"][:, None] * (lp + entropy[:, None])), 0.0)
        d.scatter_add_(1, at, g)
        out.append((d * c["scale"]).to(s["logits"].dtype))
    return out


def _plain_orthogonalize(c, s):
    a, b, cc = NS_COEFFICIENTS
    x = s["g"].float()
    tall = c["rows"] > c["cols"]
    if tall:
        x = x.mT
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    for _ in range(NS_STEPS):
        p = x @ x.mT
        x = a * x + (b * p + cc * (p @ p)) @ x
    return (x.mT if tall else x).contiguous().to(torch.bfloat16)


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"]](case, s)


def _exact_rotary(c, s):
    # the pair (u, v) as a complex number times cos + i sin
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].reshape(-1)]
    turn = (turn.conj() if c["inverse"] else turn)[:, None]
    out = []
    for name in ("q", "k"):
        x = s[name]
        y = x.double().reshape(-1, x.shape[2], x.shape[3])
        half = c["rotary"] // 2
        if c["layout"] == "half":
            u, v = slice(0, half), slice(half, 2 * half)
        else:
            u, v = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        w = torch.complex(y[..., u].contiguous(), y[..., v].contiguous()) * turn
        y[..., u], y[..., v] = w.real, w.imag
        out.append(y.reshape(x.shape))
        del y, w
    return tuple(out)


def _exact_block_norm(c, s):
    rows, width = s["x"].shape
    layer, sigmoid, alpha, eps = c["kind"] == "layer", c["sigmoid"], c["scale"], 1e-5
    groups = s["gate"].shape[0] if s["gate"] is not None else 1
    per = rows // groups
    w = {k: None if s[k] is None else s[k].double() for k in ("after", "before", "after_bias", "before_bias")}
    zero = torch.zeros(width, dtype=torch.float64, device="cuda")
    after_bias = zero if w["after_bias"] is None else w["after_bias"]
    before_bias = zero if w["before_bias"] is None else w["before_bias"]
    parts = {k: [] for k in ("h", "y", "dx", "dz", "dg")}
    sums = [zero.clone() for _ in range(4)]
    dgate = torch.zeros((groups, width), dtype=torch.float64, device="cuda")

    def moments(v):
        mean = v.sum(1, keepdim=True) / width if layer else 0.0 * v[:, :1]
        var = ((v - mean) ** 2).sum(1, keepdim=True) / width
        return mean, (var + eps) ** -0.5

    def through(d, v, mean, r):  # d loss / d v of (v - mean) r, from the loss's gradient d of that
        centred = v - mean
        dr = (d * centred).sum(1, keepdim=True)
        dv = d * r - centred * (r ** 3 * dr / width)
        return dv - dv.sum(1, keepdim=True) / width if layer else dv

    step = per if 1 < per <= 8192 else 8192 if per == 1 else per
    for r0 in range(0, rows, step):
        r1 = min(rows, r0 + step)
        x, z = s["x"][r0:r1].double(), s["z"][r0:r1].double()
        mz, qz = moments(z)
        nz = (z - mz) * qz
        u = nz * w["after"] + after_bias
        if s["gate"] is None:
            a = slope = torch.ones((1, width), dtype=torch.float64, device="cuda")
        else:
            g = s["gate"][r0:r1] if per == 1 else s["gate"][r0 // per:r0 // per + 1]
            a = 1.0 / (1.0 + torch.exp(-g.double())) if sigmoid else g.double()
            slope = a * (1.0 - a) if sigmoid else torch.ones_like(a)
        h = alpha * x + a * u
        mh, qh = moments(h)
        nh = (h - mh) * qh
        parts["h"].append(h)
        parts["y"].append(nh * w["before"] + before_bias)
        if c["train"]:
            dy = s["dy"][r0:r1].double()
            total = s["dh"][r0:r1].double() + through(dy * w["before"], h, mh, qh)
            du = total * a
            parts["dx"].append(alpha * total)
            parts["dz"].append(through(du * w["after"], z, mz, qz))
            if s["gate"] is not None:
                dg = total * u * slope
                if per == 1:
                    parts["dg"].append(dg)
                else:
                    dgate[r0 // per] += dg.sum(0)
            for k, v in enumerate((du * nz, dy * nh, du, dy)):
                sums[k] += v.sum(0)
        # what is compared is held in 64 bits; keep no more of it than that
    out = [torch.cat(parts["h"]), torch.cat(parts["y"])]
    if c["train"]:
        out += [torch.cat(parts["dx"]), torch.cat(parts["dz"])]
        if s["gate"] is not None:
            out.append(torch.cat(parts["dg"]) if per == 1 else dgate)
        out += sums[:4 if layer else 2]
    return out


def _exact_token_logprobs(c, s):
    rows, vocab = c["rows"], c["vocab"]
    step = max(1, (1 << 27) // vocab)
    logp, entropy, best, grad = [], [], [], []
    for r in range(0, rows, step):
        x = c["scale"] * s["logits"][r:r + step].double()
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        h = -(p * lp.masked_fill(p == 0, 0.0)).sum(-1)
        t = s["tokens"][r:r + step]
        hot = torch.zeros_like(p)
        hot[(t >= 0).nonzero()[:, 0], t[t >= 0]] = 1.0
        logp.append(torch.where(t >= 0, lp[torch.arange(len(t), device=t.device), t.clamp(min=0)], 0.0))
        entropy.append(h)
        if c["top"]:
            best.append(torch.sort(lp, -1, descending=True).values[:, :c["top"]])
        if c["train"]:
            g = s["g_logp"][r:r + step, None].double() * (t >= 0)[:, None]
            e = s["g_entropy"][r:r + step, None].double()
            d = g * (hot - p) - e * p * (lp.masked_fill(p == 0, 0.0) + h[:, None])
            grad.append(c["scale"] * d)
    out = [torch.cat(logp), torch.cat(entropy)]
    if c["top"]:
        out += [torch.cat(best), None]
    if c["train"]:
        out.append(torch.cat(grad))
    return out


def _exact_orthogonalize(c, s):
    a, b, cc = NS_COEFFICIENTS
    out = []
    for g in s["g"]:
        # from the side with fewer rows: the polynomial of the product of the matrix with its transpose
        x = g.double()
        x = x / (torch.linalg.matrix_norm(x) + NS_EPS)
        eye = torch.eye(min(x.shape), dtype=torch.float64, device=x.device)
        for _ in range(NS_STEPS):
            if x.shape[0] <= x.shape[1]:
                p = x @ x.T
                x = (a * eye + b * p + cc * (p @ p)) @ x
            else:
                p = x.T @ x
                x = x @ (a * eye + b * p + cc * (p @ p))
        out.append(x)
    return torch.stack(out)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    return globals()["_work_" + case["op"]](case)


def _work_rotary(c):
    rows = c["batch"] * c["tokens"]
    values = rows * (c["q_heads"] + c["k_heads"]) * c["dim"]
    turned = rows * (c["q_heads"] + c["k_heads"]) * c["rotary"]
    # inputs and outputs, positions of 8 bytes, each used row of the two tables once
    return {"bytes": 2 * values * SIZE[c["dtype"]] + 8 * rows + 4 * c["rotary"] * min(rows, c["table"]),
            "flops": 3 * turned}


def _work_block_norm(c):
    rows, width, s, w = c["rows"], c["width"], SIZE[c["dtype"]], SIZE[c["weights"]]
    gate = {"none": 0, "row": rows, "group": c.get("groups", 1), "one": 1}[c["gate"]] * width
    vectors = (4 if c["kind"] == "layer" else 2) * width
    values = rows * width
    size = s * (4 * values + gate) + w * vectors  # x, z, gate -> h, y
    flops = 14 * values
    if c["train"]:  # dh, dy beside x, z and gate once more -> dx, dz, the gate's and the weights'
        size += s * (6 * values + 2 * gate) + 2 * w * vectors
        flops += 34 * values
    return {"bytes": size, "flops": flops}


def _work_token_logprobs(c):
    values, s = c["rows"] * c["vocab"], SIZE[c["dtype"]]
    size = values * s + c["rows"] * (8 + 8 + 12 * c["top"])
    flops = 6 * values
    if c["train"]:  # the logits once more, and their gradient
        size += 2 * values * s + c["rows"] * 24
        flops += 7 * values
    return {"bytes": size, "flops": flops}


def _work_orthogonalize(c):
    lo, hi = min(c["rows"], c["cols"]), max(c["rows"], c["cols"])
    # two symmetric products of which one half is enough, and a full one, five times
    flops = c["count"] * NS_STEPS * (lo * lo * hi + lo * lo * lo + 2 * lo * lo * hi)
    return {"bytes": c["count"] * lo * hi * (SIZE[c["dtype"]] + 2), "flops": flops}

"""Embeddings, feed-forward blocks, log probabilities of a linear layer and gradient clipping against
plain 64-bit implementations (B200 only).

Bounds are derived from the arithmetic, not from runs.  E = 2^-24 is half a step of 32 bits, U[t] of the
elements' type, TINY[t] half the spacing of its smallest numbers.  The tensor cores add the products of 16
elements of K at a time to a sum in 32 bits and may truncate both those products (as they are aligned to the
largest of them) and the sum: two steps of 2^-23 of the terms' magnitude each time, `tc(k)` in all.  A
bound on what enters a product goes through it with the magnitudes of the other operand; what is rounded to
the elements' type on the way counts half a step of that."""
import math
import threading

import pytest

from .test_gpu_ops import E, U, dtype, rand, seeded

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TINY = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}
HALVES = ["bfloat16", "float16"]


@pytest.fixture(scope="module")
def ops():
    from ad_b200 import ops as o
    return o


def tc(k):
    return (k / 16 + 2) * 2.0 ** -22


def close(got, want, bound, t):
    """|got - want| <= bound and one rounding to type t; NaN and infinities in the same places."""
    got = got.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    limit = 1.05 * bound + 1.01 * U[t] * want.abs() + 1.01 * TINY[t] + 1e-300
    worst = ((got - want).abs() / limit)[fine]
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, float(worst.max())


# ------------------------------------------------------------------ embeddings

def embed64(tokens, table, scale):
    y = scale * table.double()[tokens.clamp(0, table.shape[0] - 1)]
    y[tokens < 0] = 0.0
    y[tokens >= table.shape[0]] = math.nan
    return y


def embed_grad64(dy, tokens, vocab, scale):
    """The sums, and a bound of their error in 32 bits (as many additions as terms, and a factor)."""
    dy, tokens = dy.double().reshape(-1, dy.shape[-1]), tokens.reshape(-1)
    ok = (tokens >= 0) & (tokens < vocab)
    out = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=dy.device)
    mag, count = out.clone(), torch.zeros(vocab, dtype=torch.float64, device=dy.device)
    out.index_add_(0, tokens[ok], dy[ok])
    mag.index_add_(0, tokens[ok], dy[ok].abs())
    count.index_add_(0, tokens[ok], torch.ones_like(tokens[ok], dtype=torch.float64))
    return out * scale, mag * (count[:, None] + 2) * E * abs(scale)


@pytest.mark.parametrize("t", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab,width", [(1, 1, 1), (3, 5, 2), (40, 9, 33), (33, 1000, 64), (64, 70, 256), (7, 50, 1001),
                                              (2500, 300, 130), (9, 4, 4096)])
def test_embed(ops, t, rows, vocab, width):
    gen = seeded(rows, vocab, width)
    table = rand(gen, (vocab, width), t)
    tokens = torch.randint(-1, vocab + 1, (rows,), generator=gen).cuda()
    for scale in (1.0, -3.3):
        y = ops.embed(tokens, table, scale=scale)
        close(y, embed64(tokens, table, scale), E * abs(scale) * 4, t)
    assert torch.equal(ops.embed(tokens.int(), table).nan_to_num(9.0), ops.embed(tokens, table).nan_to_num(9.0))


def test_embed_shapes_strides_and_places(ops):
    gen = seeded(3)
    store = rand(gen, (20, 40), "bfloat16")
    tokens = torch.randint(0, 20, (2, 3, 4), generator=gen).cuda()
    for table in (store, store[:, 3:36], store[1:, :8], store[::2, 8:24]):
        y = ops.embed(tokens % table.shape[0], table)
        assert y.shape == (2, 3, 4, table.shape[1]) and torch.equal(y, table[tokens % table.shape[0]])
    out = torch.full((24, 50), 7.0, device="cuda", dtype=torch.bfloat16)
    got = ops.embed(tokens.reshape(-1), store, out=out[:, 5:45])
    assert torch.equal(got, store[tokens.reshape(-1)]) and (out[:, :5] == 7).all() and (out[:, 45:] == 7).all()
    assert ops.embed(tokens[0, 0, 0], store).shape == (40,)
    assert ops.embed(tokens[:0], store).shape == (0, 3, 4, 40)


@pytest.mark.parametrize("t,o", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("rows,vocab,width", [
    (1, 1, 1), (1, 7, 64), (31, 3, 5), (32, 1, 128), (33, 1, 128), (2048, 1, 8), (2047, 50, 100), (2049, 1500, 64),
    (5000, 3, 257), (6000, 1025, 1001), (4100, 70000, 16), (8192, 9000, 40), (8193, 9000, 40), (16384, 1, 8),
    (16385, 2000000, 8), (33000, 1500, 33), (65536, 70000, 8), (65536, 1, 8), (65537, 1024, 8), (70000, 40, 32),
    (20000, 2, 2048)])
def test_embed_grad(ops, t, o, rows, vocab, width):
    gen = seeded(rows, vocab, width)
    # some tokens far more frequent than others, some outside of the vocabulary
    tokens = (vocab * torch.rand(rows, generator=gen, dtype=torch.float64) ** 3).long().clamp(max=vocab - 1)
    if rows > 2:
        tokens[::7], tokens[::11] = -1, vocab
    tokens, dy = tokens.cuda(), rand(gen, (rows, width), t)
    want, bound = embed_grad64(dy, tokens, vocab, 0.7)
    out = torch.full((vocab, width), math.nan, device="cuda", dtype=dtype(o))
    got = ops.embed_grad(dy, tokens, vocab, scale=0.7, out=out)
    assert got is out
    close(got, want, bound, o)
    again = ops.embed_grad(dy, tokens.int(), vocab, scale=0.7, out=torch.empty_like(out))
    assert torch.equal(got, again)  # whatever the order of the blocks
    base = rand(gen, (vocab, width), o)
    total = ops.embed_grad(dy, tokens, vocab, scale=0.7, out=base.clone(), accumulate=True)
    close(total, base.double() + want, bound + E * (want.abs() + base.double().abs()), o)
    absent = torch.ones(vocab, dtype=torch.bool, device="cuda")
    absent[tokens[(tokens >= 0) & (tokens < vocab)]] = False
    assert torch.equal(total[absent], base[absent])


def test_embed_grad_strides_and_nothing(ops):
    gen = seeded(11)
    store = rand(gen, (300, 90), "bfloat16")
    tokens = torch.randint(0, 40, (300,), generator=gen).cuda()
    for dy in (store[:, 1:65], store[:, 8:72], store[:1].expand(300, 90)):
        want, bound = embed_grad64(dy, tokens, 40, 1.0)
        out = torch.full((40, 100), 5.0, device="cuda")
        close(ops.embed_grad(dy, tokens, 40, out=out[:, 3:3 + dy.shape[1]]), want, bound, "float32")
        assert (out[:, :3] == 5).all() and (out[:, 3 + dy.shape[1]:] == 5).all()
    assert (ops.embed_grad(store[:0], tokens[:0], 5) == 0).all()
    assert (ops.embed_grad(store, torch.full_like(tokens, -1), 5) == 0).all()
    kept = torch.ones(5, 90, device="cuda")
    ops.embed_grad(store[:0], tokens[:0], 5, out=kept, accumulate=True)
    assert (kept == 1).all()
    inf = torch.zeros(3, 8, device="cuda")
    inf[1, 2], inf[2, 3] = math.inf, math.nan
    got = ops.embed_grad(inf, torch.tensor([0, 1, 1], device="cuda"), 3)
    assert got[1, 2] == math.inf and got[1, 3].isnan() and (got[0] == 0).all() and (got[2] == 0).all()


def test_embed_and_its_gradient_belong_together(ops):
    """<dy, embed(T)> is linear in T with the gradient's rows as its factors."""
    gen = seeded(4)
    table, dy = rand(gen, (50, 96), "float32"), rand(gen, (4, 200, 96), "float32")
    tokens = torch.randint(-2, 50, (4, 200), generator=gen).cuda()
    grad = ops.embed_grad(dy, tokens, 50, scale=0.5).double()
    step = rand(gen, (50, 96), "float32")
    change = (dy.double() * (ops.embed(tokens, table + step, scale=0.5).double() -
                             ops.embed(tokens, table, scale=0.5).double())).sum()
    want = (grad * ((table + step).double() - table.double())).sum()
    size = (dy.double().abs().sum() * 6)
    assert abs(float(change - want)) <= 8 * E * float(size)


# ------------------------------------------------------------------ feed-forward blocks

def act64(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(8 / math.pi)
    p = torch.sigmoid(k * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * k * (1 + 3 * 0.044715 * z * z)


def ffn64(x, wg, wu, wd, dy, act, t):
    """Results and bounds.  Activations are taken in 32 bits: the approximations' 1.5e-7 and a few E, of
    |z| for the value and of 2 for the slope; slopes are below 1.13 and change by at most 1.2 for 1."""
    x, wg, wu, wd = (v.double() for v in (x, wg, wu, wd))
    k = tc(x.shape[1])
    u = U[t]
    g, up = x @ wg.T, x @ wu.T
    dg, du = k * (x.abs() @ wg.abs().T), k * (x.abs() @ wu.abs().T)  # errors of g and up
    a, slope = act64(g, act)
    ea = 1.13 * dg + (3e-7 + 4 * E) * g.abs()
    h = a * up
    eh = ea * (up.abs() + du) + a.abs() * du + u * h.abs() + TINY[t]
    r = dict(g=g, eg=dg, up=up, eu=du, y=h @ wd.T, ey=eh @ wd.abs().T + tc(h.shape[1]) * (h.abs() @ wd.abs().T))
    if dy is None:
        return r
    dy = dy.double()
    es = 1.2 * dg + 1e-6 + 8 * E
    if act == "relu":
        es = (g.abs() <= dg).double()
    dh = dy @ wd
    edh = k * (dy.abs() @ wd.abs())
    zu, zg = dh * a, dh * up * slope
    ezu = (edh * (a.abs() + ea) + dh.abs() * ea) * 1.01 + u * zu.abs() + TINY[t]
    ezg = ((edh * (up.abs() + du) + dh.abs() * du) * (slope.abs() + es) + (dh * up).abs() * es) * 1.01 + u * zg.abs() + TINY[t]
    # what is rounded to the type may itself be off before that
    r["dx"] = zg @ wg + zu @ wu
    r["edx"] = ezg @ wg.abs() + ezu @ wu.abs() + tc(2 * h.shape[1]) * (zg.abs() @ wg.abs() + zu.abs() @ wu.abs())
    kt = tc(x.shape[0])
    for n, z, e in (("dwg", zg, ezg), ("dwu", zu, ezu)):
        r[n] = z.T @ x
        r["e" + n] = e.T @ x.abs() + kt * (z.abs().T @ x.abs())
    r["dwd"] = dy.T @ h
    r["edwd"] = dy.abs().T @ eh + kt * (dy.abs().T @ h.abs())
    return r


def ffn_operands(t, rows, width, hidden, lead=()):
    gen = seeded(rows, width, hidden, len(t))
    return (rand(gen, (*lead, rows, width), t), rand(gen, (hidden, width), t, width ** -0.5),
            rand(gen, (hidden, width), t, width ** -0.5), rand(gen, (width, hidden), t, hidden ** -0.5),
            rand(gen, (*lead, rows, width), t, 0.3))


def check_ffn(got, grads, r, t, wt=None):
    close(got.y, r["y"], r["ey"], t)
    if grads is not None:
        close(got.gate, r["g"], r["eg"], "float32")
        close(got.up, r["up"], r["eu"], "float32")
        close(grads.x, r["dx"], r["edx"], t)
        for v, n in ((grads.w_gate, "dwg"), (grads.w_up, "dwu"), (grads.w_down, "dwd")):
            close(v, r[n], r["e" + n], wt or t)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("rows,width,hidden", [
    (1, 1, 1), (1, 64, 64), (2, 8, 24), (3, 1000, 17), (3, 250, 66), (4, 1024, 512), (7, 65, 130), (8, 16, 2000), (9, 16, 64), (17, 65, 33),
    (64, 128, 320), (129, 200, 77), (300, 72, 1000), (1500, 520, 264)])
def test_feed_forward(ops, act, t, rows, width, hidden):
    x, wg, wu, wd, dy = ffn_operands(t, rows, width, hidden)
    r = ffn64(x, wg, wu, wd, dy, act, t)
    got = ops.feed_forward(x, wg, wu, wd, act=act, keep=True)
    grads = ops.feed_forward_grad(dy, x, wg, wu, wd, got.gate, got.up, act=act)
    check_ffn(got, grads, r, t)
    alone = ops.feed_forward(x, wg, wu, wd, act=act)
    assert torch.equal(alone.y, got.y) and alone.gate is None
    again = ops.feed_forward_grad(dy, x, wg, wu, wd, got.gate, got.up, act=act)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("rows,width,hidden", [(5000, 64, 96), (4095, 512, 640), (700, 1001, 2731), (130, 4096, 128), (20000, 40, 16), (2467, 385, 1274)])
def test_feed_forward_products_that_are_cut(ops, t, rows, width, hidden):
    """Sizes whose last round of tiles is cut along K, odd ones among them; results in 32 bits, and added."""
    x, wg, wu, wd, dy = ffn_operands(t, rows, width, hidden)
    r = ffn64(x, wg, wu, wd, dy, "silu", t)
    got = ops.feed_forward(x, wg, wu, wd, keep=True)
    check_ffn(got, ops.feed_forward_grad(dy, x, wg, wu, wd, got.gate, got.up), r, t)
    for o in ("float32", t):
        gen = seeded(rows, len(o))
        base = [rand(gen, w.shape, o) for w in (wg, wu, wd)]
        for more in (False, True):
            out = (torch.empty_like(x), *(b.clone() for b in base))
            g = ops.feed_forward_grad(dy, x, wg, wu, wd, got.gate, got.up, out=out, accumulate=more)
            q = dict(r)
            if more:
                for n, b in zip(("dwg", "dwu", "dwd"), base):
                    q[n] = r[n] + b.double()
                    q["e" + n] = r["e" + n] + E * (r[n].abs() + b.double().abs())
            check_ffn(got, g, q, t, o)


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("rows", [5, 70])
def test_feed_forward_strides_and_places(ops, t, rows):
    """Rows further apart than they are long, unaligned ones, halves of one array, and what lies between."""
    width, hidden = 72, 136
    gen = seeded(rows, len(t), 5)
    both = rand(gen, (2 * hidden, width + 9), t, 0.1)
    wg, wu = both[:hidden, 1:width + 1], both[hidden:, 8:width + 8]
    wd = rand(gen, (width, hidden + 3), t, 0.1)[:, 3:]
    x, dy = rand(gen, (rows, 2 * width), t)[:, width:], rand(gen, (rows, width + 1), t)[:, 1:]
    r = ffn64(x, wg, wu, wd, dy, "gelu", t)
    kept = torch.full((rows, 2 * hidden + 1), 3.0, device="cuda")
    y = torch.full((rows, width + 5), 3.0, device="cuda", dtype=dtype(t))
    got = ops.feed_forward(x, wg, wu, wd, act="gelu", keep=True,
                           out=(y[:, 2:width + 2], kept[:, :hidden], kept[:, hidden + 1:]))
    dw = torch.full((2, hidden, width + 2), 3.0, device="cuda", dtype=dtype(t))
    dd = torch.full((width, hidden + 1), 3.0, device="cuda", dtype=dtype(t))
    dx = torch.full((rows, width + 8), 3.0, device="cuda", dtype=dtype(t))
    grads = ops.feed_forward_grad(dy, x, wg, wu, wd, got.gate, got.up, act="gelu",
                                  out=(dx[:, :width], dw[0, :, :width], dw[1, :, 1:width + 1], dd[:, 1:]))
    check_ffn(got, grads, r, t)
    for edge in (kept[:, hidden], y[:, :2], y[:, width + 2:], dw[0, :, width:], dw[1, :, 0], dw[1, :, -1], dd[:, 0], dx[:, width:]):
        assert (edge == 3).all()
    x3 = rand(gen, (2, 3, width), t)
    z = ops.feed_forward(x3, wg, wu, wd)
    assert z.y.shape == x3.shape and torch.equal(z.y, ops.feed_forward(x3.reshape(6, width), wg, wu, wd).y.reshape(x3.shape))


def test_feed_forward_nothing_and_no_numbers(ops):
    x, wg, wu, wd, dy = ffn_operands("bfloat16", 20, 64, 96)
    none = ops.feed_forward(x[:0], wg, wu, wd, keep=True)
    assert none.y.shape == (0, 64) and none.gate.shape == (0, 96)
    g = ops.feed_forward_grad(dy[:0], x[:0], wg, wu, wd, none.gate, none.up)
    assert g.x.shape == (0, 64) and all((v == 0).all() for v in g[1:])
    kept = [torch.ones_like(w) for w in (wg, wu, wd)]
    ops.feed_forward_grad(dy[:0], x[:0], wg, wu, wd, none.gate, none.up, out=(x[:0].clone(), *kept), accumulate=True)
    assert all((v == 1).all() for v in kept)
    for rows in (4, 20):  # a row of NaN stays in its row
        bad = x[:rows].clone()
        bad[1, 5] = math.nan
        y = ops.feed_forward(bad, wg, wu, wd)
        clean = ops.feed_forward(x[:rows], wg, wu, wd)
        assert y.y[1].isnan().all() and torch.equal(y.y[2:], clean.y[2:]) and torch.equal(y.y[0], clean.y[0])


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("rows", [2, 40])
def test_feed_forward_of_large_values(ops, act, rows):
    """Saturated activations: their values and slopes are 0 or 1, not NaN.  What is large goes through the gate
    alone, so that h stays in bf16's range."""
    one = torch.eye(8, device="cuda", dtype=torch.bfloat16)
    z = torch.tensor([-1e30, -3e4, -90.0, -12.0, 12.0, 90.0, 3e4, 1e30], device="cuda").bfloat16()
    small = 1 / z.abs().clamp(min=100.0)
    x, wu = z.repeat(rows, 1), torch.diag(small)
    f = ops.feed_forward(x, one, wu, one, act=act, keep=True)
    g = ops.feed_forward_grad(torch.ones_like(x), x, one, wu, one, f.gate, f.up, act=act)
    a, slope = act64(x.double(), act if act != "gelu_tanh" else "gelu")  # the same to 1e-3 where they are this large
    u = x.double() * small.double()
    for got, want in ((f.y, a * u), (g.x, slope * u + a * small.double())):
        assert torch.isfinite(got).all()
        assert ((got.double() - want).abs() <= 2.0 ** -6 * want.abs() + 1e-3 * (1 + u.abs())).all()


def test_feed_forward_gradients_of_many_sizes_in_turn(ops):
    # the same bits whatever sizes, devices' streams and threads came before
    import threading

    gen = seeded(31)
    x = rand(gen, (70, 64), "bfloat16")
    weights = [[rand(gen, s, "bfloat16") for s in ((h, 64), (h, 64), (64, h))] for h in range(8, 8 + 33 * 24, 24)]

    def grads(w, stream=None):
        with torch.cuda.stream(stream or torch.cuda.current_stream()):
            r = ops.feed_forward(x, *w, keep=True)
            return r.y, *ops.feed_forward_grad(x, x, *w, r.gate, r.up)

    first = [grads(w) for w in weights]
    others = {}

    def work(name):
        stream = torch.cuda.Stream()
        others[name] = [grads(w, stream) for w in weights[::-1]][::-1]
        stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    again = [grads(w) for w in weights]
    torch.cuda.synchronize()
    for got in (again, others[0], others[1]):
        assert all(torch.equal(a, b) for u, v in zip(first, got) for a, b in zip(u, v))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_feed_forward_gradient_against_differences(ops, act):
    """The gradients in random directions against central differences of the 64-bit block: the truncation error
    of a step s is s^2 / 6 of a third derivative, and the gradients' errors are ffn64's."""
    t = "bfloat16"
    x, wg, wu, wd, dy = ffn_operands(t, 48, 40, 56)
    r = ffn64(x, wg, wu, wd, dy, act, t)
    f = ops.feed_forward(x, wg, wu, wd, act=act, keep=True)
    g = ops.feed_forward_grad(dy, x, wg, wu, wd, f.gate, f.up, act=act)
    gen = seeded(9)
    operands = [v.double() for v in (x, wg, wu, wd)]
    for i, (grad, bound) in enumerate(zip(g, (r["edx"], r["edwg"], r["edwu"], r["edwd"]))):
        way = torch.randn(operands[i].shape, generator=gen, dtype=torch.float64).cuda()

        def loss(s):
            v = [o + s * way if j == i else o for j, o in enumerate(operands)]
            a, _ = act64(v[0] @ v[1].T, act)
            return float(((a * (v[0] @ v[2].T)) @ v[3].T * dy.double()).sum())

        s = 1e-4
        slope = (loss(s) - loss(-s)) / (2 * s)
        err = float(((bound + U[t] * grad.double().abs()) * way.abs()).sum())
        assert abs(float((grad.double() * way).sum()) - slope) <= 1.05 * err + 1e-5 * abs(slope) + 1e-4


# ------------------------------------------------------------------ log probabilities of a linear layer

def linear64(x, w, tokens, scale, gp=None, gl=None, t=None):
    """Results and bounds: those of a row's logits are taken at their largest; weights of a sum are off by
    their exponent's error, on average over a row by no more than log V + 4 half steps; terms are added in
    at most V / 64 + 64 steps one after another."""
    x, w = x.double().reshape(-1, x.shape[-1]), w.double()
    rows, vocab = x.shape[0], w.shape[0]
    z = scale * (x @ w.T)
    ez = scale * tc(x.shape[1]) * (x.abs() @ w.abs().T)
    lse = torch.logsumexp(z, -1)
    row = ez.amax(-1)
    n = (math.log(vocab) + 4) * 4 + vocab / 64 + 64
    elf = row + n * E + 4 * E * (lse.abs() + z.amax(-1).abs())
    has, known = tokens >= 0, tokens < vocab
    at = tokens.clamp(0, vocab - 1)
    idx = torch.arange(rows, device=x.device)
    logp = torch.where(has, z[idx, at] - lse, 0.0)
    logp[~known] = math.nan
    r = dict(lse=lse, elf=elf, logp=logp, elp=elf + ez[idx, at] + 4 * E * (z[idx, at].abs() + lse.abs()))
    if t is None:
        return r
    gp = torch.zeros(rows, device=x.device) if gp is None else gp
    gl = torch.zeros(rows, device=x.device) if gl is None else gl
    gp, gl = torch.where(has, gp.double(), 0.0), gl.double()
    p = torch.softmax(z, -1)
    # the exponent's own error grows with its distance from the largest
    ep = p * (ez + elf[:, None] + 4 * E * (z.amax(-1, keepdim=True) - z) + 8 * E)
    d = p * (gl - gp)[:, None]
    d[idx, at] += gp
    d, mag = scale * d, scale * (gl.abs() + 2 * gp.abs())
    d[~known] = math.nan
    ed = scale * ep * (gl.abs() + gp.abs())[:, None] * 1.01 + 4 * E * scale * (p * (gl.abs() + gp.abs())[:, None]) + U[t] * d.abs()
    ed[idx, at] += 4 * E * scale * gp.abs()
    if t == "float16":
        ed = ed + 2.0 ** -38 * mag.nan_to_num().amax()
    ed = ed + 2.0 ** -134
    r["dx"], r["dw"] = d @ w, d.T @ x
    pieces = rows * vocab / 2 ** 28 + 2
    r["edx"] = ed @ w.abs() + (tc(vocab) + pieces * E) * (d.abs() @ w.abs())
    r["edw"] = ed.T @ x.abs() + tc(rows) * (d.abs().T @ x.abs())
    return r


def linear_operands(t, rows, width, vocab, lead=()):
    gen = seeded(rows, width, vocab, len(t))
    x, w = rand(gen, (*lead, rows, width), t), rand(gen, (vocab, width), t, 2.5 * width ** -0.5)
    tokens = torch.randint(0, vocab, (*lead, rows), generator=gen)
    if rows > 3:
        tokens[..., ::4] = -1
    return x, w, tokens.cuda(), rand(gen, (*lead, rows), "float32"), rand(gen, (*lead, rows), "float32", 0.1)


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("scale", [1.0, 0.6])
@pytest.mark.parametrize("rows,width,vocab", [
    (1, 1, 1), (1, 64, 2), (2, 8, 300), (3, 65, 77), (31, 16, 33), (64, 512, 1000), (130, 72, 257), (257, 200, 4099),
    (1000, 64, 63), (9, 1000, 20000), (600, 1001, 2048),
    (7, 512, 29204), (2, 128, 28660), (40, 2000, 9000), (200, 300, 31000)])
def test_linear_logprobs(ops, t, scale, rows, width, vocab):
    x, w, tokens, gp, gl = linear_operands(t, rows, width, vocab)
    want = linear64(x, w, tokens, scale, gp, gl, t)
    r = ops.linear_logprobs(x, w, tokens, scale=scale)
    close(r.logp, want["logp"], want["elp"], "float32")
    close(r.lse, want["lse"], want["elf"], "float32")
    g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl, scale=scale)
    close(g.x, want["dx"], want["edx"], t)
    close(g.weight, want["dw"], want["edw"], t)
    again = ops.linear_logprobs_grad(x, w, tokens.int(), r.stats, gp, gl, scale=scale)
    assert torch.equal(again.x, g.x) and torch.equal(again.weight, g.weight)
    assert torch.equal(ops.linear_logprobs(x, w, tokens.int(), scale=scale).logp, r.logp)


@pytest.mark.parametrize("t", HALVES)
def test_linear_logprobs_in_pieces(ops, t):
    """More logits than a piece holds (2^28): several pieces, the last one smaller, sums over them in 32 bits."""
    x, w, tokens, gp, gl = linear_operands(t, 9000, 24, 50003)
    want = linear64(x, w, tokens, 1.0, gp, gl, t)
    r = ops.linear_logprobs(x, w, tokens)
    close(r.logp, want["logp"], want["elp"], "float32")
    g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl)
    close(g.x, want["dx"], want["edx"], t)
    close(g.weight, want["dw"], want["edw"], t)


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("which", ["logp", "lse", "none"])
def test_linear_logprobs_gradients_apart_and_added(ops, t, which):
    x, w, tokens, gp, gl = linear_operands(t, 200, 96, 500)
    gp, gl = (gp if which == "logp" else None), (gl if which == "lse" else None)
    want = linear64(x, w, tokens, 1.0, gp, gl, t)
    r = ops.linear_logprobs(x, w, tokens)
    for o in (t, "float32"):
        base = rand(seeded(3), w.shape, o)
        out = (torch.empty_like(x), base.clone())
        g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl, out=out, accumulate=True)
        close(g.x, want["dx"], want["edx"], t)
        close(g.weight, base.double() + want["dw"], want["edw"] + E * (want["dw"].abs() + base.double().abs()), o)
    if which == "none":
        assert (g.x == 0).all() and torch.equal(g.weight, base)


def test_linear_logprobs_strides_shapes_and_nothing(ops):
    t = "bfloat16"
    gen = seeded(21)
    x, w = rand(gen, (2, 30, 70), t)[:, :, 5:69], rand(gen, (90, 80), t, 0.3)[10:, 1:65]
    x = x.contiguous().reshape(2, 30, 64)
    tokens = torch.randint(-1, 80, (2, 30), generator=gen).cuda()
    want = linear64(x, w, tokens.reshape(-1), 1.0)
    r = ops.linear_logprobs(x, w, tokens)
    assert r.logp.shape == (2, 30) and r.stats.shape == (60, 2)
    close(r.logp.reshape(-1), want["logp"], want["elp"], "float32")
    wide = rand(gen, (60, 100), t)
    for xs in (wide[:, 8:72], wide[:, 3:67]):
        want = linear64(xs, w, tokens.reshape(-1), 1.0, r.logp.reshape(-1), None, t)
        q = ops.linear_logprobs(xs, w, tokens)
        dx, dw = (torch.full(s, 3.0, device="cuda", dtype=torch.bfloat16) for s in ((60, 66), (80, 70)))
        ops.linear_logprobs_grad(xs, w, tokens, q.stats, r.logp.reshape(-1).contiguous(), out=(dx[:, 1:65], dw[:, 6:]))
        close(dx[:, 1:65], want["dx"], want["edx"], t)
        close(dw[:, 6:], want["dw"], want["edw"], t)
        assert (dx[:, 0] == 3).all() and (dx[:, 65] == 3).all() and (dw[:, :6] == 3).all()
    none = ops.linear_logprobs(x[:0], w, tokens[:0])
    assert none.logp.shape == (0, 30)
    g = ops.linear_logprobs_grad(x[:0], w, tokens[:0], none.stats)
    assert (g.weight == 0).all() and g.x.shape == (0, 30, 64)
    kept = torch.ones(80, 64, device="cuda")
    ops.linear_logprobs_grad(x[:0], w, tokens[:0], none.stats, out=(x[:0].clone(), kept), accumulate=True)
    assert (kept == 1).all()


def test_linear_logprobs_unknown_tokens_and_no_numbers(ops):
    x, w, tokens, gp, gl = linear_operands("bfloat16", 40, 64, 300)
    tokens[5], tokens[7] = 300, 1 << 40
    r = ops.linear_logprobs(x, w, tokens)
    assert r.logp[5].isnan() and r.logp[7].isnan() and r.lse.isfinite().all()
    g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp)
    rows = torch.zeros(40, dtype=torch.bool, device="cuda")
    rows[[5, 7]] = True
    assert g.x[rows].isnan().all() and g.x[~rows].isfinite().all() and g.weight.isnan().all()
    tokens[[5, 7]] = -1
    x[3, 9] = math.nan
    r = ops.linear_logprobs(x, w, tokens)
    assert r.lse[3].isnan() and r.lse[4:].isfinite().all()


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("size,scale", [(1e-3, 1.0), (30.0, 1.0), (1.0, 1e3), (1.0, 3e30), (1.0, 1e-30)])
def test_linear_logprobs_of_large_and_small_logits(ops, t, size, scale):
    """Nearly equal logits, one far ahead of the others, and scales at the ends of 32 bits."""
    gen = seeded(77)
    x, w = rand(gen, (50, 64), t, size), rand(gen, (700, 64), t, 0.3)
    tokens = torch.randint(0, 700, (50,), generator=gen).cuda()
    tokens[:10] = (x.double() @ w.double().T).argmax(-1)[:10]
    gp = torch.ones(50, device="cuda")
    want = linear64(x, w, tokens, scale, gp, None, t)
    r = ops.linear_logprobs(x, w, tokens, scale=scale)
    close(r.lse, want["lse"], want["elf"], "float32")
    close(r.logp, want["logp"], want["elp"], "float32")
    if scale < 1e10:
        g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, scale=scale)
        # where a probability's error is beyond all bounds, it is still a probability
        limit = want["edx"].clamp(max=1e300)
        if float((linear64(x, w, tokens, scale)["elf"]).max()) < 0.1:
            close(g.x, want["dx"], limit, t)
        assert g.x.isfinite().all() and g.weight.isfinite().all()


def test_linear_logprobs_gradients_of_unequal_size(ops):
    """float16 gradients from 1e-30 to 1e30: held to 2^-38 of the largest row's, times a power of two."""
    x, w, tokens, gp, gl = linear_operands("float16", 64, 32, 400)
    tokens = tokens.clamp(min=0)
    for size in (1e-30, 1e-6, 1.0, 100.0):
        g = gp * size
        r = ops.linear_logprobs(x, w, tokens)
        out = (torch.empty_like(x), torch.empty(w.shape, device="cuda"))
        got = ops.linear_logprobs_grad(x, w, tokens, r.stats, g, out=out)
        want = linear64(x, w, tokens, 1.0, g, None, "float16")
        close(got.weight, want["dw"], want["edw"], "float32")


def test_linear_logprobs_gradient_against_differences(ops):
    t = "bfloat16"
    x, w, tokens, gp, gl = linear_operands(t, 40, 48, 150)
    want = linear64(x, w, tokens, 1.3, gp, gl, t)
    r = ops.linear_logprobs(x, w, tokens, scale=1.3)
    g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl, scale=1.3)
    gen = seeded(8)
    operands = [x.double(), w.double()]
    for i, (grad, bound) in enumerate(zip(g, (want["edx"], want["edw"]))):
        way = torch.randn(operands[i].shape, generator=gen, dtype=torch.float64).cuda()

        def loss(s):
            v = [o + s * way if j == i else o for j, o in enumerate(operands)]
            q = linear64(v[0], v[1], tokens, 1.3)
            return float((q["logp"] * gp.double() + q["lse"] * gl.double()).sum())

        s = 1e-4
        slope = (loss(s) - loss(-s)) / (2 * s)
        err = float(((bound + U[t] * grad.double().abs()) * way.abs()).sum())
        assert abs(float((grad.double() * way).sum()) - slope) <= 1.05 * err + 1e-5 * abs(slope) + 1e-4


def test_linear_logprobs_agrees_with_token_logprobs(ops):
    """The same quantity as the operator on logits gives, from logits rounded to 32 bits."""
    x, w, tokens, _, _ = linear_operands("bfloat16", 100, 128, 3000)
    logits = (x.double() @ w.double().T).float()
    a, b = ops.linear_logprobs(x, w, tokens, scale=0.8), ops.token_logprobs(logits, tokens, scale=0.8)
    want = linear64(x, w, tokens, 0.8)
    assert ((a.logp - b.logp).abs() <= 2 * want["elp"] + 64 * E * (1 + want["logp"].abs())).all()
    assert ((a.lse - b.stats[:, 3]).abs() <= 2 * want["elf"] + 64 * E * (1 + want["lse"].abs())).all()


# ------------------------------------------------------------------ clipping

def clip64(grads, most):
    n = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    f = most / n if n > most and torch.isfinite(n) else torch.ones((), dtype=torch.float64, device="cuda")
    return n, [g.double() * f for g in grads]


def check_clip(ops, grads, most, **kw):
    """The norm is off by half of what squares (8 additions in 32 bits) are, and by its rounding; a
    product by that of its factor, and a rounding more."""
    n, want = clip64(grads, most)
    got = [g.clone() for g in grads]
    norm = ops.clip_norm(got, most, **kw)
    assert norm.shape == (1,)
    assert abs(float(norm) - float(n)) <= (8 * E + E) * float(n) + 1e-45
    for v, w in zip(got, want):
        close(v, w, 8 * E * w.abs(), str(v.dtype).replace("torch.", ""))
    apart = [torch.full_like(g, 9.0) for g in grads]
    before = [g.clone() for g in grads]
    assert torch.equal(ops.clip_norm(grads, most, out=apart), norm)
    assert all(torch.equal(a, b) for a, b in zip(apart, got)) and all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("t", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("sizes", [(1,), (0, 3), (4096,), (1, 2, 3, 5, 7, 8, 9, 15, 16, 17), (70001, 16384, 5), (1000003,)])
@pytest.mark.parametrize("most", [0.5, 1e9, 0.0])
def test_clip_norm(ops, t, sizes, most):
    gen = seeded(sum(sizes), len(t))
    check_clip(ops, [rand(gen, (n,), t) for n in sizes], most)


@pytest.mark.parametrize("count", [63, 64, 65, 767, 768, 769, 1600])
def test_clip_norm_of_many_arrays(ops, count):
    """One launch of up to 64 arrays, of up to 768, and several; types mixed, some of no elements."""
    gen = seeded(count)
    kinds = ("float32", "bfloat16", "float16")
    store = rand(gen, (count * 40 + 2000,), "float32")
    grads = [(store[40 * i:40 * i + (i * 7) % 41] * (1 + i % 3)).to(dtype(kinds[i % 3])) for i in range(count)]
    grads[count // 2] = rand(gen, (30000,), "bfloat16")
    check_clip(ops, grads, 1.0)


def test_clip_norm_places_and_orders(ops):
    """Views at any element, results aligned otherwise than operands, axes in any order."""
    gen = seeded(5)
    for t in ("float32", "bfloat16"):
        store = rand(gen, (9000,), t)
        views = [store[1:1500], store[1503:1511], store[2001:2002], store[3000:6001], store[7001:]]
        n, want = clip64(views, 1.0)
        other = torch.full((9100,), 4.0, device="cuda", dtype=dtype(t))
        out = [other[1 + 3 * i + v.storage_offset():][:v.numel()] for i, v in enumerate(views)]
        norm = ops.clip_norm(views, 1.0, out=out)
        assert abs(float(norm) - float(n)) <= 9 * E * float(n)
        for v, w in zip(out, want):
            close(v, w, 8 * E * w.abs(), t)
        assert (other == 4).sum() == 9100 - sum(v.numel() for v in views)
        ops.clip_norm(views, 1.0)
        for v, w in zip(views, want):
            close(v, w, 8 * E * w.abs(), t)
    m = rand(gen, (30, 50), "float32")
    check = [m.t(), rand(gen, (3, 4, 5), "bfloat16").permute(2, 0, 1), rand(gen, (), "float32")]
    n, want = clip64(check, 0.1)
    assert abs(float(ops.clip_norm(check, 0.1)) - float(n)) <= 9 * E * float(n)
    for v, w in zip(check, want):
        close(v, w, 8 * E * w.abs(), str(v.dtype).replace("torch.", ""))


@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e18, 1e25, 1e37])
def test_clip_norm_of_any_size(ops, size):
    """Squares that vanish or overflow in 32 bits."""
    gen = seeded(3)
    for t in ("float32", "bfloat16"):
        grads = [rand(gen, (n,), t, size) for n in (5000, 33)]
        n, want = clip64(grads, size)
        assert float(n) > size
        norm = ops.clip_norm(grads, size)
        if float(n) > torch.finfo(torch.float32).max:  # what is returned is rounded to 32 bits; the factor is not
            assert float(norm) == math.inf
        else:
            assert abs(float(norm) - float(n)) <= 9 * E * float(n)
        for v, w in zip(grads, want):
            close(v, w, 8 * E * w.abs(), t)
    grads = [rand(gen, (4000,), "float32", size)]  # a factor that 32 bits do not hold in full
    n, want = clip64(grads, 1e-35)
    ops.clip_norm(grads, 1e-35)
    close(grads[0], want[0], 8 * E * want[0].abs(), "float32")


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_clip_norm_that_is_no_number(ops, bad):
    gen = seeded(6)
    grads = [rand(gen, (1000,), "float32"), rand(gen, (77,), "bfloat16")]
    grads[0][500] = bad
    before = [g.clone() for g in grads]
    norm = ops.clip_norm(grads, 1.0)
    assert not torch.isfinite(norm).any()
    apart = [torch.empty_like(g) for g in grads]
    ops.clip_norm(grads, 1.0, out=apart)
    for a, b, c in zip(grads, before, apart):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and torch.equal(c.nan_to_num(7.0), b.nan_to_num(7.0))


def test_clip_norm_gives_the_norm_alone(ops):
    gen = seeded(2)
    grads = [rand(gen, (100000,), "bfloat16")]
    before = grads[0].clone()
    norm = ops.clip_norm(grads, math.inf)
    assert torch.equal(grads[0], before) and abs(float(norm) - float(before.double().norm())) <= 9 * E * float(norm)
    ops.clip_norm([torch.empty(0, device="cuda")], 1.0, norm=norm)
    assert float(norm) == 0


# ------------------------------------------------------------------ streams, graphs, threads

def calls(ops, seed):
    """A call of each operator on operands of its own: (call, operands); a call returns its results."""
    gen = seeded(seed)
    x, wg, wu, wd, dy = ffn_operands("bfloat16", 300, 136, 328)
    table, tokens = rand(gen, (500, 136), "bfloat16"), torch.randint(-1, 500, (3000,), generator=gen).cuda()
    d = rand(gen, (3000, 136), "bfloat16")
    t300 = tokens[:300].contiguous()
    f = ops.feed_forward(x, wg, wu, wd, keep=True)
    r = ops.linear_logprobs(x, table, t300)
    g = rand(gen, (300,), "float32")
    grads = [rand(gen, (70, 11), "float32"), rand(gen, (999,), "bfloat16")]
    many, wide = torch.randint(-1, 9000, (20000,), generator=gen).cuda(), rand(gen, (20000, 24), "bfloat16")
    return [
        (lambda: [ops.embed(tokens, table)], table),
        (lambda: [ops.embed_grad(d, tokens, 500)], d),
        (lambda: [ops.embed_grad(d[:200], tokens[:200], 500)], d),
        (lambda: [ops.embed_grad(wide[:6000], many[:6000], 9000)], wide),
        (lambda: [ops.embed_grad(wide[:15000], many[:15000], 9000)], wide),
        (lambda: [ops.embed_grad(wide, many, 9000)], wide),
        (lambda: [ops.feed_forward(x, wg, wu, wd).y], x),
        (lambda: [ops.feed_forward(x[:3], wg, wu, wd).y], x),
        (lambda: list(ops.feed_forward_grad(dy, x, wg, wu, wd, f.gate, f.up)), dy),
        (lambda: list(ops.linear_logprobs(x, table, t300)), x),
        (lambda: list(ops.linear_logprobs_grad(x, table, t300, r.stats, g)), g),
        (lambda: (lambda o: [ops.clip_norm(grads, 0.3, out=o), *o])([torch.empty_like(v) for v in grads]), grads[0]),
    ]


def test_replayed_graphs_follow_their_operands(ops):
    """Each call in a graph of its own, replayed after its operand has changed, and all in one graph."""
    made = calls(ops, 1)
    for call, _ in made:
        call()
    graphs = []
    for call, operand in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, call, operand, out))
    whole = torch.cuda.CUDAGraph()
    with torch.cuda.graph(whole):
        together = [call() for call, _ in made]
    for step in range(2):
        for _, _, operand, _ in graphs:
            operand.mul_(-0.5)
        for g, call, operand, out in graphs:
            g.replay()
        for g, call, operand, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, call()))
        whole.replay()
        for out, (_, call, _, _) in zip(together, graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, call()))


@pytest.mark.parametrize("which", range(7))
def test_first_call_can_be_captured(which):
    """In a process of its own, with nothing run before."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from ad_b200 import ops
torch.manual_seed(0)
x, w = torch.randn(40, 64, device="cuda").bfloat16(), torch.randn(96, 64, device="cuda").bfloat16()
d, t = torch.randn(64, 96, device="cuda").bfloat16(), torch.arange(40, device="cuda")
kept = torch.randn(2, 40, 96, device="cuda")
stats = torch.ones(40, 2, device="cuda")
call = [lambda: ops.embed(t, w), lambda: ops.embed_grad(x, t, 96), lambda: ops.feed_forward(x, w, w, d).y,
        lambda: ops.feed_forward_grad(x, x, w, w, d, kept[0], kept[1]).w_down, lambda: ops.linear_logprobs(x, w, t).lse,
        lambda: ops.linear_logprobs_grad(x, w, t, stats, stats[:, 0].contiguous()).weight,
        lambda: ops.embed_grad(x.repeat(200, 1), t.repeat(200), 96)][%d]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = call()
for _ in range(2):
    g.replay()
assert torch.equal(y, call()) and bool(y.isfinite().all())
""" % which
    r = subprocess.run([sys.executable, "-c", code], cwd=root, env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


def test_other_streams_and_threads(ops):
    made = calls(ops, 2)
    want = [call() for call, _ in made]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                for (call, _), w in zip(made[k:] + made[:k], want[k:] + want[:k]):
                    if not all(torch.equal(a, b) for a, b in zip(call(), w)):
                        wrong.append(k)
            s.synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_given_stream_and_workspace(ops):
    x, w, tokens, gp, gl = linear_operands("bfloat16", 70, 128, 900)
    f = ffn_operands("bfloat16", 70, 128, 192)
    s = torch.cuda.Stream()
    with pytest.raises(ValueError, match="have to be given"):
        ops.linear_logprobs(x, w, tokens, stream=s)
    want, wf = ops.linear_logprobs(x, w, tokens), ops.feed_forward(*f[:4])
    out = ops.LinearLogprobs(*(torch.empty_like(v) for v in want))
    work = torch.empty(max(ops.linear_logprobs_workspace(x, w), ops.feed_forward_workspace(*f[:4])), device="cuda", dtype=torch.uint8)
    y = torch.empty_like(wf.y)
    torch.cuda.synchronize()
    ops.linear_logprobs(x, w, tokens, out=out, workspace=work, stream=s)
    ops.feed_forward(*f[:4], out=(y, None, None), workspace=work, stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(y, wf.y)
    with pytest.raises(Exception, match="bytes of workspace"):
        ops.linear_logprobs(x, w, tokens, out=out, workspace=work[:256])


def test_offsets_past_32_bits(ops):
    """Rows whose elements lie more than 2^31 elements from the first one's."""
    ld, rows = 1 << 20, 2100
    store = torch.zeros(rows * ld, device="cuda", dtype=torch.bfloat16)
    table = store.as_strided((rows, 64), (ld, 1))
    gen = seeded(1)
    table.copy_(rand(gen, (rows, 64), "bfloat16"))
    tokens = torch.arange(rows - 1, -1, -1, device="cuda")
    dense = table.contiguous()
    assert torch.equal(ops.embed(tokens, table), dense.flip(0))
    w = rand(gen, (100, 64), "bfloat16")
    some = torch.randint(0, 100, (rows,), generator=gen).cuda()
    a, b = ops.linear_logprobs(table, w, some), ops.linear_logprobs(dense, w, some)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    x = rand(gen, (50, 64), "bfloat16")
    a, b = (ops.linear_logprobs(x, v, some[:50].contiguous()) for v in (table, dense))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    dy = rand(gen, (rows, 64), "bfloat16")
    got = ops.embed_grad(dy, tokens, rows, out=table)
    assert torch.equal(got, dy.flip(0)) and int((store != 0).sum()) == int((dy != 0).sum())


# ------------------------------------------------------------------ as they are used

def test_a_training_step(ops):
    """A small model whose step runs through all of them: embedding, norms around a gated feed-forward block,
    the loss over the tied vocabulary, the table's two gradients in one array, clipping, and the update of a matrix.
    Against the same in 64 bits by torch's differentiation.  Every value passes at most 14 roundings of half a step
    of bf16 on its way, each of which is a relative error of 2^-8 at most, and the operators' amplification of a
    relative error is near 1 (norms are divided out): norm-wise 14 x 2^-8 for gradients, of the loss a fraction."""
    vocab, width, hidden, rows = 600, 128, 384, 500
    gen = seeded(31)
    table = rand(gen, (vocab, width), "bfloat16", 0.5)
    wg, wu = (rand(gen, (hidden, width), "bfloat16", width ** -0.5) for _ in range(2))
    wd = rand(gen, (width, hidden), "bfloat16", hidden ** -0.5)
    n1, n2 = (1 + rand(gen, (width,), "float32", 0.1) for _ in range(2))
    tokens = torch.randint(0, vocab, (rows,), generator=gen).cuda()
    target = torch.roll(tokens, -1)
    target[-1] = -1
    # forward
    e = ops.embed(tokens, table, scale=2.0)
    zero = torch.zeros_like(e)
    x, y, s1 = ops.block_norm(e, zero, None, n1)
    f = ops.feed_forward(y, wg, wu, wd, keep=True)
    h, z, s2 = ops.block_norm(x, f.y, None, n2)
    r = ops.linear_logprobs(z, table, target)
    loss = -r.logp.sum() / (rows - 1)
    # backward
    gp = torch.full((rows,), -1.0 / (rows - 1), device="cuda")
    dtable = torch.empty(vocab, width, device="cuda")
    gl = ops.linear_logprobs_grad(z, table, target, r.stats, gp, out=(torch.empty_like(z), dtable))
    b2 = ops.block_norm_grad(torch.zeros_like(h), gl.x, x, f.y, None, n2, s2)
    gf = ops.feed_forward_grad(b2.z, y, wg, wu, wd, f.gate, f.up)
    b1 = ops.block_norm_grad(b2.x, gf.x, e, zero, None, n1, s1)
    ops.embed_grad(b1.x, tokens, vocab, scale=2.0, accumulate=True, out=dtable)
    grads = [dtable, gf.w_gate, gf.w_up, gf.w_down, b1.before_weight, b2.before_weight]
    before = [g.clone() for g in grads]
    norm = ops.clip_norm(grads, 0.01)
    update = ops.orthogonalize(grads[1])
    # the same in 64 bits
    p = [v.double().requires_grad_() for v in (table, wg, wu, wd, n1, n2)]
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    e64 = 2.0 * p[0][tokens]
    y64 = rms(e64) * p[4]
    a = y64 @ p[1].T
    h64 = e64 + (a * torch.sigmoid(a) * (y64 @ p[2].T)) @ p[3].T
    lp = torch.log_softmax((rms(h64) * p[5]) @ p[0].T, -1)
    want = -lp[torch.arange(rows - 1), target[:-1]].sum() / (rows - 1)
    want.backward()
    bound = 14 * 2.0 ** -8
    assert abs(float(loss.detach()) - float(want.detach())) <= bound * abs(float(want.detach()))
    for g, q in zip(before, p):
        assert float((g.double() - q.grad).norm()) <= bound * float(q.grad.norm())
    n64 = torch.stack([g.double().square().sum() for g in before]).sum().sqrt()
    assert abs(float(norm) - float(n64)) <= 9 * E * float(n64)
    for g, q in zip(grads, before):
        close(g, q.double() * (0.01 / n64), 8 * E * (q.double() * (0.01 / n64)).abs(), str(g.dtype).replace("torch.", ""))
    assert update.isfinite().all() and update.shape == wg.shape


def test_half_precision_example(ops):
    """The example's gradients against the same model in plain 64-bit torch.  A value passes some 14 roundings of
    bf16 forward and as many backward: norm-wise 28 x 2^-8.  And it runs."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "lm_half.py")
    spec = importlib.util.spec_from_file_location("lm_half", path)
    lm = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(lm)
    model = lm.Model(vocab=61, width=64, heads=4, hidden=160, layers=1, length=16)
    tokens = torch.randint(0, 61, (5, 16), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    p = model.leaves()
    loss = model.loss(tokens, p)
    loss.backward()
    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    rms = lambda v, w: v * (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w  # noqa: E731

    def turn(v):
        u, w = v[..., :8], v[..., 8:]
        c, s = model.cos.double()[:16, None], model.sin.double()[:16, None]
        return torch.cat((u * c - w * s, w * c + u * s), -1)

    x = q["table"][tokens].reshape(80, 64)
    y = rms(x, q["first"])
    a, b, c = (t.reshape(5, 16, 4, 16) for t in (y @ q["qkv0"].T).chunk(3, -1))
    s = torch.einsum("bthd,bshd->bhts", turn(a), turn(b)) / 4 + model.mask.double()
    z = torch.einsum("bhts,bshd->bthd", s.softmax(-1), c).reshape(80, 64) @ q["out0"].T
    x = x + torch.sigmoid(q["g10"]) * rms(z, q["a10"])
    y = rms(x, q["b10"])
    g = y @ q["gate0"].T
    z = (g * torch.sigmoid(g) * (y @ q["up0"].T)) @ q["down0"].T
    x = x + torch.sigmoid(q["g20"]) * rms(z, q["a20"])
    lp = torch.log_softmax(rms(x, q["b20"]) @ q["table"].T, -1).reshape(5, 16, 61)[:, :-1]
    want = -lp.gather(-1, tokens[:, 1:, None]).sum() / 75
    want.backward()
    bound = 28 * 2.0 ** -8
    assert abs(float(loss.detach()) - float(want.detach())) <= bound * float(want.detach())
    for k in p:
        assert float((p[k].grad.double() - q[k].grad).norm()) <= bound * float(q[k].grad.norm()), k
    assert all(math.isfinite(v) for v in lm.main(3))

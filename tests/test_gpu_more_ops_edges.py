"""Embeddings, feed-forward blocks, log probabilities of a linear layer and gradient clipping at the edges of
what they take (B200 only).  The 64-bit implementations and the bounds' derivation are those of
test_gpu_more_ops."""
import math

import pytest

from .test_gpu_more_ops import HALVES, close, linear64, linear_operands, tc
from .test_gpu_ops import E, U, dtype, rand, seeded

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from ad_b200 import ops as o
    return o


# ------------------------------------------------------------------ log probabilities of a linear layer

@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("garbage", [1e30, -3e38, math.inf, -math.inf, math.nan])
def test_linear_logprobs_gradients_of_rows_without_a_token(ops, t, garbage):
    """What g_logp holds where the token is negative has no part in anything, bit for bit; nor has the
    row of a token past the vocabulary in the gradients of other rows of x."""
    x, w, tokens, gp, gl = linear_operands(t, 64, 48, 300)
    gp, none = gp * 1e-5, tokens < 0
    assert none.any() and not none.all()
    r = ops.linear_logprobs(x, w, tokens)
    out = lambda: (torch.empty_like(x), torch.empty(w.shape, device="cuda"))  # noqa: E731
    for lse in (None, gl * 1e-5):
        want = ops.linear_logprobs_grad(x, w, tokens, r.stats, torch.where(none, 0.0, gp), lse, out=out())
        assert want.weight.count_nonzero() > 0.9 * want.weight.numel()
        got = ops.linear_logprobs_grad(x, w, tokens, r.stats, torch.where(none, garbage, gp), lse, out=out())
        assert torch.equal(got.x, want.x) and torch.equal(got.weight, want.weight)
        past = torch.where(none, 300, tokens)
        got = ops.linear_logprobs_grad(x, w, past, r.stats, torch.where(none, garbage, gp), lse, out=out())
        same = ops.linear_logprobs_grad(x, w, tokens, r.stats, torch.where(none, 0.0, gp),
                                        None if lse is None else torch.where(none, 0.0, lse), out=out())
        assert torch.equal(got.x[~none], same.x[~none]) and got.x[none].isnan().all() and got.weight.isnan().all()


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("least", [2.0 ** -12, 2.0 ** -40])
def test_linear_logprobs_gradients_of_rows_of_unequal_size(ops, t, least):
    """Rows of one call whose gradients lie up to `least` of the largest apart, some of them ignored."""
    x, w, tokens, gp, gl = linear_operands(t, 64, 32, 400)
    size = torch.logspace(0, math.log2(least), 64, base=2.0, device="cuda")[torch.randperm(64, generator=seeded(5)).cuda()]
    gp, gl = gp * size, gl * size
    r = ops.linear_logprobs(x, w, tokens)
    want = linear64(x, w, tokens, 1.0, gp, gl, t)
    g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl, out=(torch.empty_like(x), torch.empty(w.shape, device="cuda")))
    close(g.x, want["dx"], want["edx"], t)
    close(g.weight, want["dw"], want["edw"], "float32")


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("size,scale,std", [(1e30, 1.0, 1.0), (8.0, 1e-35, 1.0), (1e-38, 1e30, 1.0), (3.4e38, 1.0, 2e-3), (3e33, 1e5, 1e-3), (1e-30, 1.0, 1.0), (1e33, 1e-5, 300.0)])
def test_linear_logprobs_gradients_at_the_ends_of_32_bits(ops, t, size, scale, std):
    """Gradients of logp and lse up to the largest of 32 bits, and of logits beyond: those of the weight in
    float32 are there where 32 bits hold them.  (bfloat16, as far as its own range goes.)"""
    if t == "bfloat16" and 2 * size * scale > 3e38:
        pytest.skip("past the range of bfloat16, which takes no factor")
    gen = seeded(11, len(t))
    x, w = rand(gen, (40, 64), t, std), rand(gen, (300, 64), t, min(1.0, 0.25 / (8 * std * scale)))
    tokens = torch.randint(0, 300, (40,), generator=gen).cuda()
    gp, gl = ((2 * torch.rand(40, generator=gen) - 1).cuda() * size for _ in range(2))
    gp[0], gl[0] = size, -size
    tokens[1], gp[1] = -1, math.nan
    r = ops.linear_logprobs(x, w, tokens, scale=scale)
    want = linear64(x, w, tokens, scale, gp, gl, t)
    assert want["dw"].abs().max() < 3e38
    g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl, scale=scale,
                                 out=(torch.empty_like(x), torch.empty(w.shape, device="cuda")))
    close(g.weight, want["dw"], want["edw"], "float32")


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_linear_logprobs_gradient_of_a_row_that_is_no_number(ops, bad):
    """float16: it leaves the other rows' gradients as they would be beside a row of zeros."""
    x, w, tokens, gp, gl = linear_operands("float16", 30, 64, 200)
    gp, gl = gp * 1e-6, gl * 1e-6
    r = ops.linear_logprobs(x, w, tokens)
    gp[5], gl[5] = 0.0, 0.0
    want = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl)
    gl[5] = bad
    got = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl)
    rest = torch.arange(30) != 5
    assert torch.equal(got.x[rest], want.x[rest]) and not got.x[5].isfinite().any() and want.x[rest].count_nonzero() > 0


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("width", [64, 1024, 4096, 16384])
@pytest.mark.parametrize("place", ["first", "last", "spread"])
def test_linear_logprobs_of_exact_logits(ops, t, width, place):
    """Logits of 16 terms, whole numbers that 24 bits hold in any order of addition: nothing is lost, whatever
    the width is.  One is 16 and more ahead of the others, so the log of the sum is below 500 e^-16 < 2^-14 and off
    by no more than 2^-22 (an exponential's error and a rounding of a sum that begins with 1); beside it,
    lse and logp are rounded once."""
    gen = seeded(width, len(t))
    at = torch.tensor({"first": list(range(16)), "last": list(range(width - 16, width)),
                       "spread": list(range(3, width, width // 16))}[place])
    x, w = torch.zeros(40, width, dtype=torch.double), torch.randint(-4, 5, (500, width), generator=gen).double()
    x[:, at] = torch.randint(1, 5, (40, 16), generator=gen).double()
    x[:, at[0]], w[0], w[0, at[0]] = 4.0, 0.0, 64.0
    x, w = x.to(dtype(t)).cuda(), w.to(dtype(t)).cuda()
    z = x.double() @ w.double().T
    top, second = z.topk(2, -1).values.T
    assert (top == 256).all() and float(second.max()) <= 240
    tokens = torch.randint(0, 500, (40,), generator=gen).cuda()
    tokens[:20] = 0
    r = ops.linear_logprobs(x, w, tokens)
    lse = torch.logsumexp(z, -1)
    close(r.lse, lse, 2.0 ** -22, "float32")
    close(r.logp, z[torch.arange(40, device="cuda"), tokens] - lse, 2.0 ** -22, "float32")
    assert (r.stats[:, 0] == 256).all()


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("width", [1000, 4096])
def test_linear_logprobs_of_logits_that_grow_evenly(ops, t, width):
    """Terms of one sign, all along the width: truncation adds up, and takes away only: what lse is above its
    value comes from the exponents, their sum and the log, linear64's bound without that of logits."""
    gen = seeded(width)
    x = (0.5 + torch.rand(40, width, generator=gen)).to(dtype(t)).cuda()
    w = ((0.5 + torch.rand(300, width, generator=gen)) * 40 / width).to(dtype(t)).cuda()
    tokens = torch.randint(0, 300, (40,), generator=gen).cuda()
    want = linear64(x, w, tokens, 1.0)
    r = ops.linear_logprobs(x, w, tokens)
    close(r.lse, want["lse"], want["elf"], "float32")
    close(r.logp, want["logp"], want["elp"], "float32")
    top = (x.double() @ w.double().T).amax(-1)
    others = (math.log(300) + 4) * 4 + 300 / 64 + 64 + 4 * (want["lse"] + top)
    assert ((r.lse.double() - want["lse"]) <= 1.05 * E * others).all()


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("rows,width,vocab", [(1, 1537, 300), (9, 2500, 40000), (64, 1600, 1000), (130, 1601, 3000), (300, 4100, 700),
                                              (700, 2111, 9000), (2000, 1700, 20000)])
def test_linear_logprobs_of_wide_layers(ops, t, rows, width, vocab):
    """Widths that are summed in parts, on tiles of each size, one and several for a block; the same bits again."""
    x, w, tokens, gp, gl = linear_operands(t, rows, width, vocab)
    want = linear64(x, w, tokens, 1.0, gp, gl, t)
    r = ops.linear_logprobs(x, w, tokens)
    close(r.logp, want["logp"], want["elp"], "float32")
    close(r.lse, want["lse"], want["elf"], "float32")
    g = ops.linear_logprobs_grad(x, w, tokens, r.stats, gp, gl)
    close(g.x, want["dx"], want["edx"], t)
    close(g.weight, want["dw"], want["edw"], t)
    for _ in range(3):
        q = ops.linear_logprobs(x, w, tokens)
        h = ops.linear_logprobs_grad(x, w, tokens, q.stats, gp, gl)
        assert all(torch.equal(a, b) for a, b in zip((*r, *g), (*q, *h)))


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("width", [1000, 1536, 1600, 4096])
def test_linear_logprobs_of_a_row_that_is_sure(ops, t, width):
    """Logits of the backward pass are those of the forward one, bit for bit: where the token is far ahead, dz is 1 - 1 / sum,
    where the sum is 1 and the others' exponentials.  That is off by 4 E and by their share of it, which
    moves by at most twice a logit's error (tc) and by an exponential's (16 E, arguments below 16); p of
    another token by the same share; both are rounded once."""
    gen = seeded(width, len(t))
    w = rand(gen, (400, width), t, width ** -0.5)
    x = (12.0 * w[:40].double() + 0.01 * rand(gen, (40, width), "float32").double()).to(dtype(t))
    tokens = torch.arange(40, device="cuda")
    out = (torch.empty_like(x), torch.empty(w.shape, device="cuda"))
    r = ops.linear_logprobs(x, w, tokens)
    g = ops.linear_logprobs_grad(x, w, tokens, r.stats, torch.ones(40, device="cuda"), out=out)
    x, w = x.double(), w.double()
    p = torch.softmax(x @ w.T, -1)
    move = 2 * tc(width) * (x.abs() @ w.abs().T).amax(-1) + 16 * E
    d, ed = -p, p * move[:, None]
    rest = p.clone()
    rest[tokens, tokens] = 0
    miss = rest.sum(-1)
    assert 1e-4 < float(miss.min()) and float(miss.max()) < 2e-2
    d[tokens, tokens], ed[tokens, tokens] = miss, miss * move + 4 * E
    ed += U[t] * d.abs() + 2.0 ** -38
    close(g.weight, d.T @ x, ed.T @ x.abs() + tc(40) * (d.abs().T @ x.abs()), "float32")


# ------------------------------------------------------------------ gated feed-forward blocks

@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [2, 40])
def test_feed_forward_activations_relative_to_their_size(ops, t, act, rows):
    """act(z) u and its gradients one element at a time, far out on the negative side too.  Products have one
    term each and are exact, so what is left is the activation's share p of z in 32 bits, relative to
    itself: an exponential whose argument, of size c, is off by 3 E c at most (its own roundings; gelu_tanh's
    argument is a cubic, 3 E more), 2^-22 for it, and 16 E for the sum and quotient or the polynomial (its
    fit: 2 E)."""
    n = 512
    z = torch.linspace(-9, 9, n).to(dtype(t))
    x, wu, wd = torch.zeros(rows, n, dtype=dtype(t)), torch.zeros(n, n, dtype=dtype(t)), torch.eye(n, dtype=dtype(t))
    wg = torch.zeros(n, n, dtype=dtype(t))
    x[:, 0], wg[:, 0], wu[:, 0] = 1.0, z, 4096.0
    x, wg, wu, wd = (v.cuda() for v in (x, wg, wu, wd))
    z = z.double().cuda()
    if act == "silu":
        c, p, dp = z.abs(), torch.sigmoid(z), torch.sigmoid(z) * torch.sigmoid(-z)
    elif act == "gelu":
        c, p, dp = z * z / 2, torch.exp(torch.special.log_ndtr(z)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        k = math.sqrt(8 / math.pi)
        c = k * (z + 0.044715 * z ** 3)
        p, dp = torch.sigmoid(c), torch.sigmoid(c) * torch.sigmoid(-c) * k * (1 + 3 * 0.044715 * z * z)
        c = 2 * c.abs()
    off = (3 * c + 20) * E
    got = ops.feed_forward(x, wg, wu, wd, act=act, keep=True)
    assert torch.equal(got.gate[0].double(), z) and (got.up[0] == 4096).all()
    h = 4096 * z * p
    close(got.y[0], h, off * h.abs(), t)
    assert all(torch.equal(got.y[0], v) for v in got.y)
    dy = torch.zeros_like(x)
    dy[0] = 1.0
    out = (torch.empty_like(x), *(torch.empty(n, n, device="cuda") for _ in range(3)))
    g = ops.feed_forward_grad(dy, x, wg, wu, wd, got.gate, got.up, act=act, out=out)
    close(g.w_up[:, 0], z * p, off * (z * p).abs() + U[t] * (z * p).abs(), t)
    slope = 4096 * (p + z * dp)
    close(g.w_gate[:, 0], slope, off * 4096 * (p + (z * dp).abs()) + U[t] * slope.abs(), t)
    down = g.w_down.double()
    assert torch.equal(down, down[:1].expand(n, n))
    close(g.w_down[0], h, off * h.abs() + U[t] * h.abs(), t)


# ------------------------------------------------------------------ graphs

@pytest.mark.parametrize("which", range(3))
def test_first_call_of_clipping_can_be_captured(which):
    """In a process of its own, with nothing run before: few arrays in place and into others, and many."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from ad_b200 import ops
torch.manual_seed(0)
grads = [torch.randn(70, 11, device="cuda"), torch.randn(999, device="cuda").bfloat16()]
if %d == 2:
    grads = [torch.randn(33, device="cuda") for _ in range(100)]
out = grads if %d == 0 else [torch.empty_like(g) for g in grads]
kept = [g.clone() for g in grads]
want = torch.cat([g.double().reshape(-1) for g in grads]).norm()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    norm = ops.clip_norm(grads, 0.5, out=out)
for _ in range(2):
    for a, b in zip(grads, kept):
        a.copy_(b)
    g.replay()
    assert abs(float(norm) / float(want) - 1) < 1e-6
    for a, b in zip(out, kept):
        s = (b.double() * (0.5 / want)).to(b.dtype)
        assert torch.allclose(a, s, rtol=2 * torch.finfo(b.dtype).eps, atol=0)
""" % (which, which)
    r = subprocess.run([sys.executable, "-c", code], cwd=root, env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


def test_linear_logprobs_workspaces(ops):
    """As documented: logits' gradients of a piece of the vocabulary, at most 1.5 times 2^28 elements (and a round to 256
    columns), or 2 KB to 4 KB a row where rows are many; the sums of x's gradient in 32 bits beside several pieces; 2 x
    74 tiles of partial sums.  Forward: two floats for each row and 256 or fewer tokens."""
    for rows, width, vocab in ((1, 64, 100), (2047, 1024, 50001), (8192, 2048, 65537), (9000, 24, 50003), (1 << 18, 64, 131072),
                               (1 << 20, 512, 50000), (1 << 24, 64, 200000), (1 << 24, 64, 1)):
        x, w = (ops.DeviceArray(1 << 20, s, "bfloat16") for s in ((rows, width), (vocab, width)))
        dz = min(max(3 * 2 ** 28 + 512 * rows, 4096 * rows), 2 * rows * (vocab + 8))
        sums = 4 * rows * width if rows * vocab > 2 ** 28 else 0
        need = ops.linear_logprobs_workspace(x, w, True)
        assert need <= dz + sums + 2 * 74 * 4 * 256 * 256 + 4096, (rows, width, vocab, need)
        assert ops.linear_logprobs_workspace(x, w) <= 8 * rows * (vocab // 64 + 2) + 4096

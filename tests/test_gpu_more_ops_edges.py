"""Embeddings, feed-forward blocks, log probabilities of a linear layer and gradient clipping at the edges of
what they take (B200 only).  The 64-bit implementations and the bounds' derivation are those of
test_gpu_more_ops."""
import math

import pytest

from .test_gpu_more_ops import HALVES, close, linear64, linear_operands
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

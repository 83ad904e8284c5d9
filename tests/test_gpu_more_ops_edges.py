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

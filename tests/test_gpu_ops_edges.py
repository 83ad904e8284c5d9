"""Operators of language models at the edges of what they take (B200 only).  The 64-bit
implementations and the bounds' derivation are those of test_gpu_ops."""
import math

import pytest

from .test_gpu_ops import N_SOFT, check_logprobs, dtype, logprobs64, rand, seeded, within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from ad_b200 import ops as o
    return o


@pytest.mark.parametrize("t", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [0.7, 1.0, 1.25])
@pytest.mark.parametrize("base", [3e4, 5e5, 2e6, 1e8, 1e9, 1e10, 1e12, 1e20, 9e29, 1.1e30, 1e37])
@pytest.mark.parametrize("vocab", [50, 20000])
def test_token_logprobs_of_large_logits(ops, t, scale, base, vocab):
    """Rows that are large throughout, rows masked with a finite value that is not the type's lowest, and
    rows of such a mask alone."""
    gen = seeded(vocab, len(t), math.log2(base), 100 * scale)
    logits = rand(gen, (12, vocab), t, 2.0)
    for r, b in ((0, base), (4, -base)):
        logits[r] = b                                    # nothing but the mask
        logits[r + 1, :vocab - 9] = b                    # the mask first (or far ahead of the rest)
        logits[r + 2, 5::3] = b                          # in between
        steps = torch.randint(0, 4, (vocab,), generator=gen)
        near = torch.full((vocab,), b, dtype=dtype(t))   # some neighbouring values
        spacing = torch.nextafter(near.abs().double().to(dtype(t)), torch.tensor(math.inf, dtype=dtype(t))) - near.abs()
        logits[r + 3] = (near.double() + steps * spacing.double()).to(dtype(t)).cuda()
    logits[8, ::2], logits[8, 1::2] = base, -base        # both signs
    logits[9] = -math.inf
    logits[9, 3] = -base                                 # one value left
    logits[10, :vocab // 2], logits[10, vocab // 2:] = -base, -base / 2
    tokens = torch.randint(0, vocab, (12,), generator=gen)
    tokens[9] = 3
    g, e = rand(gen, (12,), "float32"), rand(gen, (12,), "float32", 0.1)
    r, _ = check_logprobs(ops, logits, tokens.cuda(), scale, 7, t, g, e)
    lse = logprobs64(logits, tokens, scale, 0)["lse"]
    within(r.stats[:, 3].cpu(), lse, lse.abs() + 4 + math.log(vocab), N_SOFT, "float32")

"""A small causal language model trained with the operators of ``ad_b200.ops``.

    python examples/lm_step.py [steps]

Two blocks of attention and a ReLU feed-forward.  Between the matrix products (torch's) stand the
operators: ``block_norm`` joins each block's output to the residual stream (norm after the block,
sigmoid gate, residual scale, norm before the next block), ``rotary`` turns queries and keys,
``token_logprobs`` gives the loss, and ``orthogonalize`` makes the update of the matrices from their
momentum.  Tables, embedding and norm weights take plain SGD.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ad_b200 import ops  # noqa: E402


class Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, positions):
        ctx.save_for_backward(cos, sin, positions)
        return ops.rotary(q, k, cos, sin, positions)

    @staticmethod
    def backward(ctx, dq, dk):
        return (*ops.rotary(dq.contiguous(), dk.contiguous(), *ctx.saved_tensors, inverse=True), None, None, None)


class BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, after, before, gate):
        h, y, stats = ops.block_norm(x, z, after, before, gate=gate, gate_sigmoid=True)
        ctx.save_for_backward(x, z, after, before, gate, stats)
        return h, y

    @staticmethod
    def backward(ctx, dh, dy):
        x, z, after, before, gate, stats = ctx.saved_tensors
        g = ops.block_norm_grad(dh.contiguous(), dy.contiguous(), x, z, after, before, stats, gate=gate,
                                gate_sigmoid=True)
        return g.x, g.z, g.after_weight, g.before_weight, g.gate


class TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens):
        r = ops.token_logprobs(logits, tokens)
        ctx.save_for_backward(logits, tokens, r.stats)
        return r.logp, r.entropy

    @staticmethod
    def backward(ctx, g_logp, g_entropy):
        logits, tokens, stats = ctx.saved_tensors
        return ops.token_logprobs_grad(logits, tokens, stats, g_logp.contiguous(), g_entropy.contiguous()), None


class Model:
    def __init__(self, vocab, width, heads, hidden, layers, length, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(rows, cols):
            return (torch.randn(rows, cols, device="cuda", generator=gen) / cols ** 0.5).requires_grad_()

        self.heads, self.dim = heads, width // heads
        self.matrices = [dict(qkv=matrix(3 * width, width), out=matrix(width, width), up=matrix(hidden, width),
                              down=matrix(width, hidden)) for _ in range(layers)]
        self.embedding = (0.5 * torch.randn(vocab, width, device="cuda", generator=gen)).requires_grad_()
        # a norm after and one before, and a gate, for each of a layer's two blocks
        self.vectors = [[torch.ones(width, device="cuda").requires_grad_() for _ in range(4)] +
                        [torch.zeros(1, width, device="cuda").requires_grad_() for _ in range(2)] for _ in range(layers)]
        self.first = torch.ones(width, device="cuda").requires_grad_()
        self.cos, self.sin = (torch.from_numpy(t).cuda() for t in ops.rotary_table(length, self.dim))
        self.positions = torch.arange(length, device="cuda")
        self.mask = torch.full((length, length), float("-inf"), device="cuda").triu(1)
        self.momentum = {}

    def loss(self, tokens):
        batch, length = tokens.shape
        x = self.embedding[tokens].reshape(batch * length, -1)
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * self.first
        for m, (a1, b1, a2, b2, g1, g2) in zip(self.matrices, self.vectors):
            q, k, v = (t.reshape(batch, length, self.heads, self.dim) for t in (y @ m["qkv"].T).chunk(3, -1))
            q, k = Rotary.apply(q.contiguous(), k.contiguous(), self.cos, self.sin, self.positions)
            scores = torch.einsum("bthd,bshd->bhts", q, k) / self.dim ** 0.5 + self.mask
            mixed = torch.einsum("bhts,bshd->bthd", scores.softmax(-1), v).reshape(batch * length, -1)
            x, y = BlockNorm.apply(x, mixed @ m["out"].T, a1, b1, g1)
            x, y = BlockNorm.apply(x, torch.relu(y @ m["up"].T) @ m["down"].T, a2, b2, g2)
        target = torch.cat((tokens[:, 1:], torch.full_like(tokens[:, :1], -1)), 1)  # the last position has none
        logp, _ = TokenLogprobs.apply(y @ self.embedding.T, target.reshape(-1))
        return -logp.sum() / (batch * (length - 1))

    def step(self, tokens, rate=0.02):
        loss = self.loss(tokens)
        loss.backward()
        with torch.no_grad():
            for name in self.matrices[0]:  # the layers' matrices of one shape together
                grad = torch.stack([m[name].grad for m in self.matrices])
                mom = self.momentum[name] = 0.9 * self.momentum.get(name, 0.0) + grad
                for m, update in zip(self.matrices, ops.orthogonalize(mom)):
                    m[name] -= rate * update
                    m[name].grad = None
            for p in (self.embedding, self.first, *(v for layer in self.vectors for v in layer)):
                p -= 10 * rate * p.grad
                p.grad = None
        return float(loss.detach())


def main(steps=40):
    """Sequences that count up by a step of their own: from the second token on they can be foretold."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    vocab, length = 61, 32
    model = Model(vocab, width=64, heads=4, hidden=256, layers=2, length=length)
    losses = []
    for k in range(steps):
        start = torch.randint(0, vocab, (64, 1), device="cuda", generator=gen)
        by = torch.randint(1, 5, (64, 1), device="cuda", generator=gen)
        tokens = (start + by * torch.arange(length, device="cuda")) % vocab
        losses.append(model.step(tokens))
        if k % 10 == 0 or k + 1 == steps:
            print(f"step {k}: loss {losses[-1]:.3f}")
    return losses


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 40)

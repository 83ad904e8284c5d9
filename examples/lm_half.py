"""A small causal language model in bfloat16, its matrices' products in the operators of ``ad_b200.ops``.

    python examples/lm_half.py [steps]

Attention is torch's; around it ``embed``, ``rotary``, ``block_norm``, the gated ``feed_forward`` and
``linear_logprobs``, which is the output layer and the loss in one: logits of a large vocabulary are never in
memory.  The table is the embedding's and the output layer's, so that it has two gradients.  Weights are kept in
float32 and rounded for each step; ``clip_norm`` scales the gradients, ``orthogonalize`` makes the matrices' update.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from ad_b200 import ops  # noqa: E402
from lm_step import BlockNorm, Embed, Rotary  # noqa: E402


class FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down):
        r = ops.feed_forward(x, w_gate, w_up, w_down, keep=True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, r.gate, r.up)
        return r.y

    @staticmethod
    def backward(ctx, dy):
        return tuple(ops.feed_forward_grad(dy.contiguous(), *ctx.saved_tensors))


class LinearLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, tokens):
        r = ops.linear_logprobs(x, weight, tokens)
        ctx.save_for_backward(x, weight, tokens, r.stats)
        return r.logp, r.lse

    @staticmethod
    def backward(ctx, g_logp, g_lse):
        return (*ops.linear_logprobs_grad(*ctx.saved_tensors, g_logp.contiguous(), g_lse.contiguous()), None)


class Model:
    def __init__(self, vocab, width, heads, hidden, layers, length, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(rows, cols, std=None):
            return torch.randn(rows, cols, device="cuda", generator=gen) * (std or cols ** -0.5)

        self.heads, self.dim, self.layers = heads, width // heads, layers
        self.weights = {"table": matrix(vocab, width, 0.5)}
        for i in range(layers):
            for name, rows, cols in (("qkv", 3 * width, width), ("out", width, width), ("gate", hidden, width),
                                     ("up", hidden, width), ("down", width, hidden)):
                self.weights[f"{name}{i}"] = matrix(rows, cols)
        # norms after and before the two blocks of a layer, gates of both, and the first norm
        self.norms = {f"{name}{i}": torch.ones(width, device="cuda") for i in range(layers) for name in ("a1", "b1", "a2", "b2")}
        self.gates = {f"{name}{i}": torch.zeros(1, width, device="cuda") for i in range(layers) for name in ("g1", "g2")}
        self.norms["first"] = torch.ones(width, device="cuda")
        self.cos, self.sin = (torch.from_numpy(t).cuda() for t in ops.rotary_table(length, self.dim))
        self.positions = torch.arange(length, device="cuda")
        self.mask = torch.full((length, length), float("-inf"), device="cuda").triu(1)

    def leaves(self):
        """The step's own copies: matrices and gates in bfloat16, norm weights as they are."""
        p = {k: v.bfloat16() for k, v in (*self.weights.items(), *self.gates.items())}
        p.update({k: v.clone() for k, v in self.norms.items()})
        return {k: v.requires_grad_() for k, v in p.items()}

    def loss(self, tokens, p):
        batch, length = tokens.shape
        x = Embed.apply(tokens, p["table"]).reshape(batch * length, -1)
        f = x.float()
        y = (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5) * p["first"]).bfloat16()
        for i in range(self.layers):
            q, k, v = (t.reshape(batch, length, self.heads, self.dim) for t in (y @ p[f"qkv{i}"].T).chunk(3, -1))
            q, k = Rotary.apply(q.contiguous(), k.contiguous(), self.cos, self.sin, self.positions)
            scores = torch.einsum("bthd,bshd->bhts", q, k).float() / self.dim ** 0.5 + self.mask
            mixed = torch.einsum("bhts,bshd->bthd", scores.softmax(-1).bfloat16(), v).reshape(batch * length, -1)
            x, y = BlockNorm.apply(x, mixed @ p[f"out{i}"].T, p[f"a1{i}"], p[f"b1{i}"], p[f"g1{i}"])
            z = FeedForward.apply(y, p[f"gate{i}"], p[f"up{i}"], p[f"down{i}"])
            x, y = BlockNorm.apply(x, z, p[f"a2{i}"], p[f"b2{i}"], p[f"g2{i}"])
        target = torch.cat((tokens[:, 1:], torch.full_like(tokens[:, :1], -1)), 1)  # the last position has none
        logp, _ = LinearLogprobs.apply(y, p["table"], target.reshape(-1))
        return -logp.sum() / (batch * (length - 1))

    def step(self, tokens, rate=0.02, most=1.0):
        p = self.leaves()
        loss = self.loss(tokens, p)
        loss.backward()
        ops.clip_norm([v.grad for v in p.values()], most)
        for name, w in self.weights.items():
            w -= rate * ops.orthogonalize(p[name].grad) if name != "table" else 10 * rate * p[name].grad.float()
        for some in (self.norms, self.gates):
            for name, w in some.items():
                w -= 10 * rate * p[name].grad.float()
        return float(loss.detach())


def main(steps=40):
    """Sequences that count up by a step of their own: from the second token on they can be foretold."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    vocab, length = 61, 32
    model = Model(vocab, width=64, heads=4, hidden=160, layers=2, length=length)
    losses = []
    for k in range(steps):
        start = torch.randint(0, vocab, (64, 1), device="cuda", generator=gen)
        by = torch.randint(1, 5, (64, 1), device="cuda", generator=gen)
        losses.append(model.step((start + by * torch.arange(length, device="cuda")) % vocab))
        if k % 10 == 0 or k + 1 == steps:
            print(f"step {k}: loss {losses[-1]:.3f}")
    return losses


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 40)

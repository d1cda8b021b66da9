"""A small next-token model trained and asked with the layers of token models: norm with the residual's addition, log probabilities
with their gradient, AdamW over all tensors.

    python examples/token_model.py [--steps 200] [--bits 8|32]

The network: an embedding, blocks of norm -> product -> squared positive part -> product on a residual stream, a last norm and the
product with the logits' weights.  The products are torch's; everything between them is this library's, forward and
backward, and no graph of operations is recorded: a block's backward pass is written out, as a layer's of the engine is.
Weights are kept in fp32 with a copy in bfloat16 for the products; states of the optimiser in 8 or 32 bits.
The data: sequences in which a token decides the next one nine times out of ten.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from pixienn_amd import ops  # noqa: E402

BF16 = torch.bfloat16


class TokenModel:
    def __init__(self, vocab=512, width=256, wide=1024, blocks=2, bits=8, seed=0):
        self.vocab, self.width, self.blocks = vocab, width, blocks
        g = torch.Generator(device="cuda").manual_seed(seed)
        matrix = lambda rows, columns, std: torch.randn(rows, columns, device="cuda", generator=g) * std  # noqa: E731
        self.w = {"embedding": matrix(vocab, width, 1.0), "head": matrix(vocab, width, 0.3 * width ** -0.5), "norm": torch.ones(width, device="cuda")}
        for b in range(blocks):
            self.w.update({"norm%d" % b: torch.ones(width, device="cuda"), "up%d" % b: matrix(wide, width, width ** -0.5),
                           "down%d" % b: matrix(width, wide, wide ** -0.5 / blocks)})
        names = list(self.w)
        self.copy = {k: self.w[k].to(BF16) for k in names}
        # the updates: gradients of the log likelihood, which the optimiser adds.  A norm's come in fp32, a product's in bfloat16
        self.d = {k: torch.zeros_like(self.w[k] if k.startswith("norm") else self.copy[k]) for k in names}
        self.states = ops.adamw_states([self.w[k] for k in names], bits)
        self.table = ops.AdamwTable([self.w[k] for k in names], [self.d[k] for k in names], copies=[self.copy[k] for k in names],
                                    apply_decay=[self.w[k].dim() == 2 for k in names], **self.states)
        self.norm = torch.zeros(1, device="cuda")
        self.t = 0

    def _norm(self, name, x, residual=None):
        """(result, the sum that it is the norm of, its statistic)"""
        y, rstd = torch.empty_like(x), torch.empty(len(x), device="cuda")
        total = torch.empty_like(x) if residual is not None else x
        ops.rms_norm_forward(x, y, self.copy[name], residual=residual, sum=total if residual is not None else None, rstd=rstd)
        return y, total, rstd

    def logits(self, tokens, keep=None):
        h, branch = self.copy["embedding"][tokens], None
        for b in range(self.blocks):
            # the block's branch joins the stream in the next norm
            y, h, rstd = self._norm("norm%d" % b, h, branch)
            up = y @ self.copy["up%d" % b].t()
            active = up.clamp(min=0).square()
            branch = active @ self.copy["down%d" % b].t()
            if keep is not None:
                keep.append((y, h, rstd, up, active))
        y, h, rstd = self._norm("norm", h, branch)
        if keep is not None:
            keep.append((y, h, rstd))
        return y @ self.copy["head"].t()

    def gradients(self, tokens, targets):
        """Leaves the gradient of the mean log probability of `targets` in self.d; the mean itself."""
        keep = []
        logits = self.logits(tokens, keep)
        rows = len(tokens)
        weights = torch.full((rows,), 1.0 / rows, device="cuda")
        logp = torch.empty(rows, device="cuda")
        # the gradient takes the logits' place
        d_logits = ops.token_logprobs_forward_train(logits, targets, weights, logits, logp)
        y, h, rstd = keep.pop()
        torch.mm(d_logits.t(), y, out=self.d["head"])
        dy = d_logits @ self.copy["head"]
        d_stream = torch.empty_like(h)
        ops.rms_norm_backward(dy, h, self.copy["norm"], rstd, d_stream, self.d["norm"])
        for b in reversed(range(self.blocks)):
            y, h, rstd, up, active = keep.pop()
            torch.mm(d_stream.t(), active, out=self.d["down%d" % b])
            d_up = (d_stream @ self.copy["down%d" % b]) * (2 * up.clamp(min=0))
            torch.mm(d_up.t(), y, out=self.d["up%d" % b])
            # what goes through the block and what goes past it
            ops.rms_norm_backward(d_up @ self.copy["up%d" % b], h, self.copy["norm%d" % b], rstd, d_stream, self.d["norm%d" % b], dsum=d_stream)
        self.d["embedding"].zero_().index_add_(0, tokens, d_stream)
        return logp.mean()

    def step(self, tokens, targets, lr):
        mean = self.gradients(tokens, targets)
        self.t += 1
        self.table.update(self.t, lr, 0.9, 0.95, 1e-8, 0.01, max_norm=1.0, norm_out=self.norm, seed=self.t)
        return mean

    def ask(self, tokens, top=3):
        """For the next token: the most probable ones with their log probabilities, and the entropy.  The last norm's result is
        handed to the product in 8 bits, with a scale for each 128 values, as a product in 8 bits would take it."""
        keep = []
        self.logits(tokens, keep)
        h = keep[-1][1]
        q = torch.empty(h.shape, device="cuda", dtype=torch.float8_e4m3fn)
        scales = torch.empty(len(h), -(-self.width // 128), device="cuda")
        ops.rms_norm_forward(h, q, self.copy["norm"], scales=scales, group=128)
        y = (q.float() * scales.repeat_interleave(128, 1)[:, :self.width]).to(BF16)
        logits = y @ self.copy["head"].t()
        best, ids = torch.empty(len(h), top, device="cuda"), torch.empty(len(h), top, device="cuda", dtype=torch.int32)
        entropy = torch.empty(len(h), device="cuda")
        ops.token_logprobs_forward(logits, None, None, entropy=entropy, top_logp=best, top_ids=ids)
        return ids, best, entropy


def batch(vocab, rows, generator):
    """Tokens and what follows them: 5 t + 7 nine times out of ten, anything otherwise."""
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=generator)
    follows = (5 * tokens + 7) % vocab
    other = torch.randint(0, vocab, (rows,), device="cuda", generator=generator)
    return tokens, torch.where(torch.rand(rows, device="cuda", generator=generator) < 0.9, follows, other)


def train(steps=200, bits=8, rows=4096, lr=3e-3, say=None, **size):
    model = TokenModel(bits=bits, **size)
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(steps):
        mean = model.step(*batch(model.vocab, rows, g), lr * min(1.0, (i + 1) / 10))
        if say and (i % 20 == 0 or i + 1 == steps):
            say("step %4d  mean log probability %.4f  norm of the gradients %.3f" % (i, float(mean), float(model.norm)))
    return model, float(mean)


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--bits", type=int, choices=(8, 32), default=8)
    a = parser.parse_args()
    model, _ = train(a.steps, a.bits, say=lambda s: print(s, flush=True))
    tokens = torch.tensor([1, 100, 511], device="cuda")
    ids, best, entropy = model.ask(tokens)
    for t, i, p, h in zip(tokens.tolist(), ids.tolist(), best.exp().tolist(), entropy.tolist()):
        print("after %3d (expected %3d): %s  entropy %.2f" % (t, (5 * t + 7) % model.vocab, ", ".join("%d %.3f" % x for x in zip(i, p)), h))


if __name__ == "__main__":
    main()

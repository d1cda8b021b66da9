"""A small model of sequences trained and asked with the layers of token models: embeddings by token, layer norm with the residual's
addition, a gated recurrence along each sequence, log probabilities with their gradient, AdamW over all tensors, and beam search.

    python examples/sequence_model.py [--steps 300] [--beams 4]

The network: an embedding, blocks of norm -> product -> gated recurrence -> product on a residual stream, a last norm, and the product
with the embedding's table, which both ends share.  The products are torch's; everything between them is this library's, forward and
backward.  Sequences of any lengths lie one behind the other, without padding.  When it answers, a prompt leaves a state of one row for each
block; every further token is one step from there, for all beams of all prompts at once, captured once and replayed.
The data: the first token of a sequence says by how much the others rise, so that the next one follows from the last one and the first.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from pixienn_amd import ops  # noqa: E402

BF16 = torch.bfloat16


class SequenceModel:
    def __init__(self, vocab=64, width=256, blocks=2, bits=32, seed=0):
        self.vocab, self.width, self.blocks = vocab, width, blocks
        self.scale = width ** 0.5                       # the table's rows are short, as the logits' product wants them
        g = torch.Generator(device="cuda").manual_seed(seed)
        matrix = lambda rows, columns, std: torch.randn(rows, columns, device="cuda", generator=g) * std  # noqa: E731
        self.w = {"embedding": matrix(vocab, width, width ** -0.5)}
        for name in ["norm%d" % b for b in range(blocks)] + ["norm"]:
            self.w.update({name: torch.ones(width, device="cuda"), name + "_bias": torch.zeros(width, device="cuda")})
        for b in range(blocks):
            self.w.update({"in%d" % b: matrix(3 * width, width, width ** -0.5), "out%d" % b: matrix(width, width, 2 * width ** -0.5)})
        names = list(self.w)
        self.copy = {k: self.w[k].to(BF16) for k in names}
        # the updates: gradients of the log likelihood, which the optimiser adds.  A norm's come in fp32, a product's in bfloat16
        self.d = {k: torch.zeros_like(self.w[k] if k.startswith("norm") else self.copy[k]) for k in names}
        self.table = ops.AdamwTable([self.w[k] for k in names], [self.d[k] for k in names], copies=[self.copy[k] for k in names],
                                    apply_decay=[self.w[k].dim() == 2 for k in names], **ops.adamw_states([self.w[k] for k in names], bits))
        self.t = 0

    def _norm(self, name, x, residual=None):
        """(result, the sum that it is the norm of, its statistics)"""
        y, mean, rstd = torch.empty_like(x), torch.empty(len(x), device="cuda"), torch.empty(len(x), device="cuda")
        total = torch.empty_like(x) if residual is not None else x
        ops.layer_norm_forward(x, y, self.copy[name], self.copy[name + "_bias"], residual, total if residual is not None else None, mean, rstd)
        return y, total, mean, rstd

    def _parts(self, p):
        """The recurrence's input, update and gate: the columns of one product."""
        return p[:, :self.width], p[:, self.width:2 * self.width], p[:, 2 * self.width:]

    def _logits(self, tokens, recurrence, keep=None):
        h, branch = torch.empty(len(tokens), self.width, device="cuda", dtype=BF16), None
        ops.embedding_forward(self.copy["embedding"], tokens, h, self.scale)
        for b in range(self.blocks):
            y, h, mean, rstd = self._norm("norm%d" % b, h, branch)
            p = y @ self.copy["in%d" % b].t()
            mixed = torch.empty_like(h)
            extra = recurrence(b, *self._parts(p), mixed)
            branch = mixed @ self.copy["out%d" % b].t()
            if keep is not None:
                keep.append((y, h, mean, rstd, p, mixed, extra))
        y, h, mean, rstd = self._norm("norm", h, branch)
        if keep is not None:
            keep.append((y, h, mean, rstd))
        return y @ self.copy["embedding"].t()

    def logits(self, tokens, starts, states=None, slots=None, keep=None):
        """Of every token of the sequences that begin at `starts`.  states: a tensor for each block, in whose rows slots[s] the
        sequences' last states are left."""
        def recurrence(b, x, update, gate, y):
            saved = ops.gated_scan_saved_like(x) if keep is not None else None
            ops.gated_scan_forward(x, update, y, gate, starts, final=states[b] if states else None, slots=slots, saved=saved)
            return saved
        return self._logits(tokens, recurrence, keep)

    def step_logits(self, tokens, states):
        """Of one more token for every row of the states, which move on by it."""
        return self._logits(tokens, lambda b, x, update, gate, y: ops.gated_scan_step(x, update, y, states[b], gate))

    def gradients(self, tokens, targets, starts):
        """Leaves the gradient of the mean log probability of `targets` in self.d; the mean itself.  A target outside the
        vocabulary is none."""
        keep = []
        logits = self.logits(tokens, starts, keep=keep)
        rows = len(tokens)
        weights, logp = torch.full((rows,), 1.0 / rows, device="cuda"), torch.empty(rows, device="cuda")
        d_logits = ops.token_logprobs_forward_train(logits, targets, weights, logits, logp)
        y, h, mean, rstd = keep.pop()
        torch.mm(d_logits.t(), y, out=self.d["embedding"])
        d_stream = torch.empty_like(h)
        ops.layer_norm_backward(d_logits @ self.copy["embedding"], h, self.copy["norm"], mean, rstd, d_stream, self.d["norm"], self.d["norm_bias"])
        for b in reversed(range(self.blocks)):
            y, h, mean, rstd, p, mixed, saved = keep.pop()
            torch.mm(d_stream.t(), mixed, out=self.d["out%d" % b])
            # the gradients take the places of what they are gradients of
            x, update, gate = self._parts(p)
            ops.gated_scan_backward(d_stream @ self.copy["out%d" % b], x, update, saved, x, update, gate, gate, starts)
            torch.mm(p.t(), y, out=self.d["in%d" % b])
            name = "norm%d" % b
            ops.layer_norm_backward(p @ self.copy["in%d" % b], h, self.copy[name], mean, rstd, d_stream, self.d[name], self.d[name + "_bias"],
                                    dsum=d_stream)
        # the table's share as an embedding joins that of the logits' product
        ops.embedding_backward(d_stream, tokens, self.d["embedding"], self.scale, accumulate=True)
        return logp.mean()

    def train_step(self, tokens, targets, starts, lr):
        mean = self.gradients(tokens, targets, starts)
        self.t += 1
        self.table.update(self.t, lr, 0.9, 0.95, 1e-8, 0.01, max_norm=1.0, seed=self.t)
        return mean


class Search:
    """Beam search from a model's prompts: `batch` of them with `beams` beams each, up to `longest` tokens behind the prompt."""

    def __init__(self, model, batch, beams, longest, end_token=-1, captured=True):
        self.model, self.batch, self.beams, self.longest, self.end_token = model, batch, beams, longest, end_token
        rows = batch * beams
        self.states = [torch.zeros(rows, model.width, device="cuda") for _ in range(model.blocks)]
        self.scores = torch.zeros(batch, beams, device="cuda")
        self.parents, self.tokens = (torch.zeros(batch, beams, device="cuda", dtype=torch.int32) for _ in range(2))
        self.ended = torch.zeros(batch, beams, device="cuda", dtype=torch.bool)
        self.history = torch.full((rows, longest), -1, device="cuda", dtype=torch.int32)
        self.place = torch.zeros(1, device="cuda", dtype=torch.int64)
        self.logits = torch.zeros(rows, model.vocab, device="cuda", dtype=BF16)
        self.space = torch.empty(ops.beam_select_workspace_bytes(batch, beams, model.vocab, beams) // 4 + 1, device="cuda")
        self.first = torch.arange(batch, device="cuda", dtype=torch.int32) * beams       # a prompt is its first beam's
        self.captured, self.graph = captured, None

    def _choose(self):
        ops.beam_select(self.logits, self.scores, self.scores, self.parents, self.tokens, self.ended, self.end_token, workspace=self.space)
        ops.beam_reorder([*self.states, self.history, self.ended.view(-1)], self.parents)
        self.history.index_copy_(1, self.place, self.tokens.view(-1, 1))
        self.place += 1
        self.ended |= self.tokens == self.end_token

    def _step(self):
        self.logits.copy_(self.model.step_logits(self.tokens.view(-1), self.states))
        self._choose()

    def _replay(self):
        if not self.captured:
            return self._step()
        if self.graph is None:
            # a pass outside the graph first, and what it changed put back: libraries prepare themselves in their first call
            changed = [*self.states, self.scores, self.parents, self.tokens, self.ended, self.history, self.place]
            before = [t.clone() for t in changed]
            self._step()
            for t, b in zip(changed, before):
                t.copy_(b)
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self._step()
        self.graph.replay()

    def run(self, prompts, count=None):
        """prompts: lists of tokens.  (tokens [batch, beams, longest], -1 behind the last one; their log probabilities [batch, beams])"""
        tokens = torch.tensor([t for p in prompts for t in p], device="cuda", dtype=torch.int32)
        ends = [0]
        for p in prompts:
            ends.append(ends[-1] + len(p))
        starts = torch.tensor(ends, device="cuda", dtype=torch.int32)
        logits = self.model.logits(tokens, starts, self.states, self.first)
        self.logits.zero_()
        self.logits[self.first.long()] = logits[starts[1:].long() - 1]
        # one beam to begin with: the others have no score, and all take their places behind it
        self.scores.fill_(float("-inf"))
        self.scores[:, 0] = 0
        self.ended.zero_()
        self.history.fill_(-1)
        self.place.zero_()
        self._choose()
        for _ in range((count or self.longest) - 1):
            self._replay()
        return self.history.view(self.batch, self.beams, self.longest), self.scores


def sequences(vocab, count, longest, generator):
    """(tokens, targets, starts): sequences of 2 to `longest` tokens that rise by their first one; what follows a sequence's first
    and last token is not asked for."""
    lengths = torch.randint(2, longest + 1, (count,), device="cuda", generator=generator)
    starts = torch.zeros(count + 1, device="cuda", dtype=torch.int32)
    starts[1:] = lengths.cumsum(0)
    rise = torch.randint(1, vocab, (count,), device="cuda", generator=generator)
    second = torch.randint(0, vocab, (count,), device="cuda", generator=generator)
    which = torch.repeat_interleave(torch.arange(count, device="cuda"), lengths)
    place = torch.arange(len(which), device="cuda") - starts[:-1].long()[which]
    tokens = torch.where(place == 0, rise[which], (second[which] + (place - 1) * rise[which]) % vocab)
    targets = torch.cat([tokens[1:], tokens[:1]])
    targets[(place == 0) | (place == lengths[which] - 1)] = -1
    return tokens, targets, starts


def train(steps=300, count=256, longest=24, lr=3e-3, say=None, **size):
    model = SequenceModel(**size)
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(steps):
        mean = model.train_step(*sequences(model.vocab, count, longest, g), lr * min(1.0, (i + 1) / 20))
        if say and (i % 20 == 0 or i + 1 == steps):
            say("step %4d  mean log probability %.4f" % (i, float(mean)))
    return model


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=300)
    parser.add_argument("--beams", type=int, default=4)
    a = parser.parse_args()
    model = train(a.steps, say=lambda s: print(s, flush=True))
    prompts = [[5, 1, 6], [11, 40], [2, 60, 62, 0]]
    tokens, scores = Search(model, len(prompts), a.beams, 6).run(prompts)
    for p, t, s in zip(prompts, tokens.tolist(), scores.tolist()):
        print("after %s: " % p + ", ".join("%s %.3f" % x for x in zip(t, s)))


if __name__ == "__main__":
    main()

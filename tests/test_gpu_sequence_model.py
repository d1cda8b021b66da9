"""The example of a model of sequences: embeddings, layer norm, the gated recurrence, log probabilities and beam search as they are
used together.  Its gradients against those that autograd finds for the same network in 64 bits; the log probabilities of what a search
finds, step by step, against those of whole sequences; steps in a graph against eager ones."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "sequence_model.py")
    spec = importlib.util.spec_from_file_location("sequence_model", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def log_probabilities(model, w, tokens, starts):
    """Of every next token in 64 bits, on the CPU, from the weights w."""
    norm = lambda x, name: torch.nn.functional.layer_norm(x, (model.width,), w[name], w[name + "_bias"], 1e-5)  # noqa: E731
    h = w["embedding"][tokens.long().cpu()] * model.scale
    for b in range(model.blocks):
        x, update, gate = (norm(h, "norm%d" % b) @ w["in%d" % b].t()).chunk(3, 1)
        z, rows = torch.sigmoid(update), []
        for first, end in zip(starts.tolist(), starts.tolist()[1:]):
            state = torch.zeros(model.width, dtype=torch.float64)
            for t in range(first, end):
                state = state + z[t] * (x[t] - state)
                rows.append(state)
        h = h + (torch.stack(rows) * gate * torch.sigmoid(gate)) @ w["out%d" % b].t()
    return torch.log_softmax(norm(h, "norm") @ w["embedding"].t(), 1)


def weights(model):
    return {k: t.double().cpu().requires_grad_() for k, t in model.copy.items()}


SIZES = [dict(vocab=64, width=256, blocks=2), dict(vocab=101, width=72, blocks=3), dict(vocab=37, width=129, blocks=1)]


@pytest.mark.parametrize("size", SIZES)
def test_its_gradients_are_those_of_the_network(example, size):
    model = example.SequenceModel(**size)
    tokens, targets, starts = example.sequences(size["vocab"], 40, 24, torch.Generator(device="cuda").manual_seed(5))
    mean = float(model.gradients(tokens, targets, starts))
    w = weights(model)
    logs, asked = log_probabilities(model, w, tokens, starts), targets.cpu()
    want = torch.where(asked >= 0, logs[torch.arange(len(asked)), asked.clamp(min=0)], 0).mean()
    want.backward()
    # every value between two products is rounded to 2^-8 of itself, a few of them in a row
    assert abs(mean - float(want.detach())) < 0.02
    for name, t in w.items():
        got = model.d[name].double().cpu()
        assert float((got - t.grad).norm()) < 0.03 * float(t.grad.norm()), name


def test_it_trains_and_answers(example):
    model = example.train(3, count=32)
    tokens, scores = example.Search(model, 2, 3, 4).run([[5, 1, 6], [11, 40]])
    assert tokens.shape == (2, 3, 4) and bool(((tokens >= 0) & (tokens < model.vocab)).all()) and bool(scores.isfinite().all())


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("beams", [1, 4])
def test_what_a_search_finds_has_the_log_probability_that_it_says(example, size, beams):
    model = example.SequenceModel(seed=3, **size)
    prompts = [[5, 1, 6], [11], [2, 30, 32, 0, 7, 9, 35]]
    longest = 5
    tokens, scores = example.Search(model, len(prompts), beams, longest).run(prompts)
    w = {k: t.detach() for k, t in weights(model).items()}
    for i, prompt in enumerate(prompts):
        rows = [prompt + t for t in tokens[i].tolist()]
        assert len({tuple(r) for r in rows}) == beams
        assert scores[i].tolist() == sorted(scores[i].tolist(), reverse=True)
        flat, n = torch.tensor([t for r in rows for t in r]), len(prompt) + longest
        logs = log_probabilities(model, w, flat, torch.arange(beams + 1) * n).view(beams, n, -1)
        for k in range(beams):
            want = sum(float(logs[k, t - 1, rows[k][t]]) for t in range(len(prompt), n))
            # a logit of up to 4 is rounded by 2^-8 of itself, and so is every value on the way to it: 0.1 for each token of the five.
            # Another beam's state, or another prompt's, would be off by whole units
            assert abs(float(scores[i, k]) - want) < 0.1 * longest, (i, k)
        if beams == 1:
            # each token is the best one at its place, or as good as it to the roundings above
            for t in range(len(prompt), n):
                assert float(logs[0, t - 1, rows[0][t]]) > float(logs[0, t - 1].max()) - 0.2


def test_steps_in_a_graph_are_the_eager_ones(example):
    model = example.SequenceModel(seed=4)
    end = 17
    captured, eager = (example.Search(model, 3, 4, 8, end, captured=c) for c in (True, False))
    for prompts in [[[5, 1, 6], [11, 40], [2, 60, 62, 0]], [[1], [63] * 30, [9, 9]], [[17, 17], [0, 1], [3]]]:
        got, want = captured.run(prompts), eager.run(prompts)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for a, b in zip(captured.states, eager.states):
            assert torch.equal(a, b)
        # behind the token that ends a beam only that one follows
        ended = (got[0] == end).cumsum(2) > 0
        assert bool((got[0][ended] == end).all())

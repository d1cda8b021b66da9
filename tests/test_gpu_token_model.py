"""The example of a token model: its gradients against those that autograd finds for the same network in 64 bits, and what it learns
with states in 32 and in 8 bits."""
import importlib.util
import math
import os

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "token_model.py")
    spec = importlib.util.spec_from_file_location("token_model", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def reference(model, tokens, targets):
    """The mean log probability and its gradients in 64 bits, on the CPU, from the weights that the products take."""
    w = {k: t.double().cpu().requires_grad_() for k, t in model.copy.items()}
    norm = lambda x, name: x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-6) * w[name]  # noqa: E731
    h = w["embedding"][tokens.cpu()]
    for b in range(model.blocks):
        h = h + (norm(h, "norm%d" % b) @ w["up%d" % b].t()).clamp(min=0).square() @ w["down%d" % b].t()
    logs = torch.log_softmax(norm(h, "norm") @ w["head"].t(), 1)
    mean = logs[torch.arange(len(tokens)), targets.cpu()].mean()
    mean.backward()
    return float(mean.detach()), {k: t.grad for k, t in w.items()}


@pytest.mark.parametrize("size", [dict(vocab=512, width=256, wide=1024, blocks=2), dict(vocab=101, width=72, wide=200, blocks=3)])
def test_its_gradients_are_those_of_the_network(example, size):
    model = example.TokenModel(bits=32, **size)
    tokens, targets = example.batch(size["vocab"], 512, torch.Generator(device="cuda").manual_seed(5))
    mean = float(model.gradients(tokens, targets))
    want, grads = reference(model, tokens, targets)
    # every value between two products is rounded to 2^-8 of itself, a few of them in a row
    assert abs(mean - want) < 0.02
    for name, grad in grads.items():
        got = model.d[name].double().cpu()
        assert float((got - grad).norm()) < 0.03 * float(grad.norm()), name


def test_it_learns_with_states_in_32_and_in_8_bits(example):
    # nine times out of ten one token, else any of 512: what there is to know leaves 0.9 log 0.9 + 0.1 log (0.1 / 512)
    best = 0.9 * math.log(0.9 + 0.1 / 512) + 0.1 * math.log(0.1 / 512)
    means = {}
    for bits in (32, 8):
        model, means[bits] = example.train(200, bits)
        assert best - 0.25 < means[bits] < best + 0.15, (bits, means[bits], best)
        tokens = torch.arange(512, device="cuda")
        ids, logp, entropy = model.ask(tokens)
        assert float((ids[:, 0] == (5 * tokens + 7) % 512).double().mean()) > 0.99
        assert abs(float(logp[:, 0].exp().mean()) - 0.9) < 0.1 and float(entropy.mean()) < 2.0
    assert abs(means[8] - means[32]) < 0.1


def test_a_pass_in_a_graph():
    """Norm, log probabilities of rows in parts with their alternatives, gradient and the norm's gradient, captured and replayed with other
    work between; every replay is the eager result to the bit."""
    from pixienn_amd import ops
    rows, width = 6, 20005
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, width, device="cuda", generator=g).to(torch.bfloat16)
    weight = torch.randn(width, device="cuda", generator=g).to(torch.bfloat16)
    targets = torch.arange(rows, device="cuda") * 3001
    d_logp = torch.ones(rows, device="cuda")
    norm_space = torch.empty(ops.rms_norm_workspace_bytes(rows, width) // 4, device="cuda")
    token_space = torch.empty(ops.token_logprobs_workspace_bytes(rows, width, 4) // 4 + 1, device="cuda")

    def tensors():
        t = {k: torch.zeros_like(x) for k in ("y", "dy", "dx")}
        t.update({k: torch.zeros(rows, device="cuda") for k in ("rstd", "logp", "entropy", "lse", "logp2")})
        return dict(t, dw=torch.zeros(width, device="cuda"), best=torch.zeros(rows, 4, device="cuda"), ids=torch.zeros(rows, 4, device="cuda", dtype=torch.int32))

    def run(t):
        ops.rms_norm_forward(x, t["y"], weight, rstd=t["rstd"])
        ops.token_logprobs_forward(t["y"], targets, t["logp"], t["entropy"], t["lse"], t["best"], t["ids"], workspace=token_space)
        ops.token_logprobs_forward_train(t["y"], targets, d_logp, t["dy"], t["logp2"])
        ops.rms_norm_backward(t["dy"], x, weight, t["rstd"], t["dx"], t["dw"], workspace=norm_space)

    captured, eager = tensors(), tensors()
    run(captured)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            run(captured)
    for _ in range(4):
        x.copy_(torch.randn(rows, width, device="cuda", generator=g))
        for t in captured.values():
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        run(eager)
        torch.cuda.synchronize()
        for k in captured:
            assert torch.equal(captured[k], eager[k]), k

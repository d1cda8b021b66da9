"""Beam search's selection against a stable sort of all scores in 64 bits, and the reordering of the beams' tensors to the bit.

Bounds.  u = 2^-24.  A row's sum of exponentials is added in n / 64 steps of a lane and 16 of a tree, each term with the error of its
exponent, a few u of its distance from the maximum (40 u of the sum for what counts): its logarithm is within (n / 64 + 60) u, and the
score takes one rounding.  Two continuations whose scores lie nearer than twice that may change places; equal ones of equal
rows may not."""
import math

import pytest

torch = pytest.importorskip("torch")

from pixienn_amd import capi

gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


def reference(logits, scores, count, ended=None, end_token=0, scale=1.0):
    """(scores, parents, tokens, the next score) in 64 bits."""
    batch, beams = scores.shape
    vocab = logits.shape[1]
    z = (logits.float().cpu() * torch.tensor(scale)).double()
    peak = z.amax(1, keepdim=True)
    all_ = (z - peak) - (z - peak).exp().sum(1, keepdim=True).log()
    all_ = (all_ + scores.double().cpu().view(-1, 1)).view(batch, beams, vocab)
    if ended is not None:
        over = ended.cpu().bool()
        first = scores.double().cpu()
        all_[over] = -math.inf
        all_[:, :, 0] = torch.where(over, first, all_[:, :, 0])
    all_ = torch.where(torch.isnan(all_), -math.inf, all_).view(batch, -1)
    need = count + 1
    if all_.shape[1] < need:
        all_ = torch.nn.functional.pad(all_, (0, need - all_.shape[1]), value=-math.inf)
    best, index = torch.sort(all_, dim=1, descending=True, stable=True)
    none = best[:, :count] == -math.inf
    parents, tokens = index[:, :count] // vocab, index[:, :count] % vocab
    if ended is not None:
        tokens = torch.where(ended.cpu().bool().gather(1, parents.clamp(max=beams - 1)), end_token, tokens)
    return best[:, :count], torch.where(none, -1, parents), torch.where(none, -1, tokens), best[:, count]


def run(ops, logits, scores, count, **more):
    batch = scores.shape[0]
    out = torch.full((batch, count), 7.0, device="cuda")
    parents, tokens = (torch.full((batch, count), 7, device="cuda", dtype=torch.int32) for _ in range(2))
    ops.beam_select(logits, scores, out, parents, tokens, **more)
    return out, parents, tokens


def check(ops, logits, scores, count, **more):
    got, parents, tokens = (t.cpu() for t in run(ops, logits, scores, count, **more))
    more.pop("workspace", None)
    want, want_parents, want_tokens, behind = reference(logits, scores, count, **more)
    bound = (logits.shape[1] / 64 + 60) * U
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite)
    assert torch.equal(got[~finite].double(), want[~finite])
    assert not finite.any() or float(((got.double() - want).abs() - bound - U * want.abs())[finite].max()) <= 0
    # in their places where the neighbours are far enough away, or equal (then the rows are, and so is what is formed of them)
    gaps = torch.cat([torch.full((len(want), 1), math.inf, dtype=torch.float64), -torch.cat([want, behind[:, None]], 1).diff(dim=1)], 1)
    gaps = torch.where(torch.isnan(gaps) | (gaps == 0), math.inf, gaps)
    sure = (gaps[:, :-1] > 2 * bound) & (gaps[:, 1:] > 2 * bound)
    assert sure.double().mean() > 0.5
    assert torch.equal(parents[sure].long(), want_parents[sure]) and torch.equal(tokens[sure].long(), want_tokens[sure])
    return got, parents, tokens


@gpu
@pytest.mark.parametrize("batch,beams,vocab,count", [(1, 1, 1, 1), (1, 1, 5, 5), (3, 2, 7, 9), (2, 4, 1000, 4), (5, 3, 4097, 6), (1, 4, 131072, 4),
                                                     (7, 8, 5003, 8), (2, 64, 700, 64), (1, 5, 30000, 64), (33, 12, 2111, 24), (300, 4, 1777, 4)])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("scale,pad,masked,ended", [(1.0, 0, 0.0, 0.0), (0.7, 3, 0.5, 0.4)])
def test_the_best_of_all_beams(ops, batch, beams, vocab, count, kind, scale, pad, masked, ended):
    g = torch.Generator().manual_seed(batch * 100 + beams + vocab)
    # no values twice: bfloat16's steps would make ties of different beams all over
    logits = (torch.randn(batch * beams, vocab + pad, generator=g) * 3).to(TYPES[kind])
    if masked:
        logits[torch.rand(logits.shape, generator=g) < masked] = -math.inf
        logits[:, 0] = 1.0
    logits = logits.cuda()[:, :vocab]
    scores = (torch.randn(batch, beams, generator=g) - 5).cuda()
    over = (torch.rand(batch, beams, generator=g) < ended).cuda() if ended else None
    space = torch.empty(ops.beam_select_workspace_bytes(batch, beams, vocab, count), dtype=torch.uint8, device="cuda").fill_(255)
    first = check(ops, logits, scores, count, ended=over, end_token=3, scale=scale, workspace=space)
    again = run(ops, logits, scores, count, ended=None if over is None else over.to(torch.uint8), end_token=3, scale=scale)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(first, again))
    if count == beams:
        # over the scores
        parents, tokens = (torch.empty(batch, count, device="cuda", dtype=torch.int32) for _ in range(2))
        ops.beam_select(logits, scores, scores, parents, tokens, ended=over, end_token=3, scale=scale)
        assert torch.equal(scores.cpu(), first[0]) and torch.equal(parents.cpu(), first[1]) and torch.equal(tokens.cpu(), first[2])


@gpu
@pytest.mark.parametrize("vocab", [9, 3000, 70000])
def test_ties_go_to_the_lower_beam_and_the_lower_token(ops, vocab):
    logits = torch.zeros(8, vocab, device="cuda")
    logits[:, 5] = 1.0
    scores = torch.full((2, 4), -2.0, device="cuda")
    got, parents, tokens = check(ops, logits, scores, 8)
    assert parents[0].tolist() == [0, 1, 2, 3, 0, 0, 0, 0] and tokens[0].tolist() == [5, 5, 5, 5, 0, 1, 2, 3]
    # with an ended beam: its own score among the others'
    over = torch.tensor([[False, True, False, False], [True, True, True, True]], device="cuda")
    got, parents, tokens = check(ops, logits, scores, 6, ended=over, end_token=2)
    assert parents[0].tolist()[0] == 1 and tokens[0].tolist()[0] == 2 and float(got[0, 0]) == -2.0
    assert parents[1].tolist() == [0, 1, 2, 3, -1, -1] and tokens[1].tolist() == [2, 2, 2, 2, -1, -1]
    assert got[1].tolist() == [-2.0] * 4 + [-math.inf] * 2


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_beams_that_are_not_there_and_logits_that_are_no_numbers(ops, kind):
    g = torch.Generator().manual_seed(4)
    dtype, vocab = TYPES[kind], 2500
    logits = (torch.randn(12, vocab, generator=g) * 2).to(dtype).cuda()
    scores = torch.full((3, 4), -math.inf, device="cuda")
    scores[0, 0] = 0.0                       # a first step: one beam
    scores[1, 2], scores[1, 3] = -1.0, -2.0
    got, parents, tokens = check(ops, logits, scores, 4)
    assert parents[0].tolist() == [0] * 4 and set(parents[1].tolist()) <= {2, 3}
    assert parents[2].tolist() == [-1] * 4 and tokens[2].tolist() == [-1] * 4 and bool((got[2] == -math.inf).all())
    scores = (torch.randn(3, 4, generator=g) - 3).cuda()
    logits[0] = -math.inf                    # nothing allowed
    logits[1, 3:] = -math.inf                # three tokens allowed
    logits[2, 700] = math.nan
    logits[3, 9] = math.inf
    logits[5] = torch.finfo(dtype).min       # all of the type's lowest value: numbers like any other
    logits[6] = math.nan
    scores[2, 1] = math.nan
    got, parents, tokens = check(ops, logits, scores, 4)
    assert parents[0].tolist() == [1, 1, 1, -1] and set(tokens[0].tolist()[:3]) == {0, 1, 2}
    assert 2 not in parents[1].tolist() and 1 not in parents[2].tolist()
    # a vocabulary of nothing but the lowest value: equally probable tokens
    got, parents, tokens = check(ops, torch.full((1, vocab), torch.finfo(dtype).min, device="cuda").to(dtype), torch.zeros(1, 1, device="cuda"), 3)
    assert tokens.tolist() == [[0, 1, 2]] and abs(float(got[0, 0]) + math.log(vocab)) < 1e-4


@gpu
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 4), (3, 8), (5, 3), (2, 64), (100, 2)])
def test_tensors_in_the_beams_new_order(ops, batch, beams):
    g = torch.Generator().manual_seed(batch + beams)
    rows = batch * beams
    make = lambda shape, dtype: (torch.randn(shape, generator=g) * 100).to(dtype).cuda()  # noqa: E731
    wide = make((rows, 40), torch.float32)
    tensors = [make((rows, 1), torch.uint8), make((rows, 3), torch.int16), make((rows, 7), torch.float32), make((rows, 5, 129), torch.bfloat16),
               make((rows, 4096), torch.float32), make((rows,), torch.int64), make((rows, 70001), torch.uint8), wide[:, 3:20], make((rows, 16), torch.bool)]
    tensors += [make((rows, 11), torch.int32) for _ in range(40)]           # more than one launch takes
    parents = torch.randint(0, beams, (batch, beams), generator=g).to(torch.int32)
    parents[0, 0] = -1
    parents[-1, -1] = beams
    place = torch.where((parents < 0) | (parents >= beams), torch.arange(beams), parents) + beams * torch.arange(batch)[:, None]
    want = [t[place.view(-1).cuda()] for t in tensors]
    edges = wide[:, :3].clone(), wide[:, 20:].clone()
    ops.beam_reorder(tensors, parents.cuda())
    for t, w in zip(tensors, want):
        assert torch.equal(t, w)
    assert torch.equal(wide[:, :3], edges[0]) and torch.equal(wide[:, 20:], edges[1])
    ops.beam_reorder(tensors[:1], parents.cuda())
    ops.beam_reorder([], parents.cuda())
    ops.beam_reorder([torch.empty(rows, 0, device="cuda")], parents.cuda())


@gpu
def test_in_a_graph(ops):
    """Steps of a search captured and replayed, each replay as the eager steps."""
    g = torch.Generator().manual_seed(2)
    batch, beams, vocab = 3, 4, 9000
    logits = torch.randn(batch * beams, vocab, generator=g).cuda()
    space = torch.empty(ops.beam_select_workspace_bytes(batch, beams, vocab, beams), dtype=torch.uint8, device="cuda")

    def tensors():
        return [torch.zeros(batch, beams, device="cuda"), torch.zeros(batch, beams, device="cuda", dtype=torch.int32),
                torch.zeros(batch, beams, device="cuda", dtype=torch.int32), torch.arange(batch * beams * 50, device="cuda").view(batch * beams, 50).float()]

    def step(t):
        ops.beam_select(logits, t[0], t[0], t[1], t[2], workspace=space)
        ops.beam_reorder([t[3]], t[1])

    captured, eager = tensors(), tensors()
    step(tensors())
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(captured)
    for _ in range(4):
        logits.copy_(torch.randn(batch * beams, vocab, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        step(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


@gpu
def test_what_is_refused(ops):
    logits, scores = torch.zeros(6, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    out, parents = torch.zeros(2, 4, device="cuda"), torch.zeros(2, 4, device="cuda", dtype=torch.int32)
    tokens = parents.clone()
    wide = torch.zeros(65, 10, device="cuda"), torch.zeros(1, 65, device="cuda")
    many = torch.zeros(2, 65, device="cuda")
    for call, message in [
            (lambda: ops.beam_select(logits, scores, out, parents, tokens.long()), "tokens must be"),
            (lambda: ops.beam_select(logits, scores, out, parents[:1], tokens), "parents must be"),
            (lambda: ops.beam_select(logits, scores, out, None, tokens), "parents is required"),
            (lambda: ops.beam_select(logits, scores.view(-1), out, parents, tokens), "two dimensions"),
            (lambda: ops.beam_select(logits[:5], scores, out, parents, tokens), "a row for each of 2 x 3 beams"),
            (lambda: ops.beam_select(logits, scores, out, parents, tokens, ended=scores), "ended must be"),
            (lambda: ops.beam_select(logits, scores, out, parents, tokens, ended=torch.zeros(2, 2, dtype=torch.bool, device="cuda")), "ended must hold 6"),
            (lambda: ops.beam_select(logits, scores, out, parents, tokens, scale=0.0), "scale"),
            (lambda: ops.beam_select(logits.double(), scores, out, parents, tokens), "fp32, bfloat16 or half"),
            (lambda: ops.beam_select(logits[:1].expand(6, 10), scores, out, parents, tokens), "overlap"),
            (lambda: ops.beam_select(*wide, out[:1], parents[:1], tokens[:1]), "65 beams"),
            (lambda: ops.beam_select(logits, scores, many, many.int(), many.int()), "65 continuations"),
            (lambda: ops.beam_select(logits, scores, out, parents, tokens, workspace=torch.empty(4, device="cuda")), "workspace too small"),
            (lambda: ops.beam_reorder([logits], parents), "must have 2 x 4 rows"),
            (lambda: ops.beam_reorder([logits.cpu()], parents[:, :3].contiguous()), "must live on the GPU"),
            (lambda: ops.beam_reorder([None], parents[:, :3].contiguous()), "is required"),
            (lambda: ops.beam_reorder([logits[:, ::2]], parents[:, :3].contiguous()), "next to each other"),
            (lambda: ops.beam_reorder([logits[:1].expand(6, 10)], parents[:, :3].contiguous()), "overlap"),
            (lambda: ops.beam_reorder([logits], parents[:, :3].contiguous().long()), "parents must be")]:
        with pytest.raises(capi.PxError, match=message):
            call()

"""Embeddings, layer norm, the gated scan and beam search as programs use them: captured and replayed with other work between, two graphs
that share a workspace, two streams at once, and tensors whose offsets do not fit 32 bits."""
import pytest

torch = pytest.importorskip("torch")

from pixienn_amd import ops  # noqa: E402

pytestmark = pytest.mark.gpu

ROWS, WIDTH, VOCAB, BATCH, BEAMS = 301, 1029, 777, 3, 4


class Work:
    """One call of everything, into its own results."""

    def __init__(self, seed, space=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
        half = lambda *shape: normal(*shape).to(torch.bfloat16)  # noqa: E731
        self.inputs = dict(table=half(VOCAB, WIDTH), update=half(ROWS, WIDTH), gate=half(ROWS, WIDTH), dy=half(ROWS, WIDTH), weight=half(WIDTH),
                           bias=half(WIDTH), logits=half(BATCH * BEAMS, 20005), scores=normal(BATCH, BEAMS), state=normal(2, WIDTH))
        self.tokens = torch.randint(0, VOCAB, (ROWS,), device="cuda", generator=g)
        self.starts = torch.tensor([0, 100, ROWS], device="cuda", dtype=torch.int32)
        sizes = [ops.embedding_workspace_bytes(ROWS, WIDTH), ops.layer_norm_workspace_bytes(ROWS, WIDTH), ops.gated_scan_workspace_bytes(ROWS, WIDTH),
                 ops.beam_select_workspace_bytes(BATCH, BEAMS, 20005, BEAMS)]
        self.space = torch.empty(max(sizes) // 4 + 1, device="cuda") if space is None else space

    def results(self):
        t = {k: torch.zeros(ROWS, WIDTH, device="cuda", dtype=torch.bfloat16) for k in ("x", "norm", "dx", "y", "dxs", "du", "dg")}
        t.update(d=torch.zeros(VOCAB, WIDTH, device="cuda", dtype=torch.bfloat16), more=torch.zeros(VOCAB, WIDTH, device="cuda"),
                 mean=torch.zeros(ROWS, device="cuda"), rstd=torch.zeros(ROWS, device="cuda"), dw=torch.zeros(WIDTH, device="cuda"),
                 db=torch.zeros(WIDTH, device="cuda"), saved=torch.zeros(-(-ROWS // 16), WIDTH, device="cuda"), final=torch.zeros(2, WIDTH, device="cuda"),
                 d_state=torch.zeros(2, WIDTH, device="cuda"), step=torch.zeros(2, WIDTH, device="cuda", dtype=torch.bfloat16),
                 best=torch.zeros(BATCH, BEAMS, device="cuda"), parents=torch.zeros(BATCH, BEAMS, device="cuda", dtype=torch.int32),
                 next=torch.zeros(BATCH, BEAMS, device="cuda", dtype=torch.int32), history=torch.zeros(BATCH * BEAMS, 33, device="cuda"))
        return t

    def run(self, t):
        i, space = self.inputs, self.space
        ops.embedding_forward(i["table"], self.tokens, t["x"], 2.0)
        ops.layer_norm_forward(t["x"], t["norm"], i["weight"], i["bias"], mean=t["mean"], rstd=t["rstd"])
        ops.gated_scan_forward(t["norm"], i["update"], t["y"], i["gate"], self.starts, state=i["state"], final=t["final"], saved=t["saved"], workspace=space)
        ops.gated_scan_backward(i["dy"], t["norm"], i["update"], t["saved"], t["dxs"], t["du"], i["gate"], t["dg"], self.starts, state=i["state"],
                                d_state=t["d_state"], workspace=space)
        ops.layer_norm_backward(t["dxs"], t["x"], i["weight"], t["mean"], t["rstd"], t["dx"], t["dw"], t["db"], workspace=space)
        ops.embedding_backward(t["dx"], self.tokens, t["d"], 2.0, workspace=space)
        ops.embedding_backward(t["dx"], self.tokens, t["more"], 2.0, accumulate=True, workspace=space)
        ops.gated_scan_step(t["norm"][:2], i["update"][:2], t["step"], t["final"], i["gate"][:2])
        ops.beam_select(i["logits"], i["scores"], t["best"], t["parents"], t["next"], workspace=space)
        t["history"].copy_(i["table"][:BATCH * BEAMS, :33])
        ops.beam_reorder([t["history"]], t["parents"])

    def renew(self):
        for v in self.inputs.values():
            v.copy_(torch.randn(v.shape, device="cuda", generator=self.g))
        self.tokens.copy_(torch.randint(0, VOCAB, (ROWS,), device="cuda", generator=self.g))

    def captured(self, t):
        self.run(self.results())                    # libraries prepare themselves in their first call
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                self.run(t)
        return graph


def same(a, b):
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_two_graphs_that_share_a_workspace():
    one = Work(1)
    other = Work(2, one.space)
    works = [(w, w.results()) for w in (one, other)]
    graphs = [w.captured(t) for w, t in works]
    for _ in range(4):
        for w, t in works:
            w.renew()
            for v in t.values():
                v.zero_()
        one.space.uniform_()                        # what is left in a workspace says nothing
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for w, t in works:
            eager = w.results()
            w.run(eager)
            torch.cuda.synchronize()
            same(t, eager)


def test_two_streams_at_once():
    works = [Work(3), Work(4)]
    alone = []
    for w in works:
        alone.append(w.results())
        w.run(alone[-1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = [w.results() for w in works]
    torch.cuda.synchronize()
    for _ in range(5):
        for w, t, s in zip(works, results, streams):
            with torch.cuda.stream(s):
                t["more"].zero_()
                w.run(t)
    torch.cuda.synchronize()
    for t, a in zip(results, alone):
        same(t, a)


# 2^31 values and more, of which the last rows lie behind every offset of 32 bits
LONG_ROWS, LONG_WIDTH, LAST = 262147, 8200, 37


def test_long_layer_norm_and_embedding():
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(LONG_ROWS, LONG_WIDTH, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    weight = torch.randn(LONG_WIDTH, device="cuda", generator=g)
    y, mean, rstd = torch.empty_like(x), torch.empty(LONG_ROWS, device="cuda"), torch.empty(LONG_ROWS, device="cuda")
    ops.layer_norm_forward(x, y, weight, mean=mean, rstd=rstd)
    few = x[-LAST:].clone()
    want = torch.nn.functional.layer_norm(few.double(), (LONG_WIDTH,), weight.double(), None, 1e-5)
    # half a step of bfloat16, and what fp32 statistics leave
    assert bool(((y[-LAST:].double() - want).abs() <= want.abs() * 2 ** -8 + 1e-5).all())
    # dx over dy
    h, dw = x, torch.empty(LONG_WIDTH, device="cuda")
    small_dy, small_dx = y[-LAST:].clone(), torch.empty_like(few)
    ops.layer_norm_backward(small_dy, few, weight, mean[-LAST:].contiguous(), rstd[-LAST:].contiguous(), small_dx, dw)
    ops.layer_norm_backward(y, h, weight, mean, rstd, y, dw)
    assert float((y[-LAST:].double() - small_dx.double()).norm()) <= 2 ** -8 * float(small_dx.double().norm())
    del y, h
    # a table that long: its last rows looked up, and their gradient
    tokens = torch.arange(LONG_ROWS - LAST, LONG_ROWS, device="cuda").flip(0)
    rows = torch.empty_like(few)
    ops.embedding_forward(x, tokens, rows)
    assert torch.equal(rows, few.flip(0))
    ops.embedding_backward(rows, tokens, x)
    assert torch.equal(x[-LAST:], few) and not bool(x[:-LAST].any())
    # and that many rows, all of one token or of none
    x[-LAST:] = 1
    x[:5] = 2
    where = torch.full((LONG_ROWS,), 3, device="cuda", dtype=torch.int32)
    where[100:110] = -1
    d = torch.empty(5, LONG_WIDTH, device="cuda")
    ops.embedding_backward(x, where, d)
    assert bool((d[3] == LAST + 10).all()) and not bool(d[[0, 1, 2, 4]].any())


def test_a_long_scan():
    g = torch.Generator(device="cuda").manual_seed(6)
    make = lambda: torch.empty(LONG_ROWS, LONG_WIDTH, device="cuda", dtype=torch.bfloat16).normal_(generator=g)  # noqa: E731
    x, update, dy = make(), make(), make()
    starts = torch.tensor([0, 7, LONG_ROWS - LAST, LONG_ROWS], device="cuda", dtype=torch.int32)
    saved, y = ops.gated_scan_saved_like(x), torch.empty_like(x)
    ops.gated_scan_forward(x, update, y, starts=starts, saved=saved)
    few = [t[-LAST:].clone() for t in (x, update, dy)]
    few_saved, few_y, few_dx, few_du = ops.gated_scan_saved_like(few[0]), *(torch.empty_like(few[0]) for _ in range(3))
    ops.gated_scan_forward(few[0], few[1], few_y, saved=few_saved)
    ops.gated_scan_backward(few[2], few[0], few[1], few_saved, few_dx, few_du)
    ops.gated_scan_backward(dy, x, update, saved, x, update, starts=starts)
    for got, want in ((y[-LAST:], few_y), (x[-LAST:], few_dx), (update[-LAST:], few_du)):
        # the last bits of h depend on where the sequence lies: a rounding to bfloat16 may fall the other way
        assert bool(((got.double() - want.double()).abs() <= want.double().abs() * 2 ** -7 + 1e-5).all())


def test_long_rows_of_beams_and_many_logits():
    g = torch.Generator(device="cuda").manual_seed(7)
    cache = torch.empty(4, (1 << 30) + 24, device="cuda", dtype=torch.bfloat16)
    for i in range(4):
        cache[i].fill_(i)
        cache[i, -5:] = 10 + i
    ops.beam_reorder([cache], torch.tensor([[1, 3, -1, 0]], device="cuda", dtype=torch.int32))
    for row, of in enumerate([1, 3, 2, 0]):
        assert bool((cache[row, -5:] == 10 + of).all()) and bool((cache[row, :-5] == of).all())
    del cache
    batch, beams, vocab = 4100, 4, 131073
    logits = torch.empty(batch * beams, vocab, device="cuda", dtype=torch.float16).normal_(generator=g)
    scores = torch.randn(batch, beams, device="cuda", generator=g)
    best, parents, tokens = torch.empty_like(scores), *(torch.empty(batch, beams, device="cuda", dtype=torch.int32) for _ in range(2))
    ops.beam_select(logits, scores, best, parents, tokens)
    last = torch.log_softmax(logits[-beams:].double(), 1) + scores[-1].double()[:, None]
    want, at = (t[:beams] for t in last.flatten().sort(descending=True, stable=True))
    assert float((best[-1].double() - want).abs().max()) < 1e-5
    assert (parents[-1].long() * vocab + tokens[-1]).tolist() == at.tolist()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("width,dtype", [(1664, torch.bfloat16), (1666, torch.float16), (832, torch.float32)])
def test_scans_past_the_caches_are_those_of_fewer_channels(gated, ragged, width, dtype):
    """Channels have nothing to do with each other: some of them by themselves, in a call that the caches hold, have the same bits."""
    g = torch.Generator(device="cuda").manual_seed(8)
    rows = 16384
    make = lambda: torch.empty(rows, width, device="cuda", dtype=dtype).normal_(generator=g)  # noqa: E731
    x, update, gate, dy = make(), make() - 3, make() if gated else None, make()
    assert rows * width * x.element_size() * 3 >= 128 << 20
    how = dict(starts=torch.tensor([0, 1, 77, 5000, 5000, 12345, rows - 40], device="cuda", dtype=torch.int32)) if ragged else dict(sequences=4)

    def run(columns):
        x_, u_, dy_ = (t[:, columns].contiguous() for t in (x, update, dy))
        o_ = gate[:, columns].contiguous() if gated else None
        y, dx, du = (torch.full_like(x_, 7.0) for _ in range(3))
        do, saved = torch.full_like(x_, 7.0) if gated else None, ops.gated_scan_saved_like(x_)
        ops.gated_scan_forward(x_, u_, y, gate=o_, saved=saved, **how)
        ops.gated_scan_backward(dy_, x_, u_, saved, dx, du, gate=o_, dgate=do, **how)
        return [t for t in (y, dx, du, do) if t is not None]

    whole = run(slice(None))
    for columns in (slice(0, 64), slice(width - 130, width)):
        for a, b in zip(whole, run(columns)):
            assert torch.equal(a[:, columns], b)


@pytest.mark.parametrize("rows,vocab,width,out,accumulate", [(9000, 20000, 3584, torch.bfloat16, False), (40000, 3000, 2000, torch.float32, False),
                                                             (40000, 30000, 1001, torch.float32, True), (40000, 30000, 1800, torch.bfloat16, True)])
def test_table_gradients_past_the_caches(rows, vocab, width, out, accumulate):
    g = torch.Generator(device="cuda").manual_seed(9)
    dy = torch.empty(rows, width, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    tokens = (torch.rand(rows, device="cuda", generator=g) ** 4 * (vocab + 3)).long()
    assert (rows * 2 + (0 if accumulate else vocab * out.itemsize)) * width >= 128 << 20 or accumulate
    d = torch.empty(vocab, width, device="cuda", dtype=out).normal_(generator=g) if accumulate else torch.full((vocab, width), 7.0, device="cuda", dtype=out)
    was = d.clone() if accumulate else torch.zeros_like(d)
    ops.embedding_backward(dy, tokens, d, 0.5, accumulate=accumulate)
    for columns in (slice(0, 40), slice(width - 40, width)):
        there = tokens < vocab
        part, who = dy[there][:, columns].double(), tokens[there]
        zeros = lambda: torch.zeros(vocab, part.shape[1], device="cuda", dtype=torch.float64)  # noqa: E731
        total, size = zeros().index_add_(0, who, part) * 0.5, zeros().index_add_(0, who, part.abs()) * 0.5
        count = torch.zeros(vocab, 1, device="cuda", dtype=torch.float64).index_add_(0, who, torch.ones(len(who), 1, device="cuda", dtype=torch.float64))
        want = was[:, columns].double() + total
        # a rounding of 2^-24 of what is there for each addition, and half a step of the type
        bound = (count + 2) * 2.0 ** -24 * (size + was[:, columns].double().abs()) + want.abs() * torch.finfo(out).eps / 2
        assert bool(((d[:, columns].double() - want).abs() <= bound).all())

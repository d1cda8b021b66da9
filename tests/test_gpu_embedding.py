"""Embeddings by token and the gradient of their table.  The lookup is one product rounded twice, compared to the bit.  A sum of m rows
in fp32, in any order, is within (m + 1) u of the sum of the magnitudes, u = 2^-24; then the scale's product, the rounding to the type (e),
and with what was there one more addition."""
import pytest

torch = pytest.importorskip("torch")

from pixienn_amd import capi

gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": (torch.float32, 2.0 ** -24, 2.0 ** -140), "bf16": (torch.bfloat16, 2.0 ** -8, 2.0 ** -134),
         "f16": (torch.float16, 2.0 ** -11, 2.0 ** -25)}


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


def draw(seed, rows, width, dtype, pad=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, width + pad, generator=g) * std).to(dtype).cuda()[:, :width]


@gpu
@pytest.mark.parametrize("rows,width,vocab", [(1, 1, 1), (3, 7, 5), (1000, 64, 10), (33, 1000, 77), (2, 40001, 3), (5000, 130, 4000)])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("scale,pad,wide", [(1.0, 0, True), (0.37, 3, False)])
def test_rows_by_token(ops, rows, width, vocab, kind, scale, pad, wide):
    dtype = TYPES[kind][0]
    table = draw(1, vocab, width, dtype, pad)
    g = torch.Generator().manual_seed(rows)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    outside = torch.rand(rows, generator=g) < 0.2
    tokens[outside] = torch.tensor([-1, vocab, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (int(outside.sum()),), generator=g)]
    if wide and rows > 2:
        tokens[1], outside[1] = 2 ** 32 + vocab - 1, True        # whose low half is a token
    y = torch.full((rows, width + pad), 7.0, dtype=dtype, device="cuda")
    ops.embedding_forward(table, tokens.cuda() if wide else tokens.int().cuda(), y[:, :width], scale=scale)
    # the scale as the kernel has it, in fp32
    want = (table[tokens.masked_fill(outside, 0).cuda()].float() * torch.tensor(scale, device="cuda")).to(dtype)
    want[outside.cuda()] = 0
    assert torch.equal(y[:, :width], want)
    assert bool((y[:, width:] == 7).all())


@gpu
def test_leading_dimensions_and_large_tables(ops):
    tokens = torch.tensor([[3, 99999], [50000, 0]], device="cuda")
    table = torch.randn(100000, 6400, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()     # 1.28 GB
    y = torch.empty(2, 2, 6400, device="cuda", dtype=torch.bfloat16)
    ops.embedding_forward(table, tokens, y)
    assert torch.equal(y, table[tokens])
    many = torch.arange(99999, 59999, -1, device="cuda")             # past the caches
    y = torch.empty(40000, 6400, device="cuda", dtype=torch.bfloat16)
    ops.embedding_forward(table, many, y)
    assert torch.equal(y, table[many])


def tokens_of(how, rows, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    if how == "one":
        return torch.full((rows,), vocab // 2)
    if how == "different":
        return torch.randperm(max(rows, vocab), generator=g)[:rows] % vocab
    if how == "none":
        return torch.full((rows,), -1)
    if how == "runs":            # every token a few rows in a row: runs end at many places of a part
        return (torch.arange(rows) // 5) % vocab
    # a few frequent ones, many rare ones, some outside
    tokens = (torch.rand(rows, generator=g, dtype=torch.float64).pow(6) * vocab).long().clamp(max=vocab - 1)
    tokens[torch.rand(rows, generator=g) < 0.05] = -1
    tokens[torch.rand(rows, generator=g) < 0.02] = vocab
    return tokens


def check(ops, dy, tokens, vocab, width, out, scale, accumulate, workspace=None, wide=True):
    e, least = next((e, l) for t, e, l in TYPES.values() if t is out)
    pad = 5
    wide_d = draw(9, vocab, width, out, pad) if accumulate else torch.full((vocab, width + pad), 7.0, dtype=out, device="cuda")[:, :width]
    store = torch.as_strided(wide_d, (vocab, width + pad), (width + pad, 1))
    edge = store[:, width:].clone()
    d = store[:, :width]
    was = d.clone()
    there = tokens.cuda() if wide else tokens.int().cuda()
    ops.embedding_backward(dy, there, d, scale=scale, accumulate=accumulate, workspace=workspace)
    assert torch.equal(store[:, width:], edge)
    good = (tokens >= 0) & (tokens < vocab)
    place = tokens[good].cuda()
    total, magnitude = (torch.zeros(vocab, width, dtype=torch.float64, device="cuda").index_add_(0, place, t)
                        for t in (dy[good.cuda()].double(), dy[good.cuda()].double().abs()))
    count = torch.bincount(tokens[good], minlength=vocab).cuda()
    s = float(torch.tensor(scale))
    want = total * s + (was.double() if accumulate else 0)
    bound = magnitude * s * U * (count[:, None].double() + 3) + want.abs() * (e + U) + least + (was.double().abs() * U if accumulate else 0)
    over = (d.double() - want).abs() - bound
    assert float(over.max()) <= 0, float(over.max())
    # a token of no row: zeros, or what was there
    untouched = count == 0
    assert torch.equal(d[untouched], was[untouched] if accumulate else torch.zeros_like(d[untouched]))
    # the same bits again
    again = was.clone()
    ops.embedding_backward(dy, there, again, scale=scale, accumulate=accumulate, workspace=workspace)
    assert torch.equal(again, d)


ROWS = [1, 2, 31, 32, 33, 64, 65, 2047, 2048, 2049, 5000]


@gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("how", ["text", "one", "different", "runs", "none"])
@pytest.mark.parametrize("kind,out,width,accumulate", [("bf16", "same", 72, False), ("f16", "f32", 301, True), ("f32", "f32", 13, False)])
def test_the_gradient_is_the_sum_by_token(ops, rows, how, kind, out, width, accumulate):
    dtype = TYPES[kind][0]
    vocab = 77 if how == "runs" else 1000
    dy = draw(rows, rows, width, dtype, 3, std=0.1)
    check(ops, dy, tokens_of(how, rows, vocab, rows), vocab, width, dtype if out == "same" else torch.float32, 0.75, accumulate, wide=rows % 2 == 0)


@gpu
@pytest.mark.parametrize("rows,vocab,width,how", [(70001, 500, 40, "text"), (70001, 3, 17, "one"), (66000, 70000, 8, "different"), (140000, 50, 9, "runs"),
                                                  (1, 1, 5, "one"), (40, 1, 3, "text"), (3000, 2 ** 21 - 2, 2, "text"), (3000, 2 ** 21 - 1, 2, "text"),
                                                  (5000, 3 * 10 ** 6, 1, "different"), (300, 64, 9001, "text"), (4000, 300, 2048, "text")])
def test_many_rows_and_all_vocabularies(ops, rows, vocab, width, how):
    dy = draw(rows, rows, width, torch.bfloat16, std=0.1)
    check(ops, dy, tokens_of(how, rows, vocab, rows), vocab, width, torch.float32, 1.0, False)
    check(ops, dy, tokens_of(how, rows, vocab, rows), vocab, width, torch.bfloat16, 3.0, True)


@gpu
def test_a_workspace_of_the_callers_serves_smaller_calls(ops):
    space = torch.empty(ops.embedding_workspace_bytes(5000, 301), dtype=torch.uint8, device="cuda").fill_(255)
    for rows, width in [(5000, 301), (4999, 300), (33, 301), (5000, 1)]:
        check(ops, draw(1, rows, width, torch.float32, std=0.1), tokens_of("text", rows, 90, 1), 90, width, torch.float32, 1.0, True, workspace=space)


@gpu
def test_no_rows_and_what_is_no_number(ops):
    none = torch.empty(0, 8, device="cuda")
    nothing = torch.empty(0, device="cuda", dtype=torch.int64)
    d = torch.full((5, 8), 7.0, device="cuda")
    ops.embedding_backward(none, nothing, d, accumulate=True)
    assert bool((d == 7).all())
    ops.embedding_backward(none, nothing, d)
    assert bool((d == 0).all())
    ops.embedding_forward(d, nothing, none)
    # a NaN or an infinity stays with its token
    dy = torch.ones(70, 8, device="cuda")
    dy[40], dy[50] = float("nan"), float("inf")
    tokens = torch.arange(70, device="cuda") % 5
    ops.embedding_backward(dy, tokens, d)
    assert bool(torch.isnan(d[0]).all()) or bool(torch.isinf(d[0]).all())
    assert bool((d[1:] == 14).all())


@gpu
def test_what_is_refused(ops):
    table, dy = torch.zeros(10, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    tokens = torch.zeros(4, device="cuda", dtype=torch.int64)
    for call, message in [
            (lambda: ops.embedding_forward(table, None, dy), "tokens is required"),
            (lambda: ops.embedding_forward(table, tokens[:3], dy), "tokens must hold 4"),
            (lambda: ops.embedding_forward(table, tokens.float(), dy), "tokens must be"),
            (lambda: ops.embedding_forward(table, tokens.cpu(), dy), "must live on the GPU"),
            (lambda: ops.embedding_forward(table, tokens, dy.half()), "y must be"),
            (lambda: ops.embedding_forward(table, tokens, dy[:, :4]), "y must be"),
            (lambda: ops.embedding_forward(table[:0], tokens, dy), "a table of 0 rows"),
            (lambda: ops.embedding_forward(table[:1].expand(10, 8), tokens, dy), "overlap"),
            (lambda: ops.embedding_backward(dy, tokens, table.half()), "d must be"),
            (lambda: ops.embedding_backward(dy.half(), tokens, table.bfloat16()), "d must be"),
            (lambda: ops.embedding_backward(dy, tokens, table[:, :7]), "d must be"),
            (lambda: ops.embedding_backward(dy, tokens, table, workspace=torch.empty(4, device="cuda")), "workspace too small"),
            (lambda: ops.embedding_backward(dy, tokens, table, workspace=torch.empty(4096)), "must live on the GPU")]:
        with pytest.raises(capi.PxError, match=message):
            call()

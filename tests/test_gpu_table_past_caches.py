"""The table's gradient added to what is there, where the tensors do not fit the caches: odd widths and every pair of types."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
STREAMING = 128 << 20           # bytes of a call from which on it goes past the caches


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


@pytest.mark.parametrize("rows,vocab,width,dtype,out", [(70000, 30000, 1001, torch.bfloat16, torch.float32), (70001, 5000, 1001, torch.float16, torch.float32),
                                                        (40000, 3000, 1801, torch.bfloat16, torch.bfloat16), (41000, 3000, 1803, torch.float16, torch.float16),
                                                        (40001, 9000, 901, torch.float32, torch.float32), (5000, 700, 13601, torch.bfloat16, torch.float32)])
def test_added_gradients_past_the_caches(ops, rows, vocab, width, dtype, out):
    # the table does not count where it is added to
    assert rows * width * dtype.itemsize >= STREAMING
    g = torch.Generator(device="cuda").manual_seed(width)
    dy = torch.empty(rows, width, device="cuda", dtype=dtype).normal_(generator=g)
    # few frequent tokens, many rare ones and none of some; some outside the vocabulary
    tokens = (torch.rand(rows, device="cuda", generator=g) ** 4 * (vocab + 3)).long()
    d = torch.empty(vocab, width, device="cuda", dtype=out).normal_(generator=g)
    was = d.clone()
    ops.embedding_backward(dy, tokens, d, 0.5, accumulate=True)
    there = tokens < vocab
    count = torch.bincount(tokens[there], minlength=vocab).double()[:, None]
    assert torch.equal(d[count[:, 0] == 0], was[count[:, 0] == 0])
    for columns in (slice(0, 40), slice(width // 2, width // 2 + 40), slice(width - 41, width)):
        part, who, before = dy[there][:, columns].double(), tokens[there], was[:, columns].double()
        zeros = lambda: torch.zeros(vocab, part.shape[1], device="cuda", dtype=torch.float64)  # noqa: E731
        want, size = before + zeros().index_add_(0, who, part) * 0.5, before.abs() + zeros().index_add_(0, who, part.abs()) * 0.5
        # a rounding of 2^-24 of what is there for each addition, and half a step of the type
        bound = (count + 2) * 2.0 ** -24 * size + want.abs() * torch.finfo(out).eps / 2
        assert bool(((d[:, columns].double() - want).abs() <= bound).all())

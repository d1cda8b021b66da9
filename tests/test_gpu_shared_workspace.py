"""Table gradients that share a workspace on two streams, which the interface forbids: what they leave has no meaning, but they end, and nothing beyond
their tensors and the workspace is written to."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


@pytest.mark.parametrize("rows", [(3000, 6000), (9000, 40000), (70000, 200000), (5000, 150000)])
def test_table_gradients_on_one_workspace_touch_nothing_else(ops, rows):
    g = torch.Generator(device="cuda").manual_seed(rows[0])
    width, vocab, edge = 40, 3001, 64
    need = max(ops.embedding_workspace_bytes(n, width) for n in rows)
    around = torch.full((need + 2 * 4096,), 0xA5, device="cuda", dtype=torch.uint8)
    space = around[4096:4096 + need]
    calls = []
    for n in rows:
        dy = torch.empty(n, width, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
        tokens = torch.randint(0, vocab, (n,), device="cuda", generator=g)
        table = torch.full((vocab + 2 * edge, width + 3), 7.0, device="cuda")
        calls.append((dy, tokens, table))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for stream, (dy, tokens, table) in zip(streams, calls):
            with torch.cuda.stream(stream):
                ops.embedding_backward(dy, tokens, table[edge:edge + vocab, :width], workspace=space)
    torch.cuda.synchronize()
    assert bool((around[:4096] == 0xA5).all()) and bool((around[4096 + need:] == 0xA5).all())
    for dy, tokens, table in calls:
        assert bool((table[:edge] == 7).all()) and bool((table[-edge:] == 7).all()) and bool((table[:, width:] == 7).all())
        # and alone the call is right again, whatever the workspace holds
        ops.embedding_backward(dy, tokens, table[edge:edge + vocab, :width], workspace=space)
        zeros = lambda: torch.zeros(vocab, width, device="cuda", dtype=torch.float64)  # noqa: E731
        want, size = zeros().index_add_(0, tokens, dy.double()), zeros().index_add_(0, tokens, dy.double().abs())
        count = torch.bincount(tokens, minlength=vocab)[:, None]
        # a rounding of 2^-24 of what is there for each addition
        assert bool(((table[edge:edge + vocab, :width].double() - want).abs() <= (count + 2) * 2.0 ** -24 * size).all())

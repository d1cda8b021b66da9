"""Sequences of one length side by side or one behind the other, which the distances of rows and sequences decide for scans with a gate: the same bits."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


@pytest.mark.parametrize("sequences,length,width,dtype", [(3, 2048, 2048, torch.bfloat16), (2, 4096, 2048, torch.float16), (4, 1024, 2048, torch.float32),
                                                          (5, 1024, 4096, torch.bfloat16), (3, 1920, 2048, torch.bfloat16), (3, 512, 8192, torch.bfloat16)])
def test_rows_at_any_distance_have_the_same_bits(ops, sequences, length, width, dtype):
    g = torch.Generator(device="cuda").manual_seed(length)
    rows = sequences * length
    # channels that remember: states go from chunk to chunk
    values = [torch.empty(rows, width, device="cuda").normal_(generator=g) for _ in range(3)]
    values[1] -= torch.rand(width, device="cuda", generator=g) * 8
    state = torch.empty(sequences, width, device="cuda").normal_(generator=g)

    def run(pad, pick=slice(None)):
        wide = [torch.empty(rows, width + pad, device="cuda", dtype=dtype) for _ in range(3)]
        for t, v in zip(wide, values):
            t[:, :width] = v
        x, update, gate = (t[:, :width].view(rows, width)[pick] if not pad else t[:, :width][pick] for t in wide)
        many = 1 if pick != slice(None) else sequences
        begin = state[:1].clone() if many == 1 else state.clone()
        y, final, saved = torch.empty(len(x), width, device="cuda", dtype=dtype), torch.empty_like(begin), ops.gated_scan_saved_like(x)
        ops.gated_scan_forward(x, update, y, gate=gate, sequences=many, state=begin, final=final, saved=saved)
        return y, final, saved

    near, far = run(0), run(8)
    assert all(torch.equal(a, b) for a, b in zip(near, far))
    # (its first sequence by itself, where the groups of chunks begin with it as well)
    y, final, saved = run(0, slice(0, length))
    assert torch.equal(y, near[0][:length]) and torch.equal(final[0], near[1][0])
    columns = torch.tensor([0, 1, width // 2, width - 1], device="cuda")
    z, x64, gate64 = (v[:, columns].to(dtype).double().cpu() for v in (values[1], values[0], values[2]))
    z = torch.sigmoid(z).view(sequences, length, -1)
    h, rows64 = state[:, columns].double().cpu(), []
    for t in range(length):
        h = h + z[:, t] * (x64.view(sequences, length, -1)[:, t] - h)
        rows64.append(h)
    gate64 = gate64.view(sequences, length, -1)
    want = torch.stack(rows64, 1) * gate64 * torch.sigmoid(gate64)
    got = near[0][:, columns].double().cpu().view(sequences, length, -1)
    # a step rounds h by 2^-23 of what is there (up to 6), z by 2^-24 |u| and less (up to 16): both forgotten as the state is; half a step of the type, which
    # below its least normal number is that number's (halves below 2^-14: steps of 2^-24 beside gates of 10^-5)
    kind = torch.finfo(dtype)
    bound = 1e-3 * gate64.abs() + want.abs().clamp(min=kind.smallest_normal) * kind.eps / 2
    assert bool(((got - want).abs() <= bound).all()) and float((near[1][:, columns].double().cpu() - h).abs().max()) < 1e-3

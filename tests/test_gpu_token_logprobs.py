"""Log probabilities of given tokens, entropy, alternatives, and the gradient of the logits, against the definitions in 64 bits.

Bounds.  u = 2^-24, e half a unit of the logits' type.  With D the mean of (peak - z) under the row's distribution and Q that of its
square: an exponent (l - peak) * c carries three roundings, so a term of the sum is off by 3 u (peak - z) + 2 u of itself, their sum
by the mean of that, and by u for each of the additions in turn (a 256th of the row, the tree and the workgroup).  That is the error
of the logarithm; the entropy has the mean of t beside it.  A probability of the gradient is off by two roundings of its
logarithm, by what lse is off, and the exponential."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from pixienn_amd import capi

gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": (torch.float32, 2.0 ** -24, 2.0 ** -140), "bf16": (torch.bfloat16, 2.0 ** -8, 2.0 ** -134),
         "f16": (torch.float16, 2.0 ** -11, 2.0 ** -25)}
INF = math.inf


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


def draw(seed, rows, vocab, dtype, std=2.5, pad=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab + pad, generator=g) * std).to(dtype).cuda()[:, :vocab]


class Want:
    """The definitions in 64 bits, and the bounds."""

    def __init__(self, logits, scale):
        z = self.z = logits.double() * float(np.float32(scale))
        peak = z.amax(1, keepdim=True)
        self.empty = (peak == -INF)[:, 0]
        t = z - torch.where(peak == -INF, 0.0, peak)
        e = t.exp()
        total = e.sum(1, keepdim=True)
        self.p = torch.where(total > 0, e / total, 0.0)
        far = torch.where(t == -INF, 0.0, t)
        d = -(self.p * far).sum(1)
        q = (self.p * far * far).sum(1)
        log_sum = total.log()[:, 0]
        self.lse = torch.where(self.empty, -INF, peak[:, 0] + log_sum)
        self.entropy = torch.where(self.empty, 0.0, log_sum + d)
        self.logs = z - torch.where(self.empty, INF, self.lse)[:, None]
        rel = U * (z.shape[1] / 256 + 40 + 4 + 3 * d)
        clean = lambda x: torch.nan_to_num(x, 0.0, 0.0, 0.0)  # noqa: E731
        self.lse_off = clean(rel + 2 * U * self.lse.abs())
        self.entropy_off = clean(rel * (1 + 2 * d) + 3 * U * q + 2 * U * (log_sum.abs() + d))

    def logp(self, targets):
        given = (targets >= 0) & (targets < self.z.shape[1])
        at = torch.where(given, targets, 0).long()[:, None]
        logp = self.logs.gather(1, at)[:, 0]
        return torch.where(given, logp, 0.0), self.lse_off + 6 * U * torch.nan_to_num(logp, 0.0, 0.0, 0.0).abs() + 4 * U * torch.nan_to_num(
            self.z.gather(1, at)[:, 0], 0.0, 0.0, 0.0).abs()

    def gradient(self, targets, g, h, scale, lse_off, entropy_off, e, least):
        given = (targets >= 0) & (targets < self.z.shape[1]) & ~self.empty
        row = torch.arange(len(targets), device=targets.device)
        g = torch.where(given, g.double() if g is not None else 0.0, 0.0)[:, None]
        h = torch.where(self.empty, 0.0, h.double())[:, None] if h is not None else torch.zeros_like(g)
        logs = torch.where(self.p > 0, self.logs, 0.0)
        entropy = self.entropy[:, None]
        hit = torch.zeros_like(self.p)
        hit[row, torch.where(given, targets, 0).long()] = given.double()
        d = (g * (hit - self.p) - h * self.p * (logs + entropy)) * scale
        off = self.p * (2 * U * (logs.abs() + self.z.abs().clamp(max=1e9)) + lse_off[:, None] + 6 * U)
        inner = logs.abs() + entropy
        bound = g.abs() * off + h.abs() * (off * inner + self.p * (lse_off[:, None] + entropy_off[:, None] + 4 * U * inner + 2 * U * self.z.abs().clamp(max=1e9)))
        return d, scale * (bound + 4 * U * hit * g.abs()) + d.abs() * (e + 4 * U) + least


def held(got, want, bound, what):
    got, want, bound = got.double(), want.double(), bound.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, "%s: %g over" % (what, float(over.max()))


def alternatives(logits, scale, top):
    """Largest values first, the lowest index among equal ones, NaN last."""
    z = (logits.float() * scale).cpu().numpy() + np.float32(0)
    return np.stack([np.lexsort((np.arange(len(r)), -np.where(np.isnan(r), -np.inf, r).astype(np.float64), np.isnan(r)))[:top] for r in z])


def forward(ops, logits, targets, top=0, scale=1.0, **more):
    rows = len(logits)
    out = {k: torch.full((rows,), 7.0, device="cuda") for k in ("logp", "entropy", "lse")}
    if top:
        out["top_logp"] = torch.full((rows, top), 7.0, device="cuda")
        out["top_ids"] = torch.full((rows, top), -7, device="cuda", dtype=torch.int32)
    ops.token_logprobs_forward(logits, targets, scale=scale, **out, **more)
    return out


def check_forward(ops, logits, targets, top=0, scale=1.0):
    got, want = forward(ops, logits, targets, top, scale), Want(logits, scale)
    held(got["lse"], want.lse, want.lse_off, "lse")
    held(got["entropy"], want.entropy, want.entropy_off, "entropy")
    held(got["logp"], *want.logp(targets), "logp")
    if top:
        ids = alternatives(logits, np.float32(scale), top)
        assert np.array_equal(got["top_ids"].cpu().numpy(), ids), (logits.shape, top)
        at = torch.from_numpy(ids.astype(np.int64)).cuda()
        held(got["top_logp"], want.z.gather(1, at) - want.lse[:, None],
             want.lse_off[:, None] + 4 * U * torch.nan_to_num(want.z.gather(1, at), 0.0, 0.0, 0.0).abs().clamp(max=1e9), "top_logp")
    return got, want


VOCABS = [1, 2, 7, 64, 100, 1000, 2049, 8192, 8193, 20001, 32768, 50001, 131072]


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("rows,top,scale,pad", [(1, 8, 1.0, 0), (5, 3, 0.7, 3), (65, 1, 1.5, 0), (2, 64, 1.0, 1), (300, 0, 1.0, 0)])
def test_forward_is_the_definition(ops, kind, vocab, rows, top, scale, pad):
    logits = draw(rows + vocab, rows, vocab, TYPES[kind][0], pad=pad)
    targets = torch.randint(-1, vocab + 1, (rows,), generator=torch.Generator().manual_seed(vocab)).cuda()
    if rows % 2:
        targets = targets.int()
    check_forward(ops, logits, targets, min(top, vocab), scale)


def special(vocab, dtype):
    """Rows in which something is masked, missing or tied."""
    x = draw(vocab, 12, vocab, dtype)
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(3)
    x[0] = -INF                                                   # nothing left
    x[1] = low                                                    # the type's lowest value throughout: all alike
    x[2] = -INF
    x[2, vocab // 2] = 1.5                                        # one token left
    x[3, torch.rand(vocab, generator=g).cuda() < 0.97] = -INF
    x[4, torch.rand(vocab, generator=g).cuda() < 0.5] = low
    x[5] = 0.0                                                    # all alike
    x[6] = (torch.arange(vocab) % 3).to(dtype)                    # many of the largest
    x[7] = -torch.arange(vocab).to(dtype) / 16                    # descending
    x[8] = torch.arange(vocab).to(dtype) / 16                     # ascending
    x[9, ::2] = 0.0
    x[9, 1::2] = -0.0                                             # zeros of both signs are equal
    x[10, : max(1, vocab // 5)] = 11.0                            # a run of equal ones
    x[11, vocab // 3] = 60.0                                      # certain
    return x


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [3, 300, 5000, 33000, 70001])
@pytest.mark.parametrize("rows", [None, 1])
def test_masked_and_tied_rows(ops, kind, vocab, rows):
    x = special(vocab, TYPES[kind][0])
    targets = torch.tensor([0, 1, vocab // 2, 0, 2, 0, 2, 0, vocab - 1, 0, 0, vocab // 3], device="cuda").clamp(max=vocab - 1)
    if rows is None:
        check_forward(ops, x, targets, min(9, vocab))
    else:
        for i in range(len(x)):
            check_forward(ops, x[i:i + 1], targets[i:i + 1], min(20, vocab))


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [17, 9000, 40001])
def test_infinities_and_nan_stay_in_their_rows(ops, kind, vocab):
    dtype, e, least = TYPES[kind]
    x = draw(2, 4, vocab, dtype)
    x[1, 5] = math.nan
    x[2, 11] = INF
    targets = torch.tensor([1, 2, 3, 4], device="cuda")
    got = forward(ops, x, targets, 4)
    clean = forward(ops, x[::3].contiguous(), targets[::3].contiguous(), 4)
    for k in got:
        assert torch.equal(got[k][::3], clean[k]), k
        if k != "top_ids":
            assert bool(torch.isnan(got[k][1:3]).all()), k
    assert np.array_equal(got["top_ids"].cpu().numpy(), alternatives(x, np.float32(1), 4))
    d = torch.empty_like(x)
    weights = torch.ones(4, device="cuda")
    ops.token_logprobs_forward_train(x, targets, weights, d, d_entropy=weights)
    assert bool(torch.isfinite(d[::3]).all()) and bool(torch.isnan(d[1:3]).all())


def gradients(ops, x, targets, g, h, scale, together, in_place=False, dtype_out=None):
    d = x.clone() if in_place else torch.full_like(x, 7.0)
    source = d if in_place else x
    rows = len(x)
    if together:
        out = {k: torch.full((rows,), 7.0, device="cuda") for k in ("logp", "entropy", "lse")}
        ops.token_logprobs_forward_train(source, targets, g, d, d_entropy=h, scale=scale, **out)
        return d, out
    got = forward(ops, x, targets, 0, scale)
    ops.token_logprobs_backward(source, targets, got["lse"], g, d, entropy=got["entropy"], d_entropy=h, scale=scale)
    return d, got


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", VOCABS + [4097, 16385, 81921, 163841])
@pytest.mark.parametrize("rows,with_g,with_h,scale,pad", [(3, True, False, 1.0, 0), (2, True, True, 1.3, 5), (5, False, True, 0.5, 0)])
def test_gradient_is_the_formula(ops, kind, vocab, rows, with_g, with_h, scale, pad):
    dtype, e, least = TYPES[kind]
    scale = float(np.float32(scale))
    x = draw(vocab + rows, rows, vocab, dtype, pad=pad)
    targets = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(7)).cuda()
    targets[rows // 2] = -100                                     # no token there
    gen = torch.Generator().manual_seed(9)
    g = torch.randn(rows, generator=gen).cuda() if with_g else None
    h = torch.randn(rows, generator=gen).cuda() if with_h else None
    want = Want(x, scale)
    d, bound = want.gradient(targets, g, h, scale, want.lse_off, want.entropy_off, e, least)
    apart, _ = gradients(ops, x, targets, g, h, scale, False)
    held(apart, d, bound, "backward")
    once, out = gradients(ops, x, targets, g, h, scale, True)
    held(once, d, bound, "forward and backward")
    held(out["lse"], want.lse, want.lse_off, "lse")
    held(out["entropy"], want.entropy, want.entropy_off, "entropy")
    held(out["logp"], *want.logp(targets), "logp")
    for together, first in ((True, once), (False, apart)):
        assert torch.equal(gradients(ops, x, targets, g, h, scale, together, in_place=True)[0], first)


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [3, 300, 5000, 33000, 200001])
def test_gradient_of_masked_rows(ops, kind, vocab):
    dtype, e, least = TYPES[kind]
    x = special(vocab, dtype)
    targets = torch.full((len(x),), vocab // 2, device="cuda")
    g, h = torch.ones(len(x), device="cuda"), torch.full((len(x),), 0.5, device="cuda")
    want = Want(x, 1.0)
    # a token that is masked out in a row has a gradient of 1 - 0
    d, bound = want.gradient(targets, g, h, 1.0, want.lse_off, want.entropy_off, e, least)
    for together in (True, False):
        got = gradients(ops, x, targets, g, h, 1.0, together)[0]
        assert bool((got[0] == 0).all())
        held(got, d, bound, "together %s" % together)


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [64, 8000, 200001])
def test_a_row_of_the_lowest_value_has_even_probabilities(ops, kind, vocab):
    """A row that a mask of the type's lowest value has filled, where the logarithm of the sum is lost beside the logits."""
    dtype, e, least = TYPES[kind]
    x = torch.full((2, vocab), torch.finfo(dtype).min, dtype=dtype, device="cuda")
    d, out = gradients(ops, x, torch.tensor([3, -1], device="cuda"), torch.ones(2, device="cuda"), torch.ones(2, device="cuda"), 1.0, True)
    want = torch.full((2, vocab), -1.0 / vocab, dtype=torch.float64, device="cuda")
    want[0, 3] += 1.0
    want[1] = 0.0
    # log p + entropy cancels to within the roundings of both
    near = U * (vocab / 256 + 44 + 6 * math.log(vocab))
    held(d, want, 1.0 / vocab * near * (3 + math.log(vocab)) + want.abs() * e + least, "gradient")
    held(out["entropy"], torch.full((2,), math.log(vocab), device="cuda"), torch.full((2,), near, device="cuda"), "entropy")
    held(out["logp"], torch.tensor([-math.log(vocab), 0.0], device="cuda"), torch.full((2,), near, device="cuda"), "logp")


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [3000, 30001, 66001, 140000])
def test_huge_logits(ops, kind, vocab):
    """Exponents that one multiply-add does not hold, in all of a row or in some of its lanes only."""
    dtype, e, least = TYPES[kind]
    x = draw(vocab, 6, vocab, torch.float32)
    x[0] *= 3e6
    x[1, vocab // 2:] -= 5e6
    x[2, : vocab // 3] = -2e30
    x[3] += 7e6
    x[4] = -3e7
    x[4, 17] = -2.9e7
    x = x.to(dtype)
    targets = torch.tensor([0, 1, vocab - 1, 3, 17, vocab // 2], device="cuda")
    got, want = check_forward(ops, x, targets, 5)
    g = torch.ones(6, device="cuda")
    for h in (None, g):
        d, bound = want.gradient(targets, g, h, 1.0, want.lse_off, want.entropy_off, e, least)
        for together in (True, False):
            held(gradients(ops, x, targets, g, h, 1.0, together)[0], d, bound, "together %s" % together)


@gpu
@pytest.mark.parametrize("rows,vocab,kind", [(1100, 65536, "bf16"), (700, 100001, "f16"), (9000, 4003, "f32"), (3100, 20001, "bf16"), (2000, 16384, "f32")])
def test_logits_that_do_not_fit_the_caches(ops, rows, vocab, kind):
    dtype, e, least = TYPES[kind]
    x = draw(3, rows, vocab, dtype)
    targets = torch.arange(rows, device="cuda")
    got, want = check_forward(ops, x, targets, 2)
    g = torch.ones(rows, device="cuda")
    d, bound = want.gradient(targets, g, None, 1.0, want.lse_off, want.entropy_off, e, least)
    for together in (True, False):
        held(gradients(ops, x, targets, g, None, 1.0, together)[0], d, bound, "together %s" % together)


# rows enough for every unit, taken whole by as few lanes as hold them
@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vectors,more,top", [(4097, 0, 1), (5000, 3, 64), (7168, 1, 8), (7169, 0, 3), (4096, 3, 5), (2049, 0, 0)])
def test_rows_enough_to_be_taken_whole(ops, kind, vectors, more, top):
    dtype, rows = TYPES[kind][0], 1027
    vocab = vectors * (16 // dtype.itemsize) + more
    x = draw(5, rows, vocab, dtype, pad=5)
    x[::3] = x[::3].round()             # many equal values
    x[7] = -math.inf
    x[8, 5:] = -math.inf
    x[9] = torch.finfo(dtype).min
    x[10] = 0.0
    targets = (torch.arange(rows, device="cuda") * 7919) % (vocab + 2) - 1
    _, want = check_forward(ops, x, targets, 0, 0.8)
    if top:
        got = forward(ops, x, targets, top, 0.8)
        some = torch.cat([torch.arange(16), torch.arange(rows - 5, rows)])
        ids = torch.from_numpy(alternatives(x[some], np.float32(0.8), top).astype(np.int64)).cuda()
        assert torch.equal(got["top_ids"][some].long(), ids)
        z = want.z[some].gather(1, ids)
        held(got["top_logp"][some], z - want.lse[some][:, None],
             want.lse_off[some][:, None] + 4 * U * torch.nan_to_num(z, 0.0, 0.0, 0.0).abs().clamp(max=1e9), "top_logp")


@gpu
def test_gradient_against_differences(ops):
    rows, vocab, scale = 3, 23, 0.75
    x = draw(1, rows, vocab, torch.float32)
    targets = torch.tensor([4, 22, 0], device="cuda")
    g, h = torch.tensor([0.3, -1.0, 2.0], device="cuda"), torch.tensor([1.0, 0.5, -0.7], device="cuda")
    d = torch.empty_like(x)
    ops.token_logprobs_forward_train(x, targets, g, d, d_entropy=h, scale=scale)

    def f(v):
        logs = torch.log_softmax(v * scale, 1)
        entropy = -(logs.exp() * logs).sum(1)
        return float((g.double() * logs[torch.arange(rows), targets] + h.double() * entropy).sum())

    step = 1e-5
    for i in range(rows):
        for j in range(vocab):
            one = torch.zeros(rows, vocab, dtype=torch.float64, device="cuda")
            one[i, j] = step
            assert abs(float(d[i, j]) - (f(x.double() + one) - f(x.double() - one)) / (2 * step)) < 2e-6


@gpu
def test_offsets_beyond_32_bits(ops):
    """Rows that begin more than 2^31 values, and more than 2^32 bytes, behind the first."""
    stride, vocab = (1 << 30) + 40, 1000
    wide = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    x = wide.as_strided((3, vocab), (stride, 1))
    small = draw(4, 3, vocab, torch.bfloat16)
    x.copy_(small)
    targets = torch.tensor([1, 2, 3], device="cuda")
    a, b = forward(ops, x, targets, 5), forward(ops, small, targets, 5)
    for k in a:
        assert torch.equal(a[k], b[k]), k
    g = torch.ones(3, device="cuda")
    want = torch.empty_like(small)
    ops.token_logprobs_forward_train(small, targets, g, want)
    ops.token_logprobs_forward_train(x, targets, g, x)
    assert torch.equal(x, want)
    x.copy_(small)
    ops.token_logprobs_backward(x, targets, b["lse"], g, x)
    ops.token_logprobs_backward(small, targets, b["lse"], g, want)
    assert torch.equal(x, want)


@gpu
def test_no_rows_parts_left_out_and_another_stream(ops):
    none = torch.empty(0, 50, device="cuda")
    empty = torch.empty(0, device="cuda")
    ops.token_logprobs_forward(none, empty.long(), empty)
    ops.token_logprobs_backward(none, empty.long(), empty, empty, none)
    ops.token_logprobs_forward_train(none, empty.long(), empty, none)
    x = draw(5, 6, 3001, torch.float16)
    targets = torch.arange(6, device="cuda")
    whole = forward(ops, x, targets, 4)
    entropy = torch.empty(6, device="cuda")
    ops.token_logprobs_forward(x, None, None, entropy=entropy)                # no tokens given
    assert torch.equal(entropy, whole["entropy"])
    logp = torch.empty(6, device="cuda")
    ops.token_logprobs_forward(x.view(2, 3, 3001), targets.view(2, 3), logp)     # logp alone
    assert torch.equal(logp, whole["logp"])
    other, space = torch.cuda.Stream(), torch.empty(ops.token_logprobs_workspace_bytes(6, 3001, 4) // 4 + 4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        again = forward(ops, x, targets, 4, workspace=space)
        d = torch.empty_like(x)
        ops.token_logprobs_forward_train(x, targets, logp, d)
    other.synchronize()
    for k in whole:
        assert torch.equal(whole[k], again[k]), k
    same = torch.empty_like(x)
    ops.token_logprobs_forward_train(x, targets, logp, same)
    assert torch.equal(d, same)


@gpu
def test_the_same_bits_every_time(ops):
    x = draw(6, 4, 100003, torch.bfloat16)
    targets = torch.arange(4, device="cuda")
    first = forward(ops, x, targets, 16)
    for _ in range(5):
        again = forward(ops, x, targets, 16)
        for k in first:
            assert torch.equal(first[k], again[k]), k


def test_refusals():
    p, n = 256, None
    good = dict(logits=p, targets=p, logp=p, entropy=n, lse=n, top_logp=n, top_ids=n, type=1, wide=0, rows=4, vocab=10, stride=10, top=0, scale=1.0,
                ws=n, bytes=0, stream=n)
    for change, says in [(dict(type=3), "fp32, bf16 or half"), (dict(wide=2), "wide_targets"), (dict(rows=-1), "rows"), (dict(vocab=0), "logits"),
                         (dict(stride=9), "overlap"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=INF), "scale"),
                         (dict(scale=math.nan), "scale"), (dict(logits=n), "null"), (dict(targets=n), "together"), (dict(logp=n), "together"),
                         (dict(top=11), "alternatives"), (dict(top=-1), "alternatives"), (dict(top=65, vocab=100, stride=100), "alternatives"),
                         (dict(top=2), "null")]:
        assert capi.call_raw("pxh_token_logprobs_forward", *dict(good, **change).values()) == -1, change
        assert says in capi.last_error(), (change, capi.last_error())
    assert capi.call_raw("pxh_token_logprobs_forward", *dict(good, rows=0, logits=n).values()) == 0
    good = dict(logits=p, targets=p, lse=p, entropy=n, d_logp=p, d_entropy=n, dlogits=p, type=1, wide=0, rows=4, vocab=10, stride=10, d_stride=10,
                scale=1.0, stream=n)
    for change, says in [(dict(lse=n), "null"), (dict(dlogits=n), "null"), (dict(d_entropy=p), "null"), (dict(targets=n), "without targets"),
                         (dict(d_stride=9), "overlap")]:
        assert capi.call_raw("pxh_token_logprobs_backward", *dict(good, **change).values()) == -1, change
        assert says in capi.last_error(), (change, capi.last_error())
    good = dict(logits=p, targets=p, d_logp=p, d_entropy=n, dlogits=p, logp=n, entropy=n, lse=n, type=1, wide=0, rows=4, vocab=10, stride=10,
                d_stride=10, scale=1.0, stream=n)
    for change, says in [(dict(dlogits=n), "null"), (dict(targets=n), "without targets"), (dict(d_stride=9), "overlap"), (dict(type=7), "type")]:
        assert capi.call_raw("pxh_token_logprobs_forward_train", *dict(good, **change).values()) == -1, change
        assert says in capi.last_error(), (change, capi.last_error())


@pytest.mark.parametrize("bad,says", [(torch.zeros(2, 8), "must live on the GPU"), (np.zeros((2, 8)), "torch.Tensor expected"), (7, "torch.Tensor expected")])
def test_what_is_no_tensor_of_the_device_is_named(ops, bad, says):
    t = torch.zeros(2)
    for f in (lambda: ops.token_logprobs_forward(bad, t, t), lambda: ops.token_logprobs_backward(bad, t, t, t, t),
              lambda: ops.token_logprobs_forward_train(bad, t, t, t)):
        with pytest.raises(capi.PxError, match=says):
            f()


@gpu
def test_tensors_that_do_not_fit_are_refused(ops):
    x, t, v = torch.zeros(4, 9, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.long), torch.zeros(4, device="cuda")
    ids, tops = torch.zeros(4, 3, device="cuda", dtype=torch.int32), torch.zeros(4, 3, device="cuda")
    for f in (lambda: ops.token_logprobs_forward(x, t[:3], v), lambda: ops.token_logprobs_forward(x, t.float(), v),
              lambda: ops.token_logprobs_forward(x, t.cpu(), v), lambda: ops.token_logprobs_forward(x, t, v.double()),
              lambda: ops.token_logprobs_forward(x, t, v[:3]), lambda: ops.token_logprobs_forward(x, t, None),
              lambda: ops.token_logprobs_forward(x.double(), t, v), lambda: ops.token_logprobs_forward(x.t(), t, v),
              lambda: ops.token_logprobs_forward(x, t, v, top_ids=ids), lambda: ops.token_logprobs_forward(x, t, v, top_ids=ids.long(), top_logp=tops),
              lambda: ops.token_logprobs_forward(x, t, v, top_ids=ids, top_logp=tops[:3]), lambda: ops.token_logprobs_forward(x, t, v, scale=0.0),
              lambda: ops.token_logprobs_backward(x, t, v, v, x[:3]), lambda: ops.token_logprobs_backward(x, t, v, v, x.half()),
              lambda: ops.token_logprobs_backward(x, t, v, v, x, d_entropy=v), lambda: ops.token_logprobs_forward_train(x, t, v[:2], x),
              lambda: ops.token_logprobs_forward_train(x, t, v, None), lambda: ops.token_logprobs_forward_train(x, None, v, x)):
        with pytest.raises(capi.PxError):
            f()


@gpu
def test_alternatives_without_their_places_are_refused(ops):
    x, t, v = torch.zeros(4, 9, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.long), torch.zeros(4, device="cuda")
    tops = torch.full((4, 3), 7.0, device="cuda")
    for scale in (1.0, 1):          # by the native call, which leaves a whole number, and by the function's own checks
        with pytest.raises(capi.PxError, match="go together"):
            ops.token_logprobs_forward(x, t, v, top_logp=tops, scale=scale)


# (rows, vocabulary): a row in one part of few lanes, in parts joined by a wave and by a workgroup, whole by 1024 lanes, and by 512 of 8 and of 14 vectors
PLANS = [(2, 300), (3, 9000), (2, 131072), (70, 40001), (1030, 17001), (1030, 50001)]


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,vocab", PLANS + [(1, 200001)])
def test_rows_of_nothing_but_nan(ops, kind, rows, vocab):
    x = draw(1, rows, vocab, TYPES[kind][0])
    x[0] = math.nan
    if rows > 2:
        x[1] = math.nan
        x[1, ::3] = -INF
        x[rows - 1] = -INF
        x[rows - 1, vocab - 1] = math.nan
    bad = [0, 1, rows - 1] if rows > 2 else [0]
    targets = torch.full((rows,), 3, device="cuda")
    got = forward(ops, x, targets)
    for k in got:
        assert bool(torch.isnan(got[k][bad]).all()) and int(torch.isnan(got[k]).sum()) == len(bad), k
    ones = torch.ones(rows, device="cuda")
    for together in (True, False):
        for h in (None, ones):
            d, out = gradients(ops, x, targets, ones, h, 1.0, together)
            assert bool(torch.isnan(d[bad]).all()) and int(torch.isnan(d).any(1).sum()) == len(bad)
            for k in out:
                assert bool(torch.isnan(out[k][bad]).all()), k


def only(x, row, keep, values, fill):
    """Row `row` holds `fill` but for `values` at the places `keep`."""
    x[row] = fill
    for at, value in zip(keep, values):
        x[row, at] = value


def check_alternatives(ops, x, some, top, scale=1.0):
    """The places and log probabilities of rows `some`, on outputs that hold something else before."""
    rows = len(x)
    got = forward(ops, x, torch.zeros(rows, device="cuda", dtype=torch.long), top, scale)
    some = torch.tensor(some)
    ids = torch.from_numpy(alternatives(x[some.cuda()], np.float32(scale), top).astype(np.int64)).cuda()
    assert torch.equal(got["top_ids"][some.cuda()].long(), ids), top
    want = Want(x[some.cuda()], scale)
    z = want.z.gather(1, ids)
    held(got["top_logp"][some.cuda()], z - torch.where(want.empty, math.nan, want.lse)[:, None],
         want.lse_off[:, None] + 4 * U * torch.nan_to_num(z, 0.0, 0.0, 0.0).abs().clamp(max=1e9), "top_logp")


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,vocab", PLANS)
@pytest.mark.parametrize("top", [1, 4, 9, 20])
def test_alternatives_of_rows_with_nan(ops, kind, rows, vocab, top):
    """NaNs come last, by their places, and every place is written."""
    x = draw(2, rows, vocab, TYPES[kind][0])
    last = rows - 1
    x[0] = math.nan
    only(x, last, [vocab // 3, 5], [1.5, -2.0], math.nan)
    some = [0, last]
    if rows > 2:
        only(x, 1, [7], [1.0], math.nan)
        x[1, vocab // 2:] = -INF
        some.append(1)
    if rows > 69:
        x[2, 1::2] = math.nan
        only(x, 3, [2, 3, vocab - 2], [math.nan, math.nan, 1.0], -INF)
        only(x, 4, [vocab - 1], [math.nan], -INF)
        some += [2, 3, 4]
    check_alternatives(ops, x, some, top)


@gpu
def test_alternatives_of_a_row_in_seven_parts(ops):
    """Seven parts with nine alternatives each are joined by a wave."""
    x = draw(2, 300, 100001, torch.float32)
    x[0] = math.nan
    only(x, 1, [100000, 3], [1.0, 2.0], math.nan)
    only(x, 2, [50000], [1.0], -INF)
    x[3] = -INF
    for top in (9, 20):
        check_alternatives(ops, x, [0, 1, 2, 3, 299], top)


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,vocab", PLANS)
@pytest.mark.parametrize("top", [1, 3, 8, 9, 64])
def test_alternatives_of_few_allowed_or_equal_values(ops, kind, rows, vocab, top):
    dtype = TYPES[kind][0]
    x = draw(3, rows, vocab, dtype)
    g = torch.Generator().manual_seed(vocab)
    levels = lambda n: torch.randint(0, n, (vocab,), generator=g).to(dtype)          # noqa: E731
    made = [lambda r: only(x, r, torch.randint(0, vocab, (5,), generator=g).tolist(), [1.0, 3.0, 2.0, 3.0, -4.0], -INF),
            lambda r: x[r].copy_(levels(8)), lambda r: x[r].copy_(levels(3)), lambda r: x[r].fill_(-2.0),
            lambda r: (x[r].fill_(-INF), x[r, vocab // 3:vocab // 3 + 90].copy_(levels(90)[:90])),
            lambda r: (x[r].copy_(levels(2)), x[r, :vocab // 2].fill_(-INF)),
lambda r: x[r].copy_((torch.randn(vocab, generator=g) * 3 + 100).to(torch.bfloat16)),
            lambda r: only(x, r, [vocab - 1], [0.5], -INF), lambda r: only(x, r, [0, 1, 2], [-1.0, -1.0, -2.0], -INF),
            lambda r: only(x, r, [0, vocab // 2], [torch.finfo(dtype).min, torch.finfo(dtype).min], -INF),
            # a few columns of lanes hold a great many
            lambda r: x[r].copy_(torch.where(torch.arange(vocab) % 512 < 24, levels(200).float(), -INF).to(dtype)),
            lambda r: x[r].fill_(-INF)]
    some = []
    for r, make in zip(range(rows), made):
        make(r)
        some.append(r)
    check_alternatives(ops, x, some, top)
    if rows < 4:        # the others one by one
        for make in made[rows:]:
            make(0)
            check_alternatives(ops, x, [0], top)


def fastest(f, tries=5, calls=5):
    f()
    best = INF
    for _ in range(tries):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(calls):
            f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) / calls)
    return best


@gpu
@pytest.mark.parametrize("top", [3, 8])
def test_masked_and_tied_rows_take_no_passes_of_their_own(ops, top):
    """Rows of five allowed tokens, of four levels and of coarse values are not read `top` times over."""
    rows, vocab = 2048, 50001
    x = draw(4, rows, vocab, torch.float16)
    targets = torch.zeros(rows, device="cuda", dtype=torch.long)
    ordinary = fastest(lambda: forward(ops, x, targets, top))
    g = torch.Generator("cuda").manual_seed(4)
    levels = torch.randint(0, 4, (rows, vocab), device="cuda", generator=g).half()
    coarse = (torch.randn(rows, vocab, device="cuda", generator=g) * 2.5 + 90).bfloat16()
    allowed = torch.full_like(x, -INF)
    allowed[:, [17, 4000, 20000, 33333, 50000]] = 1.0
    for what, logits in (("levels", levels), ("coarse", coarse), ("allowed", allowed)):
        taken = fastest(lambda: forward(ops, logits, targets, top))
        assert taken < 2 * ordinary, (what, taken, ordinary)


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,vocab", PLANS)
def test_alternatives_of_a_row_of_the_lowest_value(ops, kind, rows, vocab):
    """All alike: every alternative has a vocabulary's share, though the logarithm of the sum is lost beside the logits."""
    x = draw(5, rows, vocab, TYPES[kind][0])
    x[0] = torch.finfo(x.dtype).min
    got = forward(ops, x, torch.full((rows,), 4, device="cuda"), 5)
    near = U * (vocab / 256 + 44 + 6 * math.log(vocab))
    assert torch.equal(got["top_ids"][0], torch.arange(5, device="cuda", dtype=torch.int32))
    for value in [*got["top_logp"][0].tolist(), float(got["logp"][0])]:
        assert abs(value + math.log(vocab)) <= near


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("vectors,more,top", [(4097, 1, 0), (4097, 7, 3), (5600, 3, 8), (6250, 1, 64), (7168, 5, 3), (7168, 7, 9)])
@pytest.mark.parametrize("begin", [0, 1])
def test_rows_off_a_word_with_values_behind_the_last_vector(ops, kind, vectors, more, top, begin):
    """Every other row begins between two words, and is read from its second value on: what a lane's first value is comes from the lane in
    front, and at a wave's first lane from memory."""
    dtype, rows = TYPES[kind][0], 1026
    vocab = vectors * 8 + more
    wide = draw(6, rows * vocab + begin, 1, dtype).view(-1)
    x = wide[begin:].view(rows, vocab)
    assert {(x.data_ptr() + 2 * vocab * r) % 4 for r in range(2)} == {0, 2}
    for r in (2, 3):
        x[r] = -INF
        x[r, 512 * (r + 5)] = 1.0                   # a wave's first value alone
        x[r + 2, 64 * 8::512 * 8] = math.nan        # ... no number
        x[r + 4, ::512] = 9.0                       # ... the largest
        x[r + 6, ::8] = 8.0
        x[r + 8, 7::8] = 8.0
        x[r + 10] = -INF
        x[r + 12, vectors * 8:] = 12.0              # behind the last vector
        x[r + 14] = torch.finfo(dtype).min
        x[r + 16, vocab - 1] = math.nan
        x[r + 18] = -INF
        x[r + 18, vectors * 8 - 1] = 2.0            # the last vector's last
        x[r + 20] = -INF
        x[r + 20, vectors * 8] = 2.0                # the first behind it
    targets = (torch.arange(rows, device="cuda") * 7919) % (vocab + 2) - 1
    targets[2:4] = torch.tensor([512 * 7, 512 * 8])
    clean = ~torch.isnan(x).any(1)
    got = forward(ops, x, targets, top)
    want = Want(x[clean], 1.0)
    held(got["lse"][clean], want.lse, want.lse_off, "lse")
    held(got["entropy"][clean], want.entropy, want.entropy_off, "entropy")
    held(got["logp"][clean], *want.logp(targets[clean]), "logp")
    for k in ("lse", "entropy"):
        assert bool(torch.isnan(got[k][~clean]).all()), k
    if top:
        some = torch.cat([torch.arange(30), torch.arange(rows - 4, rows)]).cuda()
        assert torch.equal(got["top_ids"][some].long().cpu(), torch.from_numpy(alternatives(x[some], np.float32(1), top).astype(np.int64)))

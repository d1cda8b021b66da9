"""Beam search with a scale: logits that a product of 32 bits would make equal or infinite.

Bounds.  u = 2^-24.  A row's sum of exponentials is in fp32, its logarithm within (n / 64 + 60) u of that of the row (n / 64 additions of a lane,
a tree, and the exponents' errors), and a score takes one rounding, u of it.  In a beam, and between beams of the same row, the sums are the
same to the bit: there the order is that of the logits and scores in 64 bits, and has to be exact."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


def run(ops, logits, scores, count, scale):
    batch = scores.shape[0]
    out = torch.full((batch, count), 7.0, device="cuda")
    parents, tokens = (torch.full((batch, count), 7, device="cuda", dtype=torch.int32) for _ in range(2))
    ops.beam_select(logits.cuda(), scores.cuda(), out, parents, tokens, scale=scale)
    return out.cpu(), parents.cpu(), tokens.cpu()


def exact(logits, scores, scale):
    """Scores in 64 bits, with the scale that an fp32 argument is."""
    beams, vocab = scores.shape[1], logits.shape[1]
    below = logits.double() - logits.double().amax(1, keepdim=True)
    z = below * float(np.float32(scale))
    z = z - z.exp().sum(1, keepdim=True).log() + scores.double().view(-1, 1)
    return z.view(-1, beams * vocab)


def neighbours(vocab, seed):
    """A row with up to 400 neighbouring fp32 numbers from 30 on, scattered."""
    g = torch.Generator().manual_seed(seed)
    n = min(400, vocab)
    row = torch.full((vocab,), -20.0)
    steps = torch.randperm(n, generator=g)
    row[torch.randperm(vocab, generator=g)[:n]] = torch.from_numpy(np.float32(30.0) + steps.numpy().astype(np.float32) * np.spacing(np.float32(30.0)))
    assert len(set(row[row > 0].tolist())) == n
    return row


@pytest.mark.parametrize("scale", [0.7, 0.3, 1.3])
@pytest.mark.parametrize("vocab,rows,count", [(9, 1, 5), (700, 3, 8), (5000, 2, 64), (5000, 70, 4), (20001, 2000, 3), (131072, 1, 4), (131072, 2, 64), (300000, 1, 8)])
def test_the_larger_of_two_neighbouring_logits_comes_first(ops, vocab, rows, count, scale):
    logits = torch.stack([neighbours(vocab, i) for i in range(min(rows, 8))]).repeat(-(-rows // 8), 1)[:rows].contiguous()
    products = logits[0][logits[0] > 0] * torch.tensor(scale)
    assert vocab < 700 or products.unique().numel() < products.numel()         # some are one number times the scale
    best, parents, tokens = run(ops, logits, torch.zeros(rows, 1), count, scale)
    want, at = torch.sort(exact(logits, torch.zeros(rows, 1), scale), dim=1, descending=True, stable=True)
    assert torch.equal(tokens.long(), at[:, :count]) and bool((parents == 0).all())
    bound = (vocab / 64 + 60) * U
    assert bool(((best.double() - want[:, :count]).abs() <= bound + U * want[:, :count].abs()).all())


@pytest.mark.parametrize("vocab", [700, 5000, 131072])
@pytest.mark.parametrize("beams,count", [(3, 3), (4, 20), (16, 64)])
def test_beams_of_one_row_whose_scores_differ_by_less_than_a_step(ops, vocab, beams, count):
    """A beam's score is ahead by less than a step of the logits times the scale: the neighbour of the other beam is in front of its second."""
    step = float(np.spacing(np.float32(30.0)))
    row = neighbours(vocab, 1)
    logits = row.repeat(2 * beams, 1)
    # in front of one another by thirds of a step times the scale; two items
    scores = (torch.arange(2 * beams).view(2, beams) % 7).float() * (0.7 * step / 3 * 1.07)
    best, parents, tokens = run(ops, logits, scores, count, 0.7)
    want, at = torch.sort(exact(logits, scores, 0.7), dim=1, descending=True, stable=True)
    # equal scores of beams of one row are equal in 64 bits too
    assert torch.equal(parents.long(), at[:, :count] // vocab) and torch.equal(tokens.long(), at[:, :count] % vocab)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [5, 2500, 40000, 300000])
def test_the_type_s_lowest_and_largest_values_times_a_scale(ops, vocab, dtype):
    lowest, largest = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits = torch.full((2, vocab), lowest, dtype=dtype)
    logits[1, 1], logits[1, vocab - 1] = largest, largest
    for scale in (1.3, 3e4):
        best, parents, tokens = run(ops, logits, torch.tensor([[-1.0], [-2.0]]), 3, scale)
        assert tokens[0].tolist() == [0, 1, 2] and parents[0].tolist() == [0, 0, 0]
        assert bool(((best[0] + 1.0 + math.log(vocab)).abs() < (vocab / 64 + 60) * U + U * (1 + math.log(vocab))).all())
        # two of the largest share it
        assert tokens[1, :2].tolist() == [1, vocab - 1] and parents[1, :2].tolist() == [0, 0]
        assert bool(((best[1, :2] + 2.0 + math.log(2)).abs() < 124 * U).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [5, 2500, 300000])
@pytest.mark.parametrize("scale", [1.0, 1.3, 3e4])
def test_what_is_left_as_minus_infinity_is_no_continuation(ops, vocab, dtype, scale):
    """Beside two of the type's largest value the others have next to nothing: a number, or less than those of fp32 are."""
    lowest, largest = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits = torch.full((1, vocab), lowest, dtype=dtype)
    logits[0, 1], logits[0, vocab - 1] = largest, largest
    below = (float(lowest) - float(largest)) * float(np.float32(scale))
    third = float(torch.tensor(below - math.log(2) - 2.0, dtype=torch.float64).float())
    there = third > -math.inf
    assert there == (dtype is torch.float16)
    best, parents, tokens = run(ops, logits, torch.tensor([[-2.0]]), 3, scale)
    assert tokens[0].tolist() == [1, vocab - 1, 0 if there else -1] and parents[0].tolist() == [0, 0, 0 if there else -1]
    assert float(best[0, 2]) == third

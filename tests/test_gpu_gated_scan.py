"""The gated linear recurrence, its gradients and its step, against the definition in 64 bits, token by token on the CPU.

Bounds.  u = 2^-24, e half a unit of the type.  z has the error of its exponential: (2 |update| + 8) u of itself.  A step rounds x - h, the
fused product and sum, and what the range's Z loses, which a state is multiplied by later: together 5 u (|h| + |x|), with a sixteenth of
what joins two waves; the error of what came before goes on as the state does, by 1 - z.  So the bound is a recurrence of its own:
E[t] = (1 - z) E[t - 1] + 5 u (|h| + |x|) + 2 z of_z (|h| + |x|).  The carry of the gradients has the same one."""
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


def draw(g, rows, width, dtype, std=1.0, mean=0.0, pad=0):
    return (torch.randn(rows, width + pad, generator=g) * std + mean).to(dtype).cuda()[:, :width]


def updates(g, rows, width, dtype, pad=0):
    """Channels that forget at once and channels that remember for thousands of tokens."""
    wide = torch.randn(rows, width + pad, generator=g) + torch.linspace(-9, 2, width + pad)[torch.randperm(width + pad, generator=g)]
    return wide.to(dtype).cuda()[:, :width]


class Want:
    """Everything in 64 bits, with its bounds, for sequences [(first, last + 1, slot or -1)]."""

    def __init__(self, sequences, x, update, gate=None, state=None, dy=None, d_final=None):
        to = lambda t: None if t is None else t.double().cpu()  # noqa: E731
        x, update, gate, state, dy, d_final = map(to, (x, update, gate, state, dy, d_final))
        rows, width = x.shape
        z, rest = 1 / (1 + torch.exp(-update)), 1 / (1 + torch.exp(update))
        of_z = (2 * update.abs() + 8) * U
        self.h, self.before = torch.zeros_like(x), torch.zeros_like(x)
        of_h, of_before = torch.zeros_like(x), torch.zeros_like(x)
        self.final = {}
        for first, last, slot in sequences:
            s = state[slot].clone() if state is not None and slot >= 0 else torch.zeros(width, dtype=torch.float64)
            err = torch.zeros(width, dtype=torch.float64)
            for t in range(first, last):
                self.before[t], of_before[t] = s, err
                s = rest[t] * s + z[t] * x[t]
                err = rest[t] * err + (5 * U + 2 * z[t] * of_z[t]) * (s.abs() + x[t].abs() + self.before[t].abs())
                self.h[t], of_h[t] = s, err
            if slot >= 0:
                self.final[slot] = (s, err)
        if gate is None:
            self.y, self.of_y = self.h, of_h
        else:
            sig = 1 / (1 + torch.exp(-gate))
            of_sig = (2 * gate.abs() + 8) * U
            g = gate * sig
            self.y = self.h * g
            self.of_y = of_h * g.abs() + self.y.abs() * (of_sig + 4 * U)
        if dy is None:
            return
        G, of_G = torch.zeros_like(x), torch.zeros_like(x)
        grad = dy if gate is None else dy * g
        of_grad = torch.zeros_like(x) if gate is None else grad.abs() * (of_sig + 4 * U)
        self.d_state = {}
        for first, last, slot in sequences:
            c = d_final[slot].clone() if d_final is not None and slot >= 0 else torch.zeros(width, dtype=torch.float64)
            err = torch.zeros(width, dtype=torch.float64)
            for t in reversed(range(first, last)):
                G[t] = grad[t] + c
                of_G[t] = err + of_grad[t] + 2 * U * (grad[t].abs() + c.abs())
                c = rest[t] * G[t]
                err = rest[t] * of_G[t] + (5 * U + 2 * z[t] * of_z[t]) * (G[t].abs() + grad[t].abs())
            if slot >= 0:
                self.d_state[slot] = (c, err)
        self.dx, self.of_dx = z * G, z * of_G + (z * G).abs() * (of_z + 2 * U)
        slope = z * rest
        w = (x - self.before) * slope
        self.dupdate = G * w
        self.of_dupdate = of_G * w.abs() + G.abs() * slope * (of_before + U * (x.abs() + self.before.abs())) + self.dupdate.abs() * (3 * of_z + 8 * U)
        if gate is not None:
            slope = sig * (1 + gate * (1 - sig))
            self.dgate = dy * self.h * slope
            self.of_dgate = dy.abs() * of_h * slope.abs() + (dy * self.h).abs() * (sig + (gate * sig * (1 - sig)).abs()) * (3 * of_sig + 8 * U)


def held(got, want, bound, what, e=2.0 ** -24, least=2.0 ** -140):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    over = (got - want).abs() - (bound + want.abs() * (e + U) + least)
    assert not bool(torch.isnan(got).any()), what
    assert over.numel() == 0 or float(over.max()) <= 0, "%s: %g over" % (what, float(over.max()))


UNIFORM = [(1, 1, 1), (3, 1, 5), (2, 16, 128), (1, 127, 130), (1, 128, 7), (1, 129, 64), (4, 64, 33), (2, 300, 257), (5, 37, 200), (1, 3001, 131),
           (2, 128, 64), (7, 2, 3), (40, 128, 2)]


@gpu
@pytest.mark.parametrize("count,tokens,width", UNIFORM)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("gated,pad", [(False, 0), (True, 3)])
def test_sequences_of_one_length(ops, count, tokens, width, kind, gated, pad):
    dtype, e, least = TYPES[kind]
    g = torch.Generator().manual_seed(count * 1000 + tokens + width)
    rows = count * tokens
    x, dy = draw(g, rows, width, dtype, pad=pad), draw(g, rows, width, dtype, 0.1, pad=2 * pad)
    u = updates(g, rows, width, dtype, pad)
    gate = draw(g, rows, width, dtype, 2.0, pad=pad) if gated else None
    want = Want([(i * tokens, (i + 1) * tokens, -1) for i in range(count)], x, u, gate, dy=dy)
    wide = [torch.full((rows, width + pad), 7.0, dtype=dtype, device="cuda") for _ in range(4)]
    y, dx, du, dgate = (t[:, :width] for t in wide)
    saved = ops.gated_scan_saved_like(x).fill_(7.0)
    ops.gated_scan_forward(x, u, y, gate=gate, sequences=count, saved=saved)
    held(y, want.y, want.of_y, "y", e, least)
    plain = torch.empty_like(x)
    ops.gated_scan_forward(x, u, plain, gate=gate, sequences=count)           # without what is saved
    assert torch.equal(plain, y)
    if pad == 0:
        # as [sequences, tokens, width]
        shape = (count, tokens, width)
        third = torch.empty(shape, dtype=dtype, device="cuda")
        ops.gated_scan_forward(x.view(shape), u.view(shape), third, gate=None if gate is None else gate.view(shape))
        assert torch.equal(third.view(rows, width), y)
    ops.gated_scan_backward(dy, x, u, saved, dx, du, gate=gate, dgate=dgate if gated else None, sequences=count)
    held(dx, want.dx, want.of_dx, "dx", e, least)
    held(du, want.dupdate, want.of_dupdate, "dupdate", e, least)
    if gated:
        held(dgate, want.dgate, want.of_dgate, "dgate", e, least)
    for t in wide[:3 + gated]:
        assert bool((t[:, width:] == 7).all())
    # in place, the same bits again
    if pad == 0:
        g0, u0, o0 = dy.clone(), u.clone(), None if gate is None else gate.clone()
        ops.gated_scan_backward(g0, x, u0, saved, g0, u0, gate=o0, dgate=o0, sequences=count)
        assert torch.equal(g0, dx) and torch.equal(u0, du) and (gate is None or torch.equal(o0, dgate))
        x0 = x.clone()
        ops.gated_scan_forward(x0, u, x0, gate=gate, sequences=count)
        assert torch.equal(x0, y)


# starts, rows
RAGGED = [([0, 5], 5), ([0, 0, 3, 3, 3, 4, 130, 130], 140), ([2, 2, 20, 21, 22, 150, 400, 401], 500), ([0] + list(range(0, 600, 3)), 700),
          ([0, 128, 256, 300, 640], 640), ([0, 0, 0], 0), ([7, 7, 7], 20), ([0, 1000, 1001, 1500], 1500), ([0, 16, 32, 33, 48, 64, 127, 128, 129], 129)]


@gpu
@pytest.mark.parametrize("starts,rows", RAGGED)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("width,gated,in_place", [(130, False, True), (65, True, False)])
def test_ragged_sequences_with_states_in_slots(ops, starts, rows, kind, width, gated, in_place):
    dtype, e, least = TYPES[kind]
    g = torch.Generator().manual_seed(rows + len(starts) + width)
    count = len(starts) - 1
    slots = torch.randperm(count + 3, generator=g)[:count]
    if count > 3:
        slots[1], slots[3] = -1, count + 3              # no state is kept
    kept = lambda s: int(s) if 0 <= int(s) < count + 3 else -1  # noqa: E731
    sequences = [(starts[i], starts[i + 1], kept(slots[i])) for i in range(count)]
    x, dy, u = draw(g, rows, width, dtype), draw(g, rows, width, dtype, 0.1), updates(g, rows, width, dtype)
    gate = draw(g, rows, width, dtype, 2.0) if gated else None
    state, d_final = draw(g, count + 3, width, torch.float32, 0.5), draw(g, count + 3, width, torch.float32, 0.1)
    want = Want(sequences, x, u, gate, state, dy, d_final)
    there = torch.tensor(starts, dtype=torch.int32, device="cuda"), slots.int().cuda()
    y, dx, du, dgate = (torch.full((rows, width), 7.0, dtype=dtype, device="cuda") for _ in range(4))
    saved = ops.gated_scan_saved_like(x)
    began = state.clone()
    final = state if in_place else torch.full_like(state, 9.0)
    edge = final.clone()
    ops.gated_scan_forward(x, u, y, gate=gate, starts=there[0], state=state, final=final, slots=there[1], saved=saved)
    covered = torch.zeros(rows, dtype=torch.bool)
    covered[starts[0]:starts[-1]] = True
    held(y.cpu()[covered], want.y[covered], want.of_y[covered], "y", e, least)
    assert bool((y.cpu()[~covered] == 7).all())
    for slot in range(count + 3):
        if slot in want.final:
            held(final[slot], want.final[slot][0], want.final[slot][1], "final")
        else:
            assert torch.equal(final[slot], edge[slot])
    d_state = d_final if in_place else torch.full_like(d_final, 9.0)
    edge = d_state.clone()
    ops.gated_scan_backward(dy, x, u, saved, dx, du, gate=gate, dgate=dgate if gated else None, starts=there[0], state=began, d_final=d_final,
                            d_state=d_state, slots=there[1])
    held(dx.cpu()[covered], want.dx[covered], want.of_dx[covered], "dx", e, least)
    held(du.cpu()[covered], want.dupdate[covered], want.of_dupdate[covered], "dupdate", e, least)
    if gated:
        held(dgate.cpu()[covered], want.dgate[covered], want.of_dgate[covered], "dgate", e, least)
    for t in (dx, du) + ((dgate,) if gated else ()):
        assert bool((t.cpu()[~covered] == 7).all())
    for slot in range(count + 3):
        if slot in want.d_state:
            held(d_state[slot], want.d_state[slot][0], want.d_state[slot][1], "d_state")
        else:
            assert torch.equal(d_state[slot], edge[slot])


@gpu
@pytest.mark.parametrize("rows,width,count,kind", [(40000, 130, 1, "bf16"), (40000, 2, 3, "f32"), (9000, 1100, 2, "f16"), (20000, 64, 160, "bf16")])
def test_long_sequences_from_chunk_to_chunk(ops, rows, width, count, kind):
    """Hundreds of workgroups that wait for each other; the same bits every time."""
    dtype, e, least = TYPES[kind]
    g = torch.Generator().manual_seed(rows)
    rows = rows // count * count
    x, dy, u = draw(g, rows, width, dtype), draw(g, rows, width, dtype, 0.1), updates(g, rows, width, dtype)
    u[:, 0] = -12.0                     # a memory of 10^5 tokens
    want = Want([(i * (rows // count), (i + 1) * (rows // count), -1) for i in range(count)], x, u, None, dy=dy)
    y, dx, du = (torch.empty_like(x) for _ in range(3))
    saved = ops.gated_scan_saved_like(x)
    ops.gated_scan_forward(x, u, y, sequences=count, saved=saved)
    ops.gated_scan_backward(dy, x, u, saved, dx, du, sequences=count)
    held(y, want.y, want.of_y, "y", e, least)
    held(dx, want.dx, want.of_dx, "dx", e, least)
    held(du, want.dupdate, want.of_dupdate, "dupdate", e, least)
    space = torch.empty(ops.gated_scan_workspace_bytes(rows, width) + 16, dtype=torch.uint8, device="cuda").fill_(1)
    for _ in range(5):
        again, saved2, dx2, du2 = torch.empty_like(y), torch.empty_like(saved), torch.empty_like(dx), torch.empty_like(du)
        ops.gated_scan_forward(x, u, again, sequences=count, saved=saved2, workspace=space)
        ops.gated_scan_backward(dy, x, u, saved2, dx2, du2, sequences=count, workspace=space)
        assert torch.equal(again, y) and torch.equal(saved2, saved) and torch.equal(dx2, dx) and torch.equal(du2, du)


@gpu
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 130), (64, 4096), (513, 77), (2, 4099)])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("gated,with_slots,pad", [(False, False, 0), (True, True, 5)])
def test_a_step_is_a_sequence_of_one_token(ops, rows, width, kind, gated, with_slots, pad):
    dtype, e, least = TYPES[kind]
    g = torch.Generator().manual_seed(rows + width)
    x, u = draw(g, rows, width, dtype, pad=pad), updates(g, rows, width, dtype, pad)
    gate = draw(g, rows, width, dtype, 2.0, pad=pad) if gated else None
    state = draw(g, rows + 4, width, torch.float32)
    slots = torch.randperm(rows + 4, generator=g)[:rows] if with_slots else torch.arange(rows)
    if with_slots and rows > 2:
        slots[2] = -1
    want = Want([(i, i + 1, int(slots[i])) for i in range(rows)], x, u, gate, state)
    before, y = state.clone(), torch.full((rows, width + pad), 7.0, dtype=dtype, device="cuda")
    ops.gated_scan_step(x, u, y[:, :width], state, gate=gate, slots=slots.int().cuda() if with_slots else None)
    held(y[:, :width], want.y, want.of_y, "y", e, least)
    assert bool((y[:, width:] == 7).all())
    for slot in range(rows + 4):
        if slot in want.final:
            held(state[slot], want.final[slot][0], want.final[slot][1], "state")
        else:
            assert torch.equal(state[slot], before[slot])
    # and what the forward pass makes of it, to the bit
    y2 = torch.empty_like(y[:, :width])
    ops.gated_scan_forward(x, u, y2, gate=gate, sequences=rows, state=before, final=before, slots=slots.int().cuda() if with_slots else None)
    assert torch.equal(y2, y[:, :width]) and torch.equal(before, state)


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_what_is_no_number_is_not_forgotten(ops, kind):
    """Updates after a few hundred of which nothing of a number is left: what is none stays, from chunk to chunk."""
    dtype = TYPES[kind][0]
    g = torch.Generator().manual_seed(6)
    starts = [0, 50, 5050, 5100]
    rows, width = starts[-1], 70
    x, u, dy = draw(g, rows, width, dtype), draw(g, rows, width, dtype, 2.0), draw(g, rows, width, dtype, 0.1)
    there = torch.tensor(starts, dtype=torch.int32, device="cuda")
    x[300, 3], x[301, 4], x[4000, 5], u[2000, 6] = float("nan"), float("inf"), float("-inf"), float("nan")
    dy[4500, 7], dy[100, 8], dy[4900, 9] = float("nan"), float("inf"), float("-inf")
    y, dx, du, saved = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), ops.gated_scan_saved_like(x)
    ops.gated_scan_forward(x, u, y, starts=there, saved=saved)
    ops.gated_scan_backward(dy, x, u, saved, dx, du, starts=there)
    none = torch.zeros(rows, width, dtype=torch.bool)
    none[300:5050, 3], none[302:5050, 4], none[4001:5050, 5], none[2000:5050, 6] = True, True, True, True
    assert torch.equal(torch.isnan(y).cpu(), none)
    got = torch.isnan(dx).cpu()
    # against the tokens, to the sequence's first one: from there where it is no number, from the one in front of an infinite one
    assert bool(got[50:4501, 7].all()) and not bool(got[4501:, 7].any()) and not bool(got[:50, 7].any())
    for column, first in ((8, 100), (9, 4900)):
        # (an infinite G times 1 - z is infinite where z < 1, and so is what is added to it: no number where signs meet or z is 1)
        lost = ~torch.isfinite(dx[:, column].cpu())
        assert bool(lost[50:first + 1].all()) and not bool(lost[first + 1:].any()) and not bool(lost[:50].any())


@gpu
@pytest.mark.parametrize("count", [62, 63, 64, 200, 5000])
def test_many_ragged_sequences(ops, count):
    """Some without a token, some of many: against each by itself, where only the last bits of h can differ."""
    g = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 40, (count,), generator=g)
    lengths[count // 2], lengths[3], lengths[4] = 700, 0, 0
    starts = torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)]) + 5
    rows, width = int(starts[-1]) + 9, 66
    x, u = draw(g, rows, width, torch.float32), draw(g, rows, width, torch.float32)
    state = draw(g, count, width, torch.float32)
    y, final = torch.full_like(x, 7.0), torch.empty_like(state)
    ops.gated_scan_forward(x, u, y, starts=starts.int().cuda(), state=state, final=final)
    z, h = torch.sigmoid(u.double()).cpu(), state.double().cpu()
    want, xs = torch.full((rows, width), 7.0, dtype=torch.float64), x.double().cpu()
    for t in range(int(lengths.max())):
        on = (lengths > t).nonzero()[:, 0]
        at = starts[on] + t
        h[on] = h[on] + z[at] * (xs[at] - h[on])
        want[at] = h[on]
    # a step rounds h by 2^-23 of what is there at most, of which less than all is kept: 700 of them
    bound = 700 * 2.0 ** -23 * 6
    assert float((y.double().cpu() - want).abs().max()) < bound and float((final.double().cpu() - h).abs().max()) < bound
    assert bool((y[:5] == 7).all()) and bool((y[-9:] == 7).all())


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_what_is_no_number_stays_in_its_sequence_and_closed_gates_keep_the_state(ops, kind):
    dtype = TYPES[kind][0]
    g = torch.Generator().manual_seed(5)
    lengths = [300, 40, 1, 500, 3, 90]
    starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    rows, width = starts[-1], 70
    x, u, dy = draw(g, rows, width, dtype), updates(g, rows, width, dtype), draw(g, rows, width, dtype, 0.1)
    there = torch.tensor(starts, dtype=torch.int32, device="cuda")

    def run(x, u, dy):
        y, dx, du, saved = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), ops.gated_scan_saved_like(x)
        ops.gated_scan_forward(x, u, y, starts=there, saved=saved)
        ops.gated_scan_backward(dy, x, u, saved, dx, du, starts=there)
        return y, dx, du

    good = run(x, u, dy)
    bx, bu, bdy = x.clone(), u.clone(), dy.clone()
    bx[starts[1] + 3, 5] = float("nan")
    bx[starts[3] + 100, 6] = float("inf")
    bu[starts[3] + 200, 7] = float("nan")
    bdy[starts[3] + 250] = float("nan")
    bad = run(bx, bu, bdy)
    for a, b in zip(good, bad):
        for i in (0, 2, 4, 5):
            assert torch.equal(a[starts[i]:starts[i + 1]], b[starts[i]:starts[i + 1]])
    assert bool(torch.isnan(bad[0][starts[1] + 3:starts[2], 5]).all()) and bool(torch.isnan(bad[0][starts[3] + 200:starts[4], 7]).all())
    assert not bool(torch.isnan(bad[0][starts[1]:starts[1] + 3]).any())
    # updates of minus infinity and of the type's lowest value: the state as it was; of plus infinity: x
    state = draw(g, 1, width, torch.float32)
    for low in (float("-inf"), torch.finfo(dtype).min):
        u = torch.full((200, width), low, device="cuda").to(dtype)
        final, y = torch.empty_like(state), torch.empty(200, width, dtype=dtype, device="cuda")
        ops.gated_scan_forward(x[:200], u, y, state=state, final=final)
        assert torch.equal(final, state) and torch.equal(y, state.to(dtype).expand(200, width))
        saved, dx, du = ops.gated_scan_saved_like(u), torch.empty_like(y), torch.empty_like(y)
        d = torch.empty_like(state)
        ops.gated_scan_forward(x[:200], u, y, state=state, saved=saved)
        ops.gated_scan_backward(dy[:200], x[:200], u, saved, dx, du, state=state, d_state=d)
        assert bool((dx == 0).all()) and bool((du == 0).all())
        total = dy[:200].double().sum(0)
        assert bool(((d[0].double() - total).abs() <= 200 * U * dy[:200].double().abs().sum(0)).all())
    u = torch.full((200, width), float("inf"), device="cuda").to(dtype)
    ops.gated_scan_forward(x[:200], u, y, state=state)
    assert bool(((y.double() - x[:200].double()).abs() <= (x[:200].double().abs() + 4) * (TYPES[kind][1] + 4 * U)).all())


@gpu
def test_the_gradients_are_those_of_differences(ops):
    """Central differences of the definition in 64 bits."""
    rows, width, step = 23, 3, 1e-6
    g = torch.Generator().manual_seed(3)
    starts = [0, 6, 6, 23]
    leaves = {k: draw(g, rows, width, torch.float32) for k in ("x", "update", "gate", "dy")}
    leaves["state"], leaves["d_final"] = draw(g, 3, width, torch.float32), draw(g, 3, width, torch.float32)
    there = torch.tensor(starts, dtype=torch.int32, device="cuda")
    x, u, gate = leaves["x"], leaves["update"], leaves["gate"]
    y, saved, final = torch.empty_like(x), ops.gated_scan_saved_like(x), torch.empty_like(leaves["state"])
    ops.gated_scan_forward(x, u, y, gate=gate, starts=there, state=leaves["state"], final=final, saved=saved)
    grads = {k: torch.empty_like(leaves[k]) for k in ("x", "update", "gate", "state")}
    ops.gated_scan_backward(leaves["dy"], x, u, saved, grads["x"], grads["update"], gate=gate, dgate=grads["gate"], starts=there,
                            state=leaves["state"], d_final=leaves["d_final"], d_state=grads["state"])
    at = {k: t.double().cpu() for k, t in leaves.items()}
    sequences = [(starts[i], starts[i + 1], i) for i in range(3)]

    def loss():
        w = Want(sequences, at["x"], at["update"], at["gate"], at["state"])
        return float((w.y * at["dy"]).sum() + sum((w.final[i][0] * at["d_final"][i]).sum() for i in range(3)))

    for name, grad in grads.items():
        flat, got = at[name].view(-1), grad.cpu().view(-1)
        for i in range(0, flat.numel(), 4 if name != "state" else 1):
            was = float(flat[i])
            flat[i] = was + step
            up = loss()
            flat[i] = was - step
            down = loss()
            flat[i] = was
            assert abs((up - down) / (2 * step) - float(got[i])) < 1e-5, (name, i)


@gpu
def test_on_another_stream_and_in_a_graph(ops):
    """Two calls at once on two streams with workspaces of their own, and captured passes, replayed with other work between."""
    g = torch.Generator().manual_seed(9)
    rows, width = 5000, 300
    x, u = draw(g, rows, width, torch.bfloat16), updates(g, rows, width, torch.bfloat16)
    spaces = [torch.empty(ops.gated_scan_workspace_bytes(rows, width), dtype=torch.uint8, device="cuda") for _ in range(3)]

    def run(space, x, sequences=2):
        y, saved, dx, du = torch.empty_like(x), ops.gated_scan_saved_like(x), torch.empty_like(x), torch.empty_like(x)
        ops.gated_scan_forward(x, u, y, sequences=sequences, saved=saved, workspace=space)
        ops.gated_scan_backward(y, x, u, saved, dx, du, sequences=sequences, workspace=space)
        return y, dx, du

    want = run(spaces[0], x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for _ in range(4):
        for stream, space in zip(streams, spaces):
            with torch.cuda.stream(stream):
                results.append(run(space, x))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    inside = x.clone()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            captured = run(spaces[2], inside)
    for i in range(4):
        inside.copy_(x * (i + 1))
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = run(spaces[0], inside)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


@gpu
def test_what_is_refused(ops):
    x = torch.zeros(12, 8, device="cuda")
    state = torch.zeros(3, 8, device="cuda")
    saved = ops.gated_scan_saved_like(x)
    starts, slots = torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    y = x.clone()
    big = torch.zeros(400, 8, device="cuda")
    for call, message in [
            (lambda: ops.gated_scan_forward(x, None, y), "update is required"),
            (lambda: ops.gated_scan_forward(x, x.half(), y), "update must be"),
            (lambda: ops.gated_scan_forward(x, x, y[:5]), "y must be"),
            (lambda: ops.gated_scan_forward(x, x, y, gate=x[:, :4]), "gate must be"),
            (lambda: ops.gated_scan_forward(x, x, y, sequences=5), "not 5 sequences of one length"),
            (lambda: ops.gated_scan_forward(x, x, y, sequences=0), "0 sequences"),
            (lambda: ops.gated_scan_forward(x, x, y, sequences=-1), "-1 sequences"),
            (lambda: ops.gated_scan_forward(x, x, y, starts=starts.long()), "starts must be"),
            (lambda: ops.gated_scan_forward(x, x, y, starts=starts[:0]), "one more value"),
            (lambda: ops.gated_scan_forward(x, x, y, starts=starts.cpu()), "must live on the GPU"),
            (lambda: ops.gated_scan_forward(x, x, y, sequences=4, state=state), "3 slots for 4 sequences"),
            (lambda: ops.gated_scan_forward(x, x, y, starts=starts, state=state, final=state[:2]), "final must be"),
            (lambda: ops.gated_scan_forward(x, x, y, starts=starts, state=state[:, :4].contiguous()), "state must be"),
            (lambda: ops.gated_scan_forward(x, x, y, starts=starts, state=state.half()), "state must be"),
            (lambda: ops.gated_scan_forward(x, x, y, starts=starts, slots=slots), "slots without states"),
            (lambda: ops.gated_scan_forward(x, x, y, starts=starts, state=state, slots=slots[:1]), "slots must hold 2"),
            (lambda: ops.gated_scan_forward(x, x, y, saved=saved[:, :4].contiguous()), "saved must hold"),
            (lambda: ops.gated_scan_forward(x[:1].expand(12, 8), x, y), "overlap"),
            (lambda: ops.gated_scan_forward(big, big, big.clone(), workspace=torch.empty(8, device="cuda")), "workspace too small"),
            (lambda: ops.gated_scan_backward(x, x, x, saved, y, y.clone(), gate=x), "gate and dgate go together"),
            (lambda: ops.gated_scan_backward(x, x, x, None, y, y.clone()), "null pointer"),
            (lambda: ops.gated_scan_backward(x, x, x, saved, y, y.half()), "dupdate must be"),
            (lambda: ops.gated_scan_step(x, x, y, None), "state is required"),
            (lambda: ops.gated_scan_step(x, x, y, state), "3 slots for 12 sequences"),
            (lambda: ops.gated_scan_step(x, x, y, state, slots=slots), "slots must hold 12")]:
        with pytest.raises(capi.PxError, match=message):
            call()

"""AdamW over a table of tensors, states in 32 and in 8 bits, against the formulas in 64 bits.

Bounds, u = 2^-24: m is a sum of two products, within 3 u of the sum of their magnitudes M; v is a sum of positive ones, within
5 u of itself, and its root within 4 u; the step m / c1 / (root / c2 + eps) is within 12 u of M / c1 / (root / c2 + eps), and the
weight has three roundings more.  A state in 8 bits is one of the two e4m3 values around what it is rounded from, that one known
to 8 u; its scale is within 8 u."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from pixienn_amd import capi

gpu = pytest.mark.gpu
U = 2.0 ** -24
SIZES = [1, 3, 4, 255, 256, 257, 0, 1000, 4095, 4096, 4097, 8192, 20001, 70000]
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


def normal(g, n, std):
    return (torch.randn(n, generator=g) * std).cuda()


def off_grid(x, by):
    """The same values in a tensor that begins `by` values into a buffer."""
    wide = torch.zeros(x.numel() + by + 3, dtype=x.dtype, device=x.device)
    wide[by:by + x.numel()] = x
    return wide[by:by + x.numel()]


def encoded(x):
    """x as e4m3 values with a scale per 256."""
    blocks = -(-x.numel() // 256)
    wide = torch.nn.functional.pad(x, (0, blocks * 256 - x.numel())).view(blocks, 256)
    scale = (wide.abs().amax(1) / 448.0).clamp(min=2.0 ** -126)
    code = (wide / scale[:, None]).to(torch.float8_e4m3fn)
    return code.view(-1)[: x.numel()].clone(), scale


def decoded(code, scale):
    return code.double() * scale.double().repeat_interleave(256)[: code.numel()]


class Model:
    def __init__(self, ops, bits, sizes=SIZES, kinds=("f32", "bf16", "f16"), copies=True, unaligned=True, seed=1, gradient=1e-2):
        g = torch.Generator().manual_seed(seed)
        self.bits = bits
        place = (lambda x, i: off_grid(x, i % 4)) if unaligned else (lambda x, i: x)
        self.w = [place(normal(g, n, 0.05), i) for i, n in enumerate(sizes)]
        self.d = [place((normal(g, n, gradient)).to(DTYPES[kinds[i % len(kinds)]]), i + 1) for i, n in enumerate(sizes)]
        m = [normal(g, n, gradient / 3) for n in sizes]
        root = [normal(g, n, 0.1).exp_() * gradient for n in sizes]
        self.copy = [place(torch.zeros(n, dtype=(torch.bfloat16, torch.float16)[i % 2], device="cuda"), i + 2) if i % 3 or not unaligned else None
                     for i, n in enumerate(sizes)] if copies else None
        self.decay = [i % 2 == 0 for i in range(len(sizes))]
        if bits == 8:
            pairs = [encoded(x) for x in m], [encoded(x) for x in root]
            self.m, self.v = ([place(c.view(torch.uint8), i + 1).view(torch.float8_e4m3fn) for i, (c, _) in enumerate(p)] for p in pairs)
            self.ms, self.vs = ([s for _, s in p] for p in pairs)
        else:
            self.m, self.v = [place(x, i + 3) for i, x in enumerate(m)], [place(x.square(), i + 2) for i, x in enumerate(root)]
            self.ms = self.vs = None
        self.table = ops.AdamwTable(self.w, self.d, self.m, self.v, self.ms, self.vs, self.copy, self.decay)

    def states(self):
        if self.bits == 32:
            return [x.double() for x in self.m], [x.double() for x in self.v]
        return [decoded(*x) for x in zip(self.m, self.ms)], [decoded(*x).square() for x in zip(self.v, self.vs)]

    def everything(self):
        lists = [self.w, self.d, [x.view(torch.uint8) for x in self.m], [x.view(torch.uint8) for x in self.v], self.ms or [], self.vs or [],
                 [c for c in self.copy or [] if c is not None]]
        return [t.clone() for group in lists for t in group]


def wanted(model, t, lr, beta1, beta2, eps, decay, d_scale, max_norm):
    """What a step leaves of every tensor in 64 bits, with the bounds."""
    f = lambda x: float(np.float32(x))  # noqa: E731
    lr, eps, d_scale, max_norm, shrink = f(lr), f(eps), f(d_scale), f(max_norm), f(lr) * f(decay)
    norm = math.sqrt(sum(float((d.double() * d_scale).square().sum()) for d in model.d))
    factor = max_norm / norm if max_norm and norm > max_norm else 1.0
    ms, vs = model.states()
    result = []
    for w, d, m, v, flag in zip(model.w, model.d, ms, vs, model.decay):
        g = d.double() * d_scale * factor
        size = (beta1 * m).abs() + ((1 - beta1) * g).abs()
        m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
        root = v.sqrt()
        bottom = (1 - beta1 ** t) * (root / math.sqrt(1 - beta2 ** t) + eps)
        new = w.double() + lr * m / bottom - (shrink * w.double() if flag else 0.0)
        result.append((new, lr * size / bottom * 14 * U + 4 * U * (w.double().abs() + new.abs()), m, 5 * U * size, v, root))
    return norm, result


def held(got, want, bound, what):
    assert bool(((got.double() - want).abs() <= bound).all()), what


def check_step(model, t=7, lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, decay=0.1, d_scale=0.5, max_norm=0.0, seed=5):
    norm, want = wanted(model, t, lr, beta1, beta2, eps, decay, d_scale, max_norm)
    got_norm = torch.full((1,), 7.0, device="cuda")
    before = [d.clone() for d in model.d]
    model.table.update(t, lr, beta1, beta2, eps, decay, d_scale=d_scale, max_norm=max_norm, norm_out=got_norm, seed=seed)
    assert abs(float(got_norm) - norm) <= norm * 8 * U
    for i, (w, bound, m, m_bound, v, root) in enumerate(want):
        held(model.w[i], w, bound, "w of %d" % i)
        assert torch.equal(model.d[i], before[i])
        if model.copy and model.copy[i] is not None:
            assert torch.equal(model.copy[i], model.w[i].to(model.copy[i].dtype)), i
        if model.bits == 32:
            held(model.m[i], m, m_bound, "m of %d" % i)
            held(model.v[i], v, 6 * U * v, "v of %d" % i)
        elif m.numel():
            check_codes(model.m[i], model.ms[i], m, m_bound, False)
            check_codes(model.v[i], model.vs[i], root, 5 * U * root, True)


def check_codes(code, scale, exact, bound, positive):
    n = exact.numel()
    wide = torch.nn.functional.pad(exact, (0, len(scale) * 256 - n)).view(-1, 256)
    want = (wide.abs().amax(1) / 448.0).clamp(min=2.0 ** -126)
    slack = torch.nn.functional.pad(bound, (0, len(scale) * 256 - n)).view(-1, 256).amax(1) / 448.0
    assert bool(((scale.double() - want).abs() <= slack + 8 * U * want).all())
    s = scale.double().repeat_interleave(256)[:n]
    x, off = exact / s, bound / s + 8 * U * (exact / s).abs()
    step = torch.exp2(torch.floor(torch.log2((x.abs() - off).clamp(min=2.0 ** -6))) - 3)       # of e4m3 at x
    got = code.double()
    assert bool(torch.isfinite(got).all())
    # one of the neighbours: less than a step away (a whole one where the step doubles between them), and on the other side never
    assert bool(((got - x).abs() < 2 * step + off).all())
    lower = torch.floor((x.abs() - off).clamp(min=0) / step) * step
    upper = torch.ceil((x.abs() + off) / step) * step
    assert bool(((got.abs() >= lower - 1e-12) & (got.abs() <= torch.clamp(upper + step * (off > 0) * ((x.abs() + off) > (x.abs() - off) * (1 + 2.0 ** -3)), max=448.0) + 1e-12)).all())
    assert bool(((got == 0) | (torch.sign(got) == torch.sign(x)) | (x.abs() <= off)).all())
    if positive:
        assert bool(((got > 0) | (exact == 0)).all())


@gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("kinds", [("f32",), ("bf16",), ("f16",), ("f32", "bf16", "f16")])
@pytest.mark.parametrize("max_norm,unaligned", [(0.0, True), (0.3, True), (1e6, False)])
def test_a_step_is_the_formula(ops, bits, kinds, max_norm, unaligned):
    model = Model(ops, bits, kinds=kinds, unaligned=unaligned)
    assert model.table.count == len(SIZES) - 1
    check_step(model, max_norm=max_norm)
    check_step(model, t=8, max_norm=max_norm, seed=6, decay=0.0)
    check_step(model, t=1, beta1=0.0, beta2=0.999, eps=1e-3, max_norm=max_norm, d_scale=-1.0, seed=7)


@gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_a_table_that_streams_past_the_caches(ops, bits):
    check_step(Model(ops, bits, sizes=[9000001, 300], kinds=("bf16",), unaligned=bits == 8), max_norm=0.1)


@gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors(ops, bits):
    check_step(Model(ops, bits, sizes=[1 + 37 * i % 600 for i in range(3000)], kinds=("f32", "f16")), max_norm=0.5)


@gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_from_zero_states(ops, bits):
    """The first step, with gradients of zero among the others: zeros stay, and nothing is divided by zero."""
    sizes = [300, 5000]
    ws = [torch.ones(n, device="cuda") for n in sizes]
    ds = [torch.linspace(-1, 1, n, device="cuda") * (torch.arange(n, device="cuda") % 3 != 0) for n in sizes]
    states = ops.adamw_states(ws, bits)
    table = ops.AdamwTable(ws, ds, **states)
    table.update(1, 1e-2, seed=1)
    for i, (w, d) in enumerate(zip(ws, ds)):
        want = 1.0 + 1e-2 * torch.sign(d) * (d.abs() / (d.abs() + 1e-8))
        assert float((w - want).abs().max()) < 1e-6
        assert torch.equal(states["vs"][i].float() == 0, d == 0) and bool((states["ms"][i].float()[d == 0] == 0).all())


@gpu
def test_no_root_rounds_to_zero(ops):
    """Values far below their block's largest one: a root keeps at least the least value there is."""
    n = 512
    d = torch.full((n,), 1e-9, device="cuda")
    d[0] = 1.0
    w = torch.zeros(n, device="cuda")
    states = ops.adamw_states([w], 8)
    table = ops.AdamwTable([w], [d], **states)
    for t in range(1, 30):
        table.update(t, 1e-3, eps=0.0, seed=t)
        assert bool((states["vs"][0].float() > 0).all()) and bool(torch.isfinite(w).all())
    # the quotient of two states never exceeds what 32 bits allow: a step is a few lr at most
    assert float(w.abs().max()) < 29 * 1e-3 * 8


@gpu
def test_rounding_has_no_drift(ops):
    """The mean over many seeds is what was rounded, within five deviations of a rounding that moves by a step at most."""
    n, tries = 2048, 400
    g = torch.Generator().manual_seed(3)
    d = normal(g, n, 1.0)
    sums = torch.zeros(2, n, dtype=torch.float64, device="cuda")
    squares = torch.zeros_like(sums)
    for seed in range(tries):
        w = torch.zeros(n, device="cuda")
        states = ops.adamw_states([w], 8)
        ops.AdamwTable([w], [d], **states).update(1, 1e-3, 0.9, 0.99, seed=seed)
        got = torch.stack([decoded(states["ms"][0], states["m_scales"][0]), decoded(states["vs"][0], states["v_scales"][0])])
        sums += got
        squares += got * got
    mean = sums / tries
    want = torch.stack([d.double() * (1 - float(np.float32(0.9))), d.double().abs() * math.sqrt(1 - float(np.float32(0.99)))])
    normal_range = want.abs() > torch.stack([states["m_scales"][0], states["v_scales"][0]]).double().repeat_interleave(256, 1) * 2.0 ** -6
    step = want.abs() / 8
    off = (mean - want).abs()
    assert bool((off[normal_range] <= (5 * step / 2 / math.sqrt(tries) + 1e-6 * want.abs())[normal_range]).all())
    # and the bits differ from place to place and from seed to seed
    spread = (squares / tries - mean * mean).clamp(min=0).sqrt()
    assert float((spread[normal_range] > 0).double().mean()) > 0.95


@gpu
def test_slow_averages_move_in_eight_bits(ops):
    """With beta2 = 0.999 a step changes a root by a two-thousandth of itself, far less than half a step of e4m3: on average it still
    goes where the average in 32 bits goes, up and down again."""
    n = 4096
    w = torch.zeros(n, device="cuda")
    d = torch.full((n,), 0.5, device="cuda")
    states = ops.adamw_states([w], 8)
    table = ops.AdamwTable([w], [d], **states)
    v = 0.0
    for t in range(1, 2401):
        if t == 1201:
            d.fill_(0.125)
        v = 0.999 * v + 0.001 * float(d[0]) ** 2 if t in (1, 1201) else 0.999 * v + 0.001 * (0.25 if t < 1201 else 0.015625)
        table.update(t, 0.0, 0.9, 0.999, seed=t)
        if t in (1200, 2400):
            mean = float(decoded(states["vs"][0], states["v_scales"][0]).square().mean())
            assert abs(mean / v - 1) < 0.1, (t, mean, v)


@gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_norm_that_is_not_finite_leaves_the_step_out(ops, bits, bad):
    model = Model(ops, bits)
    model.d[8][100] = bad
    before = model.everything()
    norm = torch.zeros(1, device="cuda")
    model.table.update(3, 1e-3, max_norm=1.0, norm_out=norm, seed=1)
    for a, b in zip(before, model.everything()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert not bool(torch.isfinite(norm).any())
    # without clipping it is what the formulas make of it: visible in that value
    model.table.update(3, 1e-3, seed=1)
    assert int((~torch.isfinite(model.w[8])).sum()) == 1 and not bool(torch.isfinite(model.w[8][100]))
    assert all(bool(torch.isfinite(w).all()) for i, w in enumerate(model.w) if i != 8)


@gpu
def test_the_same_bits_every_time_on_any_stream(ops):
    a, b = Model(ops, 8, sizes=[50000, 777, 4096] * 20), Model(ops, 8, sizes=[50000, 777, 4096] * 20)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for t in (1, 2, 3):
        a.table.update(t, 1e-3, max_norm=0.2, seed=t)
        with torch.cuda.stream(other):
            b.table.update(t, 1e-3, max_norm=0.2, seed=t)
    torch.cuda.synchronize()
    for x, y in zip(a.everything(), b.everything()):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@gpu
def test_a_step_in_a_graph(ops):
    """Captured with its clipping, and replayed with other work between."""
    a, b = Model(ops, 8), Model(ops, 8)
    norm = torch.zeros(1, device="cuda")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            a.table.update(5, 1e-3, max_norm=0.2, norm_out=norm, seed=9)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        b.table.update(5, 1e-3, max_norm=0.2, seed=9)
        for x, y in zip(a.everything(), b.everything()):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        for d, e in zip(a.d, b.d):
            e.mul_(0.5)
            d.mul_(0.5)


def test_refusals():
    lib = capi.load()
    handle = ctypes.c_void_p()
    table = (capi.AdamwTensor * 2)()

    def fill(**change):
        for t in table:
            for k, v in dict(dict(w=256, d=256, m=256, v=256, m_scale=256, v_scale=256, copy=0, n=10, d_type=1, copy_type=0, apply_decay=0), **change).items():
                setattr(t, k, v)
        return ctypes.addressof(table)

    for args, says in [((2, fill(), 16), "8 or 32"), ((-1, fill(), 8), "bad argument"), ((2, None, 8), "bad argument")]:
        assert capi.call_raw("pxh_adamw_table_create", *args, ctypes.byref(handle)) == -1
        assert says in capi.last_error() and not handle.value
    for change, says in [(dict(w=0), "null"), (dict(m_scale=0), "null"), (dict(d_type=3), "gradients"), (dict(copy=256, copy_type=0), "copy"),
                         (dict(n=1 << 31), "2^31")]:
        assert capi.call_raw("pxh_adamw_table_create", 2, fill(**change), 8, ctypes.byref(handle)) == -1, change
        assert says in capi.last_error() and not handle.value
    assert capi.call_raw("pxh_adamw_table_create", 2, fill(), 8, None) == -1
    # a table of nothing: no device is asked for
    assert capi.call_raw("pxh_adamw_table_create", 2, fill(n=0), 8, ctypes.byref(handle)) == 0
    assert handle.value and lib.pxh_adamw_table_count(handle) == 0
    good = [handle, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 0.0, None, 0, None]
    assert capi.call_raw("pxh_adamw_update_table", *good) == 0
    for at, value, says in [(0, None, "null table"), (1, 0, "step"), (3, 1.0, "beta"), (4, -0.1, "beta"), (4, math.nan, "beta"), (5, -1.0, "eps"),
                            (8, -1.0, "max_norm"), (8, math.nan, "max_norm")]:
        args = list(good)
        args[at] = value
        assert capi.call_raw("pxh_adamw_update_table", *args) == -1
        assert says in capi.last_error()
    lib.pxh_adamw_table_destroy(handle)
    lib.pxh_adamw_table_destroy(None)


def test_lists_that_do_not_fit_are_refused(ops):
    t = torch.zeros(4)
    for args, more in [(([t], [t], [t], [t, t]), {}), (([t], [t], [t], [t]), dict(m_scales=[t])), (([t], [t], [t], [t]), dict(apply_decay=[True, False])),
                       (([t], [t], [t], [t]), {}), (([7], [t], [t], [t]), {})]:
        with pytest.raises(capi.PxError):
            ops.AdamwTable(*args, **more)
    with pytest.raises(capi.PxError):
        ops.adamw_states([t], 16)


@gpu
def test_tensors_that_do_not_fit_are_refused(ops):
    w = torch.zeros(300, device="cuda")
    s8 = {k: v for k, v in ops.adamw_states([w], 8).items()}
    s32 = ops.adamw_states([w], 32)
    for ds, states, more in [([w[:299]], s32, {}), ([w.double()], s32, {}), ([w], dict(s32, ms=[w.half()]), {}), ([w], dict(s8, m_scales=[w[:1]]), {}),
                             ([w], dict(s8, ms=s32["ms"]), {}), ([w], s32, dict(copies=[w.clone()])), ([w], s32, dict(copies=[w[:5].half()])),
                             ([w.cpu()], s32, {})]:
        with pytest.raises(capi.PxError):
            ops.AdamwTable([w], ds, **states, **more)
    with pytest.raises(capi.PxError):
        ops.AdamwTable([w.view(20, 15).t()], [w], **s32)
    table = ops.AdamwTable([w], [w.clone()], **s32)
    for bad in (dict(t=0), dict(t=1, norm_out=w), dict(t=1, norm_out=torch.zeros(1)), dict(t=1, max_norm=-1.0)):
        with pytest.raises(capi.PxError):
            table.update(lr=1e-3, **bad)
    table.close()
    with pytest.raises(capi.PxError):
        table.update(1, 1e-3)


@gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("size,d_scale", [(1e38, 1.0), (3e38, 2.0), (2e38, -2.5)])
def test_a_norm_beyond_the_largest_number_leaves_the_step_out(ops, bits, size, d_scale):
    """Every gradient is a number, and so is their norm in 64 bits, but not as the fp32 value that clips them."""
    model = Model(ops, bits, kinds=("f32",))
    model.d[7].fill_(size)
    before = model.everything()
    norm = torch.zeros(1, device="cuda")
    model.table.update(3, 1e-3, d_scale=d_scale, max_norm=1.0, norm_out=norm, seed=1)
    for a, b in zip(before, model.everything()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert float(norm) == math.inf
    # the largest that is one clips as any other
    model.d[7].fill_(0.0)
    model.d[7][100] = 3.4e38
    model.table.update(3, 1e-3, max_norm=1.0, norm_out=norm, seed=1)
    assert float(norm) == float(np.float32(3.4e38))
    assert all(bool(torch.isfinite(x.float()).all()) for group in (model.w, model.m, model.v) for x in group)
    assert not torch.equal(model.w[7], before[7])


@gpu
def test_the_norm_is_the_nearest_number(ops):
    """Sums that are exact in 64 bits: the norm is the fp32 number next to their root."""
    norm = torch.zeros(1, device="cuda")
    for n in range(1, 60):
        w = torch.zeros(n, device="cuda")
        table = ops.AdamwTable([w], [torch.ones(n, device="cuda")], **ops.adamw_states([w], 32))
        table.update(1, 1e-3, d_scale=0.5, norm_out=norm)
        assert float(norm) == float(np.float32(0.5 * math.sqrt(n))), n


@gpu
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_value_that_is_no_number_is_kept_as_its_blocks_largest(ops, bad):
    """States in 8 bits, without clipping: the value's own weight is lost and nothing beside it, in this step or in the next."""
    model, clean = Model(ops, 8, kinds=("f32",)), Model(ops, 8, kinds=("f32",))
    at = 300                                        # in the second block of 1000 values
    for a in (model, clean):
        for state in (a.m[7], a.v[7]):
            state.view(torch.uint8)[at] = 0         # nothing that could be the block's largest
        a.d[7][at] = 0.0
    model.d[7][at] = bad
    for a in (model, clean):
        a.table.update(3, 1e-3, seed=1)
    others = torch.arange(1000, device="cuda") != at
    assert not bool(torch.isfinite(model.w[7][at])) and torch.equal(model.w[7][others], clean.w[7][others])
    assert float(model.m[7][at]) == 448.0 and float(model.v[7][at]) == 448.0
    for name in ("m", "v"):
        got, want = getattr(model, name), getattr(clean, name)
        assert torch.equal(got[7].view(torch.uint8)[others], want[7].view(torch.uint8)[others]), name
        assert torch.equal(getattr(model, name + "s")[7], getattr(clean, name + "s")[7]), name
    model.d[7][at] = 0.0
    for t in (4, 5):
        model.table.update(t, 1e-3, seed=t)
    assert bool(torch.isfinite(model.w[7][others]).all()) and bool(torch.isfinite(model.v[7].float()).all())
    assert bool(torch.isfinite(model.ms[7]).all()) and bool(torch.isfinite(model.vs[7]).all())


def test_more_values_than_a_launch_takes():
    """Refused before a list of their chunks has been made, which would be larger than memory."""
    count = 1 << 16
    table = (capi.AdamwTensor * count)()
    for t in table:
        t.w = t.d = t.m = t.v = 256
        t.n, t.d_type = (1 << 31) - 1, 0
    handle = ctypes.c_void_p()
    assert capi.call_raw("pxh_adamw_table_create", count, ctypes.addressof(table), 32, ctypes.byref(handle)) == -2
    assert "one launch" in capi.last_error() and not handle.value


@gpu
def test_scales_are_the_largest_magnitude_times_a_448th(ops):
    """To the bit what elementary operations in fp32 give, as the norm's scales are: an ulp of a scale turns single codes."""
    n = 256 * 3000
    g = torch.Generator().manual_seed(11)
    w, d = torch.zeros(n, device="cuda"), normal(g, n, 1.0)
    states = ops.adamw_states([w], 8)
    ops.AdamwTable([w], [d], **states).update(1, 1e-3, 0.5, 0.75, seed=3)
    m, root = 0.5 * d, (0.25 * (d * d)).cpu().numpy()
    root = np.sqrt(root).reshape(-1, 256).max(1)                    # numpy's root is the rounded one
    recip = np.float32(1.0) / np.float32(448.0)
    assert np.array_equal(states["m_scales"][0].cpu().numpy(), m.abs().cpu().numpy().reshape(-1, 256).max(1) * recip)
    assert np.array_equal(states["v_scales"][0].cpu().numpy(), root * recip)

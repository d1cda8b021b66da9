"""The root-mean-square norm with the residual's addition and its gradients, against the formulas in 64 bits.

Bounds.  With u = 2^-24 and e = half a unit of the tensors' type (2^-24, 2^-8, 2^-11: a significand of 24, 8, 11 bits; at least 2^-25, half of the least
step, for half precision): the sum of squares of n values, added in n / (lanes * vectors) steps and trees, is within
(n / 64 + 16) u of its value, of which rstd takes half, and two more roundings; y has three more products and the rounding to
its type.  A gradient's dot product is bounded by the same number of additions times the sum of the magnitudes; dw is added up by
at most 1024 workers, whose sums 16 lanes take turns to add."""
import math

import numpy as np
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


def draw(seed, shape, std, dtype, pad=0):
    """Values on the device in a slice of rows that are `pad` values wider."""
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(shape[0], shape[1] + pad, generator=g) * std
    return wide.to(dtype).cuda()[:, :shape[1]]


def additions(n):
    return n / 64 + 16


def held(got, want, bound, what):
    """|got - want| <= bound, value by value; NaN and infinities where they are wanted."""
    got, want = got.double().cpu(), want.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    over = ((got - want).abs() - torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(want))[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, "%s: %g over" % (what, float(over.max()))


def formula(x, residual, weight, eps):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = h.double()
    rstd = 1.0 / torch.sqrt(d.square().mean(1) + eps)
    return h, rstd, d * rstd[:, None] * weight.double()


SHAPES = [(1, 1), (3, 2), (1, 64), (5, 127), (9, 512), (2, 513), (33, 1000), (7, 2048), (4, 2049), (3, 8192), (2, 8200), (2, 32768),
          (1, 32769), (2, 40007), (300, 96)]


@gpu
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("residual,pad,wide_weight", [(False, 0, False), (True, 3, True), (True, 0, False)])
def test_forward_is_the_formula(ops, rows, width, kind, residual, pad, wide_weight):
    dtype, e, least = TYPES[kind]
    x = draw(rows * 31 + width, (rows, width), 1.7, dtype, pad)
    r = draw(width, (rows, width), 0.5, dtype, pad + 1 if pad else 0) if residual else None
    weight = draw(5, (1, width), 1.0, torch.float32 if wide_weight else dtype)[0].contiguous()
    y = torch.full((rows, width + pad), 7.0, dtype=dtype, device="cuda")
    total = torch.empty_like(x) if residual else None
    rstd = torch.empty(rows, device="cuda")
    ops.rms_norm_forward(x, y[:, :width], weight, residual=r, sum=total, rstd=rstd, eps=1e-5)
    h, want_rstd, want = formula(x, r, weight, 1e-5)
    held(rstd, want_rstd, want_rstd * U * (additions(width) / 2 + 3), "rstd")
    held(y[:, :width], want, want.abs() * (U * (additions(width) / 2 + 6) + e) + least, "y")
    assert bool((y[:, width:] == 7).all())                      # nothing behind a row
    if residual:
        assert torch.equal(total, h)
        # in place: the sum over the residual, the result over x; the same bits
        before = y[:, :width].clone()
        xi = x.clone().contiguous()
        ri = r.clone().contiguous()
        ops.rms_norm_forward(xi, xi, weight, residual=ri, sum=ri, eps=1e-5)
        assert torch.equal(ri, h) and torch.equal(xi, before)


@gpu
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("group,residual,pad", [(0, False, 0), (128, True, 0), (0, True, 5), (128, False, 5)])
def test_eight_bits_are_the_scaled_values(ops, rows, width, kind, group, residual, pad):
    dtype, e, least = TYPES[kind]
    x = draw(rows * 7 + width, (rows, width), 3.0, dtype, pad)
    x[rows // 2] = 0                                              # a row of zeros has zeros
    r = draw(width + 1, (rows, width), 0.5, dtype, pad) if residual else None
    if residual:
        r[rows // 2] = 0
    weight = draw(6, (1, width), 1.0, dtype)[0].contiguous()
    y = torch.zeros(rows, width + pad, dtype=torch.float8_e4m3fn, device="cuda")[:, :width]
    groups = -(-width // 128) if group else 1
    scales = torch.empty(rows, groups, device="cuda")
    ops.rms_norm_forward(x, y, weight, residual=r, scales=scales, eps=1e-5, group=group)
    want = formula(x, r, weight, 1e-5)[2]
    near = U * (additions(width) / 2 + 10)
    size = group or width
    padded = torch.nn.functional.pad(want, (0, groups * size - width)).view(rows, groups, size)
    want_scales = (padded.abs().amax(2) / 448.0).clamp(min=2.0 ** -126)
    held(scales, want_scales, want_scales * near, "scales")
    # half a step of e4m3: 2^-4 of the value, and 2^-10 of the scale below the least normal value
    got = y.float().double() * scales.double().repeat_interleave(size, 1)[:, :width]
    step = scales.double().repeat_interleave(size, 1)[:, :width] * 2.0 ** -10
    held(got, want, torch.maximum(want.abs() * 2.0 ** -4, step) * (1 + 20 * near) + want.abs() * near, "values")
    # the largest of a group is the largest value there is
    assert torch.equal(torch.nn.functional.pad(y.float(), (0, groups * size - width)).view(rows, groups, size).abs().amax(2) == 448.0,
                       want_scales > 2.0 ** -126)


@gpu
@pytest.mark.parametrize("rows,width,kind", [(9000, 4097, "bf16"), (70000, 500, "f16"), (2100, 16384, "f32")])
def test_tensors_that_do_not_fit_the_caches(ops, rows, width, kind):
    dtype, e, least = TYPES[kind]
    x, r = (torch.randn(rows, width, device="cuda", generator=torch.Generator("cuda").manual_seed(i)).to(dtype) for i in (1, 2))
    weight = draw(6, (1, width), 1.0, dtype)[0].contiguous()
    y, total, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda")
    ops.rms_norm_forward(x, y, weight, residual=r, sum=total, rstd=rstd, eps=1e-5)
    h, want_rstd, want = formula(x, r, weight, 1e-5)
    assert torch.equal(total, h)
    held(rstd, want_rstd, want_rstd * U * (additions(width) / 2 + 3), "rstd")
    held(y, want, want.abs() * (U * (additions(width) / 2 + 6) + e) + least, "y")
    dx, dw = torch.empty_like(x), torch.empty(width, device="cuda")
    ops.rms_norm_backward(r, h, weight, rstd, dx, dw, dsum=x)
    want, dot, parts, want_dw, sum_dw = gradients(r, h, weight, rstd, x)
    held(dx, want, dot * U * additions(width) + parts * 6 * U + want.abs() * (e + U) + least, "dx")
    # the rows of one of 256 workers (of 1024 for narrow rows) in turn, then the workers
    held(dw, want_dw, sum_dw * U * (rows / 256 + 64 + 20) + 1e-30, "dw")


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("width", [96, 3000, 40000])
def test_infinities_and_nan_stay_in_their_rows(ops, kind, width):
    dtype = TYPES[kind][0]
    x = draw(8, (4, width), 1.0, dtype)
    x[1, 17] = math.inf
    x[2, width - 1] = math.nan
    weight = torch.ones(width, dtype=dtype, device="cuda")
    y = torch.empty_like(x)
    ops.rms_norm_forward(x, y, weight)
    clean = torch.empty(2, width, dtype=dtype, device="cuda")
    ops.rms_norm_forward(x[::3].contiguous(), clean, weight)
    assert torch.equal(y[::3], clean)
    assert bool(torch.isnan(y[1, 17])) and int(torch.isnan(y[1]).sum()) == 1 and bool((y[1].nan_to_num(0.0) == 0).all())
    assert bool(torch.isnan(y[2]).all())
    q, scales = torch.empty(4, width, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(4, 1, device="cuda")
    ops.rms_norm_forward(x, q, weight, scales=scales)
    q = q.float()
    assert bool(torch.isfinite(q[::3]).all()) and bool(torch.isnan(q[1, 17])) and bool(torch.isnan(q[2]).all())


def gradients(dy, h, weight, rstd, dsum):
    g, x, r = dy.double(), h.double() * rstd.double()[:, None], rstd.double()[:, None]
    gw = g * weight.double()
    c = (gw * x).mean(1, keepdim=True)
    size = (gw * x).abs().mean(1, keepdim=True)
    dx = r * (gw - x * c)
    if dsum is not None:
        dx = dx + dsum.double()
    return dx, r * x.abs() * size, r * (gw.abs() + (x * c).abs()), (g * x).sum(0), (g * x).abs().sum(0)


@gpu
@pytest.mark.parametrize("rows,width", SHAPES + [(1500, 64), (2100, 33), (70, 16385)])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("stream,pad,wide_weight", [(False, 0, True), (True, 3, False)])
def test_backward_is_the_formula(ops, rows, width, kind, stream, pad, wide_weight):
    dtype, e, least = TYPES[kind]
    h, dy = draw(rows + width, (rows, width), 1.5, dtype, pad), draw(rows - width, (rows, width), 0.3, dtype)
    dsum = draw(3, (rows, width), 0.3, dtype, pad + 2 if pad else 0) if stream else None
    weight = draw(4, (1, width), 1.0, torch.float32 if wide_weight else dtype)[0].contiguous()
    rstd = (1.0 / torch.sqrt(h.double().square().mean(1) + 1e-6)).float()
    dx = torch.empty(rows, width + pad, dtype=dtype, device="cuda")[:, :width]
    dw = torch.full((width,), 3.0, device="cuda")
    ops.rms_norm_backward(dy, h, weight, rstd, dx, dw, dsum=dsum)
    want, dot, parts, want_dw, sum_dw = gradients(dy, h, weight, rstd, dsum)
    held(dx, want, dot * U * additions(width) + parts * 6 * U + want.abs() * (e + U) + least, "dx")
    held(dw, want_dw, sum_dw * U * (rows / 1024 + min(rows, 1024) / 16 + 20) + 1e-30, "dw")
    again = dw.clone()
    over = dy.clone()
    ops.rms_norm_backward(over, h, weight, rstd, over, again, dsum=dsum, accumulate=True)
    assert torch.equal(over, dx)
    held(again, 2 * dw.double(), dw.double().abs() * 4 * U, "added dw")
    if stream:
        over = dsum.clone()
        ops.rms_norm_backward(dy, h, weight, rstd, over, again, dsum=over)
        assert torch.equal(over, dx) and torch.equal(again, dw)


@gpu
def test_backward_against_differences(ops):
    """The gradients of sum(y * c) by central differences of the forward's formula in 64 bits."""
    rows, width = 3, 40
    x, c = draw(1, (rows, width), 1.0, torch.float32), draw(2, (rows, width), 1.0, torch.float32)
    weight = draw(3, (1, width), 1.0, torch.float32)[0].contiguous()
    y, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
    ops.rms_norm_forward(x, y, weight, rstd=rstd)
    dx, dw = torch.empty_like(x), torch.empty(width, device="cuda")
    ops.rms_norm_backward(c, x, weight, rstd, dx, dw)
    f = lambda x, w: (x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-6) * w * c.double().cpu()).sum()  # noqa: E731
    x, w, step = x.double().cpu(), weight.double().cpu(), 1e-5
    for at in np.ndindex(rows, width):
        one = torch.zeros_like(x)
        one[at] = step
        assert abs(float(dx[at]) - float(f(x + one, w) - f(x - one, w)) / (2 * step)) < 1e-5
    for at in range(width):
        one = torch.zeros_like(w)
        one[at] = step
        assert abs(float(dw[at]) - float(f(x, w + one) - f(x, w - one)) / (2 * step)) < 1e-5


@gpu
def test_no_rows_a_workspace_and_another_stream(ops):
    weight = torch.ones(64, device="cuda")
    none = torch.empty(0, 64, device="cuda")
    ops.rms_norm_forward(none, none, weight)
    dw = torch.full((64,), 3.0, device="cuda")
    ops.rms_norm_backward(none, none, weight, torch.empty(0, device="cuda"), none, dw, accumulate=True)
    assert bool((dw == 3).all())
    ops.rms_norm_backward(none, none, weight, torch.empty(0, device="cuda"), none, dw)
    assert bool((dw == 0).all())
    # a workspace of the caller's, on a stream of its own, and three dimensions; the same bits
    h, dy = draw(1, (50, 64), 1.0, torch.float32), draw(2, (50, 64), 1.0, torch.float32)
    y, rstd, dx = torch.empty_like(h), torch.empty(50, device="cuda"), torch.empty_like(h)
    ops.rms_norm_forward(h, y, weight, rstd=rstd)
    ops.rms_norm_backward(dy, h, weight, rstd, dx, dw)
    space = torch.empty(ops.rms_norm_workspace_bytes(50, 64) // 4, device="cuda")
    other, dx2, dw2, y2 = torch.cuda.Stream(), torch.empty_like(dx), torch.empty_like(dw), torch.empty_like(y)
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        ops.rms_norm_forward(h.view(5, 10, 64), y2.view(5, 10, 64), weight)
        ops.rms_norm_backward(dy, h, weight, rstd, dx2, dw2, workspace=space)
    other.synchronize()
    assert torch.equal(y, y2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)


def test_refusals():
    p, n = 256, None
    good = dict(x=p, residual=n, sum=n, weight=p, y=p, scales=n, rstd=n, type=0, weight_type=0, y_type=0, rows=4, width=8, xs=8, rs=0,
                ss=0, ys=8, group=0, eps=1e-6, stream=n)
    for change, says in [(dict(type=3), "fp32, bf16 or half"), (dict(weight_type=1), "weights"), (dict(y_type=1), "e4m3"),
                         (dict(y_type=3), "scales"), (dict(group=64), "128"), (dict(sum=p), "without a residual"), (dict(x=n), "null"),
                         (dict(xs=7), "overlap"), (dict(width=0), "values"), (dict(rows=-1), "rows"), (dict(eps=-1.0), "eps"),
                         (dict(residual=p, rs=3), "overlap")]:
        assert capi.call_raw("pxh_rms_norm_forward", *dict(good, **change).values()) == -1, change
        assert says in capi.last_error(), (change, capi.last_error())
    assert capi.call_raw("pxh_rms_norm_forward", *dict(good, rows=0, x=n).values()) == 0
    good = dict(dy=p, h=p, weight=p, rstd=p, dsum=n, dx=p, dw=p, type=1, weight_type=1, rows=4, width=8, a=8, b=8, c=0, d=8, accumulate=0,
                ws=p, bytes=1 << 20, stream=n)
    for change, code, says in [(dict(dw=n), -1, "null"), (dict(rstd=n), -1, "null"), (dict(d=4), -1, "overlap"),
                               (dict(dsum=p), -1, "overlap"), (dict(bytes=16), -3, "too small"), (dict(ws=p + 4), -3, "aligned"),
                               (dict(weight_type=2), -1, "weights")]:
        assert capi.call_raw("pxh_rms_norm_backward", *dict(good, **change).values()) == code, change
        assert says in capi.last_error(), (change, capi.last_error())


def test_a_workspace_serves_every_smaller_shape():
    size = capi.load().pxh_rms_norm_workspace_bytes
    for width in (1, 100, 16384, 16385, 20000, 32768, 32769, 600000):
        for rows in (1, 31, 32, 33, 256, 1000, 1024, 5000):
            for w in (1, 64, 16384, 16385, 32768, 32769):
                if w <= width:
                    assert size(rows, w) <= size(rows, width) <= size(rows + 1, width)
    assert size(0, 64) == 0


@pytest.mark.parametrize("bad,says", [(torch.zeros(2, 8), "must live on the GPU"), (np.zeros((2, 8)), "torch.Tensor expected"),
                                      (7, "torch.Tensor expected")])
def test_what_is_no_tensor_of_the_device_is_named(ops, bad, says):
    good = torch.zeros(2, 8)
    with pytest.raises(capi.PxError, match=says):
        ops.rms_norm_forward(bad, good, good[0])
    with pytest.raises(capi.PxError, match=says):
        ops.rms_norm_backward(bad, good, good[0], good[0], good, good[0])


@gpu
def test_tensors_that_do_not_fit_are_refused(ops):
    x, weight, rstd = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda"), torch.zeros(4, device="cuda")
    half = x.half()
    for f in (lambda: ops.rms_norm_forward(x, torch.empty_like(x), weight[:7]), lambda: ops.rms_norm_forward(x, half, weight),
              lambda: ops.rms_norm_forward(x.t(), torch.empty(8, 4, device="cuda"), weight[:4]),
              lambda: ops.rms_norm_forward(x.double(), x.double(), weight.double()),
              lambda: ops.rms_norm_forward(x, x, weight, residual=x[:3]),
              lambda: ops.rms_norm_forward(x, half.to(torch.float8_e4m3fn), weight),
              lambda: ops.rms_norm_forward(x, half.to(torch.float8_e4m3fn), weight, scales=rstd, group=7),
              lambda: ops.rms_norm_forward(x, half.to(torch.float8_e4m3fn), weight, scales=rstd[:3]),
              lambda: ops.rms_norm_forward(x, x, weight.bfloat16()), lambda: ops.rms_norm_forward(x, x, weight, rstd=rstd.half()),
              lambda: ops.rms_norm_forward(x, x, weight, sum=x),
              lambda: ops.rms_norm_backward(x, half, weight, rstd, x, weight.clone()),
              lambda: ops.rms_norm_backward(x, x, weight, rstd, x, weight.half()),
              lambda: ops.rms_norm_backward(x, x, weight, rstd[:2], x, weight.clone())):
        with pytest.raises(capi.PxError):
            f()


@gpu
@pytest.mark.parametrize("bad", [lambda: torch.zeros(1 << 20), lambda: torch.zeros(1, device="cuda").expand(1 << 20), lambda: torch.zeros(1 << 21, device="cuda")[::2],
                                 lambda: np.zeros(1 << 20)])
def test_a_workspace_that_is_no_packed_memory_of_the_device_is_refused(ops, bad):
    x, weight, rstd = torch.ones(4, 8, device="cuda"), torch.ones(8, device="cuda"), torch.ones(4, device="cuda")
    with pytest.raises(capi.PxError, match="workspace"):
        ops.rms_norm_backward(x, x, weight, rstd, torch.empty_like(x), torch.empty_like(weight), workspace=bad())
    with pytest.raises(capi.PxError, match="workspace"):
        ops.token_logprobs_forward(x, None, None, entropy=rstd, workspace=bad())


@gpu
@pytest.mark.parametrize("other", [lambda x: x[:0], lambda x: x[:0].half(), lambda x: x[:0].t(), lambda x: x.new_empty(0), lambda x: x[:, :0]])
def test_an_empty_tensor_is_no_missing_one(ops, other):
    x, weight, rstd = torch.ones(4, 8, device="cuda"), torch.ones(8, device="cuda"), torch.ones(4, device="cuda")
    bad, dw = other(x), torch.ones(8, device="cuda")
    y = torch.empty_like(x)
    for f in (lambda: ops.rms_norm_forward(x, y, weight, residual=bad), lambda: ops.rms_norm_forward(x, y, weight, residual=x, sum=bad),
              lambda: ops.rms_norm_forward(x, bad, weight), lambda: ops.rms_norm_backward(x, x, weight, rstd, y, dw, dsum=bad),
              lambda: ops.rms_norm_backward(x, bad, weight, rstd, y, dw), lambda: ops.rms_norm_backward(x, x, weight, rstd, bad, dw)):
        with pytest.raises(capi.PxError):
            f()


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("width", [96, 1000, 4096, 20001, 40007])
@pytest.mark.parametrize("group", [0, 128])
def test_eight_bits_are_the_rounded_quotients(ops, kind, width, group):
    """To the bit what elementary operations in fp32 make of the statistic that the call leaves."""
    rows, dtype = 2000000 // width, TYPES[kind][0]
    x = (torch.randn(rows, width, device="cuda", generator=torch.Generator("cuda").manual_seed(width)) * 3).to(dtype)
    weight = draw(6, (1, width), 1.0, dtype)[0].contiguous()
    groups = -(-width // 128) if group else 1
    y, scales, rstd = torch.empty(rows, width, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(rows, groups, device="cuda"), torch.empty(rows, device="cuda")
    ops.rms_norm_forward(x, y, weight, scales=scales, rstd=rstd, group=group)
    h, w, r = x.float().cpu(), weight.float().cpu(), rstd.cpu()[:, None]
    value = h * r * w
    size = group or width
    parts = lambda t: torch.nn.functional.pad(t, (0, groups * size - width)).view(rows, groups, size)      # noqa: E731
    # a row's scale is found before its statistic
    peak = parts(value).abs().amax(2) if group else (h * w).abs().amax(1, keepdim=True) * r
    want = (peak * float(np.float32(1.0) / np.float32(448.0))).clamp(min=2.0 ** -126)
    assert torch.equal(scales.cpu(), want)
    codes = (parts(value) / want[:, :, None]).to(torch.float8_e4m3fn).view(rows, groups * size)[:, :width]
    assert torch.equal(y.cpu().view(torch.uint8), codes.contiguous().view(torch.uint8))


@gpu
@pytest.mark.parametrize("group", [0, 128])
def test_an_infinite_value_leaves_the_others_of_its_group(ops, group):
    """A weight of infinity: NaN in its column, zeros beside it, and numbers where another scale is."""
    x = draw(3, (5, 300), 1.0, torch.float32)
    weight = torch.ones(300, device="cuda")
    weight[140] = math.inf
    y, scales = torch.empty(5, 300, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(5, 3 if group else 1, device="cuda")
    ops.rms_norm_forward(x, y, weight, scales=scales, group=group)
    y = y.float()
    assert bool(torch.isnan(y[:, 140]).all()) and int(torch.isnan(y).sum()) == 5 and bool(torch.isfinite(scales).all())
    beside = y[:, 128:256] if group else y
    assert bool((beside.nan_to_num(0.0) == 0).all())
    if group:
        assert bool((y[:, :128] != 0).any(1).all()) and bool((y[:, 256:] != 0).any(1).all())

"""Layer norm with the residual's addition and its gradients, against the formulas in 64 bits.

Bounds.  With u = 2^-24 and e = half a unit of the tensors' type: a sum of n values is added in n / 64 steps of a lane and 16 of a tree, so
that it is within (n / 64 + 16) u of the sum of their magnitudes.  The mean takes one division more; the squares' sum half of it in rstd, and a
mean that is off by d adds d^2 to the variance, nothing in the first order.  y has the mean's error times weight and rstd, and three
roundings of its own.  A gradient's two sums are bounded by the same number of additions; those over the rows by the rows of a worker and the
256 or 1024 workers, whose sums 16 lanes take turns to add."""
import pytest

torch = pytest.importorskip("torch")

from pixienn_amd import capi

gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": (torch.float32, 2.0 ** -24, 2.0 ** -140), "bf16": (torch.bfloat16, 2.0 ** -8, 2.0 ** -134),
         "f16": (torch.float16, 2.0 ** -11, 2.0 ** -25)}
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    from pixienn_amd import ops as o
    return o


def draw(seed, shape, std, dtype, pad=0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(shape[0], shape[1] + pad, generator=g) * std + mean
    return wide.to(dtype).cuda()[:, :shape[1]]


def additions(n):
    return n / 64 + 16


def held(got, want, bound, what):
    got, want = got.double().cpu(), want.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    over = ((got - want).abs() - torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(want))[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, "%s: %g over" % (what, float(over.max()))


def formula(x, residual, weight, bias, eps=EPS):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = h.double()
    mean = d.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((d - mean).square().mean(1, keepdim=True) + eps)
    y = (d - mean) * rstd * weight.double()
    return h, mean, rstd, y if bias is None else y + bias.double()


def bounds(h, mean, rstd, y, weight, e, least):
    n = h.shape[1]
    d = h.double()
    of_mean = U * (additions(n) * d.abs().mean(1, keepdim=True) + 2 * mean.abs())
    of_rstd = U * (additions(n) / 2 + 4) * rstd
    scaled = ((d - mean) * rstd * weight.double()).abs()
    return of_mean, of_rstd, of_mean * rstd * weight.double().abs() + scaled * U * (additions(n) / 2 + 8) + y.abs() * (2 * U + e) + least


SHAPES = [(1, 1), (3, 2), (1, 64), (5, 127), (9, 512), (2, 513), (33, 1000), (7, 2048), (4, 2049), (3, 8192), (2, 8200), (2, 32768),
          (1, 32769), (2, 40007), (300, 96)]


@gpu
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("residual,pad,wide_weight,with_bias", [(False, 0, False, True), (True, 3, True, True), (True, 0, False, False)])
def test_forward_is_the_formula(ops, rows, width, kind, residual, pad, wide_weight, with_bias):
    dtype, e, least = TYPES[kind]
    x = draw(rows * 31 + width, (rows, width), 1.7, dtype, pad, mean=0.8)
    r = draw(width, (rows, width), 0.5, dtype, pad + 1 if pad else 0) if residual else None
    of = torch.float32 if wide_weight else dtype
    weight = draw(5, (1, width), 1.0, of)[0].contiguous()
    bias = draw(6, (1, width), 1.0, of)[0].contiguous() if with_bias else None
    y = torch.full((rows, width + pad), 7.0, dtype=dtype, device="cuda")
    total = torch.empty_like(x) if residual else None
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ops.layer_norm_forward(x, y[:, :width], weight, bias=bias, residual=r, sum=total, mean=mean, rstd=rstd)
    h, want_mean, want_rstd, want = formula(x, r, weight, bias)
    of_mean, of_rstd, of_y = bounds(h, want_mean, want_rstd, want, weight, e, least)
    held(mean, want_mean[:, 0], of_mean[:, 0], "mean")
    held(rstd, want_rstd[:, 0], of_rstd[:, 0], "rstd")
    held(y[:, :width], want, of_y, "y")
    assert bool((y[:, width:] == 7).all())                      # nothing behind a row
    if residual:
        assert torch.equal(total, h)
        # in place: the sum over the residual, the result over x; the same bits, and the same without the statistics
        before = y[:, :width].clone()
        xi = x.clone().contiguous()
        ri = r.clone().contiguous()
        ops.layer_norm_forward(xi, xi, weight, bias=bias, residual=ri, sum=ri)
        assert torch.equal(ri, h) and torch.equal(xi, before)
        xi = x.clone().contiguous()
        ops.layer_norm_forward(xi, xi, weight, bias=bias, residual=r)
        assert torch.equal(xi, before)


@gpu
@pytest.mark.parametrize("rows,width,kind", [(9000, 4097, "bf16"), (70000, 500, "f16"), (2100, 16384, "f32")])
def test_many_rows_past_the_caches(ops, rows, width, kind):
    dtype, e, least = TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, width, device="cuda", generator=g).to(dtype)
    r = torch.randn(rows, width, device="cuda", generator=g).to(dtype)
    weight, bias = x[0].clone(), r[0].clone()
    y, total = torch.empty_like(x), torch.empty_like(x)
    ops.layer_norm_forward(x, y, weight, bias=bias, residual=r, sum=total)
    few = torch.cat([torch.arange(0, 40), torch.arange(rows - 40, rows)]).cuda()
    h, mean, rstd, want = formula(x[few], r[few], weight, bias)
    assert torch.equal(total[few], h)
    held(y[few], want, bounds(h, mean, rstd, want, weight, e, least)[2], "y")
    # a row's result does not depend on the others: the same row twice
    x[rows // 2], r[rows // 2] = x[3], r[3]
    ops.layer_norm_forward(x, y, weight, bias=bias, residual=r, sum=total)
    assert torch.equal(y[rows // 2], y[3])


@gpu
@pytest.mark.parametrize("width", [1, 7, 640, 5000, 33001])
def test_constant_rows_large_means_and_what_is_no_number(ops, width):
    x = torch.full((6, width), 3.0, device="cuda")
    x[1] = 0.0
    x[2] += 1e4 + torch.randn(width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x[3, width // 2] = float("nan")
    x[4, width - 1] = float("inf")
    weight, bias = torch.full((width,), 2.0, device="cuda"), torch.full((width,), 0.5, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    ops.layer_norm_forward(x, y, weight, bias=bias, mean=mean, rstd=rstd)
    assert bool((y[1] == 0.5).all()) and float(mean[1]) == 0.0
    good = [0, 1, 2, 5]
    h, want_mean, want_rstd, want = formula(x[good], None, weight, bias)
    held(y[good], want, bounds(h, want_mean, want_rstd, want, weight, U, 0.0)[2], "y")
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[4]).all())          # infinity minus an infinite mean


def gradient(dy, h, weight, mean, rstd, dsum):
    dy, d, w = dy.double(), h.double(), weight.double()
    mean, rstd = mean.double()[:, None], rstd.double()[:, None]
    xhat = (d - mean) * rstd
    g = dy * w
    c0, c1 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    dx = rstd * (g - c0 - xhat * c1)
    n = h.shape[1]
    bound = rstd * U * ((additions(n) + 4) * (g.abs().mean(1, keepdim=True) + xhat.abs() * (g * xhat).abs().mean(1, keepdim=True))
                        + 8 * (g.abs() + c0.abs() + (xhat * c1).abs()) + 2 * c1.abs() * rstd * (d.abs() + mean.abs()))
    if dsum is not None:
        dx = dx + dsum.double()
    rows = h.shape[0]
    adds = U * (rows / min(rows, 32) + 16 + 64 + 6)
    dw, db = dy * xhat, dy
    of_dw = adds * dw.abs().sum(0) + 2 * U * (dy.abs() * rstd * (d.abs() + mean.abs())).sum(0)
    return dx, bound, dw.sum(0), of_dw, db.sum(0), adds * db.abs().sum(0)


@gpu
@pytest.mark.parametrize("rows,width", SHAPES + [(1500, 300), (700, 2100), (600, 9003), (300, 16383), (500, 8191)])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("with_sum,pad,wide_weight,with_bias", [(False, 0, False, True), (True, 5, True, True), (True, 0, True, False)])
def test_gradients_are_the_formula(ops, rows, width, kind, with_sum, pad, wide_weight, with_bias):
    dtype, e, least = TYPES[kind]
    h = draw(rows + width, (rows, width), 1.3, dtype, pad, mean=-0.7)
    dy = draw(rows + width + 1, (rows, width), 0.3, dtype, pad)
    dsum = draw(rows + width + 2, (rows, width), 0.3, dtype, 2 * pad) if with_sum else None
    weight = draw(5, (1, width), 1.0, torch.float32 if wide_weight else dtype)[0].contiguous()
    _, mean, rstd, _ = formula(h, None, weight, None)
    mean, rstd = mean[:, 0].float(), rstd[:, 0].float()
    dx = torch.full((rows, width + pad), 7.0, dtype=dtype, device="cuda")
    dw = torch.full((width,), 3.0, device="cuda")
    db = torch.full((width,), 3.0, device="cuda") if with_bias else None
    ops.layer_norm_backward(dy, h, weight, mean, rstd, dx[:, :width], dw, db=db, dsum=dsum)
    want, of_dx, want_dw, of_dw, want_db, of_db = gradient(dy, h, weight, mean, rstd, dsum)
    held(dx[:, :width], want, of_dx + want.abs() * (e + 2 * U) + least + (U * dsum.double().abs() if with_sum else 0), "dx")
    assert bool((dx[:, width:] == 7).all())
    held(dw, want_dw, of_dw, "dw")
    if with_bias:
        held(db, want_db, of_db, "db")
    # added to, with dx over dy: the same dx, and the sums on top
    first, first_db = dw.clone(), None if db is None else db.clone()
    dyi = dy.clone().contiguous()
    space = torch.empty(ops.layer_norm_workspace_bytes(rows, width), dtype=torch.uint8, device="cuda")
    ops.layer_norm_backward(dyi, h.contiguous(), weight, mean, rstd, dyi, dw, db=db, dsum=None if dsum is None else dsum.contiguous(),
                            accumulate=True, workspace=space)
    assert torch.equal(dyi, dx[:, :width])
    if with_sum:
        # and over dsum
        over = dsum.clone().contiguous()
        ops.layer_norm_backward(dy, h, weight, mean, rstd, over, torch.empty_like(dw), db=None, dsum=over)
        assert torch.equal(over, dx[:, :width])
    assert torch.equal(dw, first + first) and (db is None or torch.equal(db, first_db + first_db))


@gpu
def test_the_gradient_is_that_of_differences(ops):
    """Central differences of the formula in 64 bits."""
    rows, width, step = 3, 37, 1e-6
    h, dy = draw(1, (rows, width), 1.0, torch.float32).contiguous(), draw(2, (rows, width), 1.0, torch.float32).contiguous()
    weight, bias = draw(3, (1, width), 1.0, torch.float32)[0].contiguous(), draw(4, (1, width), 1.0, torch.float32)[0].contiguous()
    y, mean, rstd = torch.empty_like(h), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ops.layer_norm_forward(h, y, weight, bias=bias, mean=mean, rstd=rstd)
    dx, dw, db = torch.empty_like(h), torch.empty(width, device="cuda"), torch.empty(width, device="cuda")
    ops.layer_norm_backward(dy, h, weight, mean, rstd, dx, dw, db=db)
    at = {"h": h.cpu().double(), "w": weight.cpu().double(), "b": bias.cpu().double()}
    loss = lambda: float((formula(at["h"], None, at["w"], at["b"])[3] * dy.cpu().double()).sum())  # noqa: E731
    for name, got in (("h", dx), ("w", dw), ("b", db)):
        flat, grads = at[name].view(-1), got.cpu().view(-1)
        for i in range(0, flat.numel(), 5):
            was = float(flat[i])
            flat[i] = was + step
            up = loss()
            flat[i] = was - step
            down = loss()
            flat[i] = was
            # the differences' own error: 64-bit roundings of a sum of 111 terms over the step, and step^2
            assert abs((up - down) / (2 * step) - float(grads[i])) < 1e-5, (name, i)


@gpu
def test_no_rows(ops):
    none = torch.empty(0, 8, device="cuda")
    weight = torch.ones(8, device="cuda")
    dw, db = torch.full((8,), 3.0, device="cuda"), torch.full((8,), 3.0, device="cuda")
    ops.layer_norm_forward(none, none, weight, bias=weight)
    ops.layer_norm_backward(none, none, weight, none[:, 0].contiguous(), none[:, 0].contiguous(), none, dw, db=db, accumulate=True)
    assert bool((dw == 3).all()) and bool((db == 3).all())
    ops.layer_norm_backward(none, none, weight, none[:, 0].contiguous(), none[:, 0].contiguous(), none, dw, db=db)
    assert bool((dw == 0).all()) and bool((db == 0).all())


@gpu
def test_what_is_refused(ops):
    x = torch.zeros(4, 16, device="cuda")
    w, r = x[0].clone(), x[:, 0].clone()
    for call, message in [
            (lambda: ops.layer_norm_forward(x, x.half(), w), "y must be"),
            (lambda: ops.layer_norm_forward(x, x[:2], w), "y must be"),
            (lambda: ops.layer_norm_forward(x, x, w[:8]), "weight must hold 16"),
            (lambda: ops.layer_norm_forward(x, x, w, bias=w.half()), "bias must be"),
            (lambda: ops.layer_norm_forward(x, x, w, sum=x.clone()), "sum without a residual"),
            (lambda: ops.layer_norm_forward(x, x, w, mean=r[:3]), "mean must hold 4"),
            (lambda: ops.layer_norm_forward(x, x, w, eps=-1.0), "eps"),
            (lambda: ops.layer_norm_forward(x, x, w.half()), "weights are of the tensors' type or fp32"),
            (lambda: ops.layer_norm_forward(x.t(), x.t(), r), "next to each other"),
            (lambda: ops.layer_norm_forward(x[:1].expand(4, 16), x, w), "overlap"),
            (lambda: ops.layer_norm_forward(x.double(), x.double(), w), "fp32, bfloat16 or half"),
            (lambda: ops.layer_norm_backward(x, x, w, r, r, x, w, db=w[:4]), "db must hold 16"),
            (lambda: ops.layer_norm_backward(x, x, w, r, r, x, None), "null pointer"),
            (lambda: ops.layer_norm_backward(x, x, w, None, r, x, w), "null pointer"),
            (lambda: ops.layer_norm_backward(x, x.half(), w, r, r, x, w), "h must be"),
            (lambda: ops.layer_norm_backward(x, x, w, r, r, x.clone(), w.clone(), workspace=torch.empty(16, device="cuda")), "workspace too small")]:
        with pytest.raises(capi.PxError, match=message):
            call()

"""Operators of token models: what is timed, through `pixienn_amd.ops`, and the same in plain torch operations.

What stands between the matrix products of a network over tokens, in training and in serving.  The products themselves are
not part of it: every case starts from synthetic products of realistic distributions.  Kinds of case:

  norm           root-mean-square norm with the residual's addition in front of it; the output in the tensors' own type, or in
                 8 bits (e4m3) with a scale for each row or for each 128 values of a row
  norm_backward  its gradients, with the gradient that arrives along the residual stream added
  tokens         log probabilities of given tokens, entropy, and the most probable alternatives
  tokens_backward, tokens_train
                 the gradient of the logits for given gradients of log probability and entropy; both in one call
  adamw          a step over all parameter tensors of a model, states in 32 or in 8 bits, gradients clipped by their common norm

`run` computes in plain torch operations, or, with `own`, by the calls that a user makes.  Both update the optimiser's
parameters and states in place.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6                      # of the norm
GROUP = 128                     # values with one scale, of an 8-bit output scaled in groups
E4M3_MAX = 448.0
LEAST_SCALE = 2.0 ** -126
BLOCK = 256                     # values with one scale, of an 8-bit optimiser state
BETA1, BETA2, ADAM_EPS, DECAY = 0.9, 0.95, 1e-8, 0.1


def listed():
    return [
        # serving: the running sequences' newest tokens, quantised for the product behind the norm
        dict(name="norm_8x4096_bf16_e4m3", kind="norm", rows=8, width=4096, type="bf16", residual=True, out="row", pad=0),
        # serving: a batch of prompts, a scale for each 128 values
        dict(name="norm_4096x8192_bf16_e4m3", kind="norm", rows=4096, width=8192, type="bf16", residual=True, out="group", pad=0),
        # training in full precision on a slice of wider rows, odd width, the row's statistic kept
        dict(name="norm_1111x1537_f32", kind="norm", rows=1111, width=1537, type="f32", residual=False, out="same", pad=63),
        # a training step's gradient of one norm
        dict(name="norm_backward_16384x4096_bf16", kind="norm_backward", rows=16384, width=4096, type="bf16", residual=True, pad=0),
        # the same for a short odd batch in half precision
        dict(name="norm_backward_777x5121_f16", kind="norm_backward", rows=777, width=5121, type="f16", residual=False, pad=0),
        # serving: log probability of the chosen tokens and what else was likely
        dict(name="tokens_8x131072_bf16_top8", kind="tokens", rows=8, vocab=131072, type="bf16", top=8, masked=0.0, scale=1.25),
        # scoring a batch of texts under a mask of allowed tokens, odd vocabulary
        dict(name="tokens_4096x50001_f16_top3", kind="tokens", rows=4096, vocab=50001, type="f16", top=3, masked=0.5, scale=1.0),
        # training: the loss and its gradient where the rows' weights are known
        dict(name="tokens_train_8192x32768_bf16", kind="tokens_train", rows=8192, vocab=32768, type="bf16", entropy=False, scale=1.0),
        # training on a function of the log probabilities and the entropy: the gradient alone
        dict(name="tokens_backward_1000x100001_f32", kind="tokens_backward", rows=1000, vocab=100001, type="f32", entropy=True, scale=0.9),
        # a token model of 185 M parameters, gradients and a second copy of the weights in bf16, states in 8 bits
        dict(name="adamw_185m_8bit", kind="adamw", model="tokens", blocks=12, width=1024, wide=4096, vocab=32768, bits=8,
             gradients="bf16", copies=True, max_norm=1.0),
        # a detector's 174 tensors, everything in 32 bits
        dict(name="adamw_detector_32bit", kind="adamw", model="detector", blocks=23, width=1024, wide=0, vocab=0, bits=32,
             gradients="f32", copies=False, max_norm=0.0),
        # adapters: many small tensors of odd sizes
        dict(name="adamw_small_8bit", kind="adamw", model="odd", blocks=60, width=301, wide=0, vocab=0, bits=8, gradients="f16",
             copies=False, max_norm=0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, step):
    """Spread over the logarithm: a power of two, a multiple of `step`, or odd."""
    n = _log_int(rng, lo, hi)
    return rng.choice([max(lo, 1 << n.bit_length() - 1), max(lo, n // step * step), n | 1])


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_backward", "tokens", "tokens", "tokens_train", "tokens_backward", "adamw", "adamw"])
    kind_of_type = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("norm", "norm_backward"):
        width = _size(rng, 64, 16384, 80)
        rows = _log_int(rng, 1, min(16384, (16384 * 4096 if kind_of_type != "f32" else 8192 * 4096) // width))
        case = dict(kind=kind, rows=rows, width=width, type=kind_of_type, residual=rng.random() < 0.6, pad=rng.choice([0, 0, 8, 13]))
        if kind == "norm":
            case["out"] = rng.choice(["same", "row", "group"])
        return case
    if kind.startswith("tokens"):
        vocab = _size(rng, 1000, 160000, 80)
        most = 8192 * 32768 if kind_of_type != "f32" else 4096 * 32768
        case = dict(kind=kind, rows=_log_int(rng, 1, min(8192, most // vocab)), vocab=vocab, type=kind_of_type,
                    scale=rng.choice([1.0, 1.0, 0.7, 1.3]))
        if kind == "tokens":
            case.update(top=rng.choice([0, 1, 5, 8, 20]), masked=rng.choice([0.0, 0.0, 0.3, 0.95]))
        else:
            case["entropy"] = rng.random() < 0.5
        return case
    model = rng.choice(["tokens", "detector", "odd"])
    bits, gradients = rng.choice([8, 8, 32]), kind_of_type
    common = dict(kind=kind, model=model, bits=bits, gradients=gradients, copies=rng.random() < 0.5, max_norm=rng.choice([0.0, 0.5, 1.0]))
    if model == "tokens":
        width = _size(rng, 128, 1024, 80)
        return dict(common, blocks=rng.randint(1, 7), width=width, wide=rng.choice([2, 4]) * width, vocab=_size(rng, 1000, 32768, 80))
    if model == "detector":
        return dict(common, blocks=rng.randint(3, 23), width=rng.choice([256, 512, 1024]), wide=0, vocab=0)
    return dict(common, blocks=_log_int(rng, 2, 400), width=_log_int(rng, 9, 400), wide=0, vocab=0)


# ---------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=g)


def _rows(g, case, std=1.0):
    """rows x width, a slice of rows that are `pad` values wider."""
    rows, width, pad = case["rows"], case["width"], case["pad"]
    return _normal(g, (rows, width + pad), std, TYPES[case["type"]])[:, :width]


def _parameters(case):
    """(values, takes weight decay) of every parameter tensor of a model."""
    blocks, width, wide, vocab = case["blocks"], case["width"], case["wide"], case["vocab"]
    if case["model"] == "tokens":
        block = [(width, False)] + [(width * width, True)] * 4 + [(width, False)] + [(width * wide, True)] * 2
        return [(vocab * width, True)] + block * blocks + [(width, False)]
    if case["model"] == "detector":
        # residual blocks of a 1x1 and a 3x3 convolution with scale and bias each, at doubling widths, and three heads
        tensors, per = [], max(1, blocks // 5)
        for stage in range(5):
            c = width >> (4 - stage)
            for _ in range(per):
                tensors += [(c * c // 2, True), (c // 2, False), (c // 2, False), (9 * c * c // 2, True), (c, False), (c, False)]
        for c in (width, width // 2, width // 4):
            tensors += [(c * c // 2, True), (9 * c * c // 2, True), (c, False), (c, False), (255 * c, True), (255, False)] * 3
        return tensors
    return [((width + 7 * i) * (i % 5 + 1) ** 2 | 1 if i % 3 else width + i, i % 3 != 0) for i in range(blocks)]


def _arena(case):
    """Where each tensor begins in a buffer in which all begin at a multiple of BLOCK values, and that buffer's length."""
    starts, at = [], 0
    for n, _ in _parameters(case):
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def _views(flat, case):
    return [flat[a:a + n] for a, (n, _) in zip(_arena(case)[0], _parameters(case))]


def _blocks_max(x):
    return x.view(-1, BLOCK).abs().amax(1)


def _adamw_state(case, g):
    starts, total = _arena(case)
    sizes = _parameters(case)
    real = torch.zeros(total, device="cuda", dtype=torch.bool)
    decays = torch.zeros(total // BLOCK, device="cuda")
    # gradients of tensors differ in size, and so do those of the values of one
    size = torch.zeros(total // BLOCK, device="cuda")
    for i, (a, (n, decay)) in enumerate(zip(starts, sizes)):
        real[a:a + n] = True
        decays[a // BLOCK:(a + n + BLOCK - 1) // BLOCK] = float(decay)
        size[a // BLOCK:(a + n + BLOCK - 1) // BLOCK] = 1e-4 * 2.0 ** (i % 7)
    size = size.repeat_interleave(BLOCK).mul_(_normal(g, total, 0.7).exp_())
    w = _normal(g, total, 0.02).mul_(real)
    d = (_normal(g, total) * size).mul_(real).to(TYPES[case["gradients"]])
    m = _normal(g, total, 0.3).mul_(size).mul_(real)
    root = size.mul_(real).mul_(_normal(g, total, 0.1).exp_())             # square root of the second moment
    state = {"w": w, "d": d, "decays": decays, "copy": w.bfloat16() if case["copies"] else None, "norm": torch.zeros(1, device="cuda")}
    if case["bits"] == 8:
        for name, x in (("m", m), ("v", root)):
            scale = (_blocks_max(x) / E4M3_MAX).clamp_(min=LEAST_SCALE)
            state[name] = (x.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
            state[name + "_scale"] = scale
    else:
        state["m"], state["v"] = m, root.square_()
    if own:
        from pixienn_amd import ops
        scales = [[t[a // BLOCK:(a + n + BLOCK - 1) // BLOCK] for a, (n, _) in zip(starts, sizes)]
                  for t in (state["m_scale"], state["v_scale"])] if case["bits"] == 8 else (None, None)
        state["table"] = ops.AdamwTable(*(_views(state[k], case) for k in "wdmv"), m_scales=scales[0], v_scales=scales[1],
                                        copies=_views(state["copy"], case) if case["copies"] else None,
                                        apply_decay=[decay for _, decay in sizes])
    return state


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    state = {"case": dict(case)}
    if kind in ("norm", "norm_backward"):
        rows, width, kind_of_type = case["rows"], case["width"], TYPES[case["type"]]
        state["weight"] = (1.0 + _normal(g, width, 0.2)).to(kind_of_type)
        x = _rows(g, case)
        # a few channels of a residual stream are far larger than the others
        x[:, torch.randint(0, width, (max(1, width // 200),), device="cuda", generator=g)] *= 15.0
        empty = lambda: torch.empty(rows, width, device="cuda", dtype=kind_of_type)  # noqa: E731
        if kind == "norm":
            state["x"] = x
            if case["residual"]:
                state["residual"], state["sum"] = _rows(g, case, 2.0), empty()
            state["rstd"] = torch.empty(rows, device="cuda")
            if case["out"] == "same":
                state["y"] = empty()
            else:
                state["y"] = torch.empty(rows, width, device="cuda", dtype=torch.float8_e4m3fn)
                state["scales"] = torch.empty(rows, 1 if case["out"] == "row" else -(-width // GROUP), device="cuda")
            return state
        state["h"], state["dy"] = x, _rows(g, case, 1e-2)
        state["rstd"] = torch.rsqrt(x.float().square().mean(1) + EPS)
        state["dsum"] = _rows(g, case, 1e-2) if case["residual"] else None
        state["dx"], state["dw"] = empty(), torch.empty(width, device="cuda")
        return state
    if kind.startswith("tokens"):
        rows, vocab = case["rows"], case["vocab"]
        logits = _normal(g, (rows, vocab), 2.5, TYPES[case["type"]])
        targets = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
        # the given token is a likely one, as a trained model has it
        logits.scatter_add_(1, targets[:, None], _normal(g, (rows, 1), 3.0).add_(9.0).to(logits.dtype))
        if case.get("masked"):
            allowed = torch.rand(rows, vocab, device="cuda", generator=g) >= case["masked"]
            allowed.scatter_(1, targets[:, None], True)
            logits.masked_fill_(~allowed, -math.inf)
        state.update(logits=logits, targets=targets)
        if kind != "tokens":
            targets.masked_fill_(torch.rand(rows, device="cuda", generator=g) < 0.03, -1)       # nothing to be learned there
            state["d_logp"] = torch.rand(rows, device="cuda", generator=g).add_(0.5).div_(rows)
            state["d_entropy"] = _normal(g, rows, 0.1 / rows) if case["entropy"] else None
            state["dlogits"] = torch.empty_like(logits)
        state["logp"], state["entropy"], state["lse"] = (torch.empty(rows, device="cuda") for _ in range(3))
        if kind == "tokens_backward":
            z = logits.double() * case["scale"]
            state["lse"] = torch.logsumexp(z, 1).float()
            state["entropy"] = (torch.logsumexp(z, 1) - (torch.softmax(z, 1) * z).sum(1)).float()
        if case.get("top"):
            state["top_logp"] = torch.empty(rows, case["top"], device="cuda")
            state["top_ids"] = torch.empty(rows, case["top"], device="cuda", dtype=torch.int32)
        return state
    state.update(_adamw_state(case, g), t=100, lr=5e-5, d_scale=0.5, seed=seed * 7919 + 13)
    return state


# ---------------------------------------------------------------- plain forms
def _plain_norm(s):
    case = s["case"]
    h = s["x"]
    out = {}
    if case["residual"]:
        h = (h.float() + s["residual"].float()).to(h.dtype)
        out["sum"] = h
    h = h.float()
    rstd = torch.rsqrt(h.square().mean(1) + EPS)
    y = h * rstd[:, None] * s["weight"].float()
    if case["out"] == "same":
        y = y.to(s["x"].dtype)
    else:
        rows, width = y.shape
        group = width if case["out"] == "row" else GROUP
        groups = -(-width // group)
        y = torch.nn.functional.pad(y, (0, groups * group - width)).view(rows, groups, group)
        scales = (y.abs().amax(2) / E4M3_MAX).clamp(min=LEAST_SCALE)
        y = (y / scales[:, :, None]).to(torch.float8_e4m3fn).view(rows, groups * group)[:, :width]
        out["scales"] = scales
    return dict(out, y=y, rstd=rstd)


def _plain_norm_backward(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = s["h"].float() * rstd
    dyw = dy * s["weight"].float()
    dx = rstd * (dyw - xhat * (dyw * xhat).mean(1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    return {"dx": dx.to(s["h"].dtype), "dw": (dy * xhat).sum(0)}


def _plain_statistics(s):
    z = s["logits"].float() * s["case"]["scale"]
    peak = z.amax(1, keepdim=True)
    shifted = z - torch.where(peak == -math.inf, 0.0, peak)
    e = shifted.exp()
    total = e.sum(1, keepdim=True)
    lse = torch.where(peak == -math.inf, peak, peak + total.log())
    entropy = total.log() - (e * shifted.clamp(min=-128.0)).sum(1, keepdim=True) / total
    entropy = torch.where(peak == -math.inf, 0.0, entropy)
    return z, lse, entropy


def _plain_logp(s, z, lse):
    target = s["targets"][:, None]
    given = (target >= 0) & (target < z.shape[1])
    logp = z.gather(1, torch.where(given, target, 0)) - lse
    logp = torch.where(lse == -math.inf, lse, logp)
    return torch.where(given, logp, 0.0)[:, 0], given


def _plain_gradient(s, z, lse, entropy):
    target = s["targets"][:, None]
    given = (target >= 0) & (target < z.shape[1])
    g = torch.where(given, s["d_logp"][:, None], 0.0)
    logs = (z - lse).clamp(min=-128.0)
    p = (z - lse).exp()
    d = -g * p
    if s["d_entropy"] is not None:
        d = d - s["d_entropy"][:, None] * p * (logs + entropy)
    d.scatter_add_(1, torch.where(given, target, 0), g)
    return torch.where(lse == -math.inf, 0.0, d * s["case"]["scale"]).to(s["logits"].dtype)


def _plain_tokens(s):
    z, lse, entropy = _plain_statistics(s)
    out = {"logp": _plain_logp(s, z, lse)[0], "entropy": entropy[:, 0], "lse": lse[:, 0]}
    if s["case"]["top"]:
        # one whole number per value that orders by value, then by the lowest index
        bits = z.add(0.0).view(torch.int32).to(torch.int64)
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        index = torch.arange(z.shape[1], device=z.device)
        key = order * (1 << 31) + ((1 << 31) - 1 - index)
        ids = (1 << 31) - 1 - (key.topk(s["case"]["top"], dim=1).values & ((1 << 31) - 1))
        out.update(top_ids=ids.to(torch.int32), top_logp=z.gather(1, ids) - lse)
    return out


def _plain_tokens_train(s):
    z, lse, entropy = _plain_statistics(s)
    return {"dlogits": _plain_gradient(s, z, lse, entropy), "logp": _plain_logp(s, z, lse)[0], "entropy": entropy[:, 0], "lse": lse[:, 0]}


def _plain_tokens_backward(s):
    z = s["logits"].float() * s["case"]["scale"]
    return {"dlogits": _plain_gradient(s, z, s["lse"][:, None], s["entropy"][:, None])}


def _mix(x):
    """A 32-bit mix of whole numbers held in 32 bits: two rounds of an odd factor and the high bits folded into the low ones."""
    for factor, shift in ((0x9E3779B9, 15), (0x6A09E667, 13)):
        x = x * (factor - (1 << 32) if factor >= 1 << 31 else factor)
        x = x ^ ((x >> shift) & ((1 << (32 - shift)) - 1))
    return x


def _random(total, seed):
    """32 random bits for each place, as signed whole numbers."""
    start = torch.full((1,), (seed & 0x7FFFFFFF), device="cuda", dtype=torch.int32)
    return _mix(torch.arange(total, device="cuda", dtype=torch.int32) ^ _mix(start + 1))


def _stochastic(x, noise, least):
    """Values in blocks rounded to e4m3 by 20 random bits: up with the probability of the part that is cut off."""
    scale = (x.abs().amax(1) / E4M3_MAX).clamp(min=LEAST_SCALE)
    small = (x.abs() / scale[:, None]).clamp(max=E4M3_MAX) * 2.0 ** -120   # the exponent's field is e4m3's then
    code = ((small.view(torch.int32) + noise) >> 20).clamp(max=0x7E)
    code = torch.where(x != 0, code.clamp(min=least), code)
    return (code | ((x < 0).to(torch.int32) << 7)).to(torch.uint8).view(torch.float8_e4m3fn), scale


def _plain_adamw(s):
    case = s["case"]
    d = s["d"].float() * s["d_scale"]
    if case["max_norm"]:
        s["norm"].copy_(d.square().sum().sqrt())
        d = d * torch.where(s["norm"] > case["max_norm"], case["max_norm"] / s["norm"], 1.0)
    eight = case["bits"] == 8
    m, v = s["m"], s["v"]
    if eight:
        m = (m.float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1).square()
    m = BETA1 * m + (1.0 - BETA1) * d
    v = BETA2 * v + (1.0 - BETA2) * d.square()
    root = v.sqrt()
    step = (m / (1.0 - BETA1 ** s["t"])) / (root / math.sqrt(1.0 - BETA2 ** s["t"]) + ADAM_EPS)
    shrink = (s["w"].view(-1, BLOCK) * (s["lr"] * DECAY * s["decays"][:, None])).view(-1)
    s["w"].add_(s["lr"] * step).sub_(shrink)
    if eight:
        noise = _random(d.numel(), s["seed"])
        for name, x, bits, least in (("m", m, (noise >> 12) & 0xFFFFF, 0), ("v", root, noise & 0xFFFFF, 1)):
            code, scale = _stochastic(x.view(-1, BLOCK), bits.view(-1, BLOCK), least)
            s[name].copy_(code.view(-1))
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if s["copy"] is not None:
        s["copy"].copy_(s["w"])
    return _adamw_outputs(s)


def _adamw_outputs(s):
    out = {k: s[k] for k in ("w", "m", "v", "m_scale", "v_scale", "copy") if s.get(k) is not None}
    if s["case"]["max_norm"]:
        out["norm"] = s["norm"]
    return out


PLAIN = {"norm": _plain_norm, "norm_backward": _plain_norm_backward, "tokens": _plain_tokens, "tokens_train": _plain_tokens_train,
         "tokens_backward": _plain_tokens_backward, "adamw": _plain_adamw}


# ---------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return PLAIN[kind](s)
    from pixienn_amd import ops
    if kind == "norm":
        ops.rms_norm_forward(s["x"], s["y"], s["weight"], residual=s.get("residual"), sum=s.get("sum"), scales=s.get("scales"),
                             rstd=s["rstd"], eps=EPS, group=GROUP if case["out"] == "group" else 0)
        return {k: s[k] for k in ("sum", "y", "scales", "rstd") if k in s}
    if kind == "norm_backward":
        ops.rms_norm_backward(s["dy"], s["h"], s["weight"], s["rstd"], s["dx"], s["dw"], dsum=s["dsum"])
        return {"dx": s["dx"], "dw": s["dw"]}
    if kind == "tokens":
        ops.token_logprobs_forward(s["logits"], s["targets"], s["logp"], entropy=s["entropy"], lse=s["lse"],
                                   top_logp=s.get("top_logp"), top_ids=s.get("top_ids"), scale=case["scale"])
        return {k: s[k] for k in ("logp", "entropy", "lse", "top_logp", "top_ids") if k in s}
    if kind == "tokens_train":
        ops.token_logprobs_forward_train(s["logits"], s["targets"], s["d_logp"], s["dlogits"], s["logp"], entropy=s["entropy"],
                                         lse=s["lse"], d_entropy=s["d_entropy"], scale=case["scale"])
        return {k: s[k] for k in ("dlogits", "logp", "entropy", "lse")}
    if kind == "tokens_backward":
        ops.token_logprobs_backward(s["logits"], s["targets"], s["lse"], s["d_logp"], s["dlogits"], entropy=s["entropy"],
                                    d_entropy=s["d_entropy"], scale=case["scale"])
        return {"dlogits": s["dlogits"]}
    s["table"].update(s["t"], s["lr"], BETA1, BETA2, ADAM_EPS, DECAY, d_scale=s["d_scale"], max_norm=case["max_norm"],
                      norm_out=s["norm"] if case["max_norm"] else None, seed=s["seed"])
    return _adamw_outputs(s)


def work(case):
    kind = case["kind"]
    if kind == "adamw":
        n = sum(n for n, _ in _parameters(case))
        state = 2 * 2 + 16 / BLOCK if case["bits"] == 8 else 16
        size = 2 if case["gradients"] != "f32" else 4
        # clipping by the norm of all gradients needs them all before the first step: they are read again
        return {"bytes": n * (8 + state + size * (2 if case["max_norm"] else 1) + (2 if case["copies"] else 0)), "flops": 16.0 * n}
    size = 4 if case["type"] == "f32" else 2
    rows = case["rows"]
    if kind == "norm":
        n = rows * case["width"]
        out = n * size if case["out"] == "same" else n + 4 * rows * (1 if case["out"] == "row" else -(-case["width"] // GROUP))
        return {"bytes": n * size * (3 if case["residual"] else 1) + out + 4 * rows + size * case["width"], "flops": 5.0 * n}
    if kind == "norm_backward":
        n = rows * case["width"]
        return {"bytes": n * size * (4 if case["residual"] else 3) + 4 * rows + (size + 4) * case["width"], "flops": 9.0 * n}
    n = rows * case["vocab"]
    if kind == "tokens":
        return {"bytes": n * size + rows * (20 + 8 * case["top"]), "flops": 5.0 * n}
    return {"bytes": 2 * n * size + rows * 28, "flops": (9.0 if kind == "tokens_train" else 5.0) * n}


# ---------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        h = s["x"].double()
        out = {}
        if case["residual"]:
            h = out["sum"] = h + s["residual"].double()
            h = h.to(s["x"].dtype).double()            # the norm is that of the sum as it is kept
        power = torch.linalg.vector_norm(h, dim=1) ** 2 / case["width"]
        out["rstd"] = 1.0 / torch.sqrt(power + EPS)
        y = s["weight"].double() * h * out["rstd"][:, None]
        if case["out"] != "same":
            parts = y.split(case["width"] if case["out"] == "row" else GROUP, dim=1)
            scales = [torch.linalg.vector_norm(p, ord=math.inf, dim=1, keepdim=True) / E4M3_MAX for p in parts]
            y = torch.cat([p / c for p, c in zip(parts, scales)], 1)
            out["scales"] = torch.cat(scales, 1)
        return dict(out, y=y)
    if kind == "norm_backward":
        h = s["h"].double().requires_grad_()
        w = s["weight"].double().requires_grad_()
        with torch.enable_grad():
            y = h * w / torch.sqrt((h * h).sum(1, keepdim=True) / case["width"] + EPS)
            dx, dw = torch.autograd.grad(y, (h, w), s["dy"].double())
        return {"dx": dx if s["dsum"] is None else dx + s["dsum"].double(), "dw": dw}
    if kind.startswith("tokens"):
        z = s["logits"].double() * case["scale"]
        logs = torch.log_softmax(z, 1)
        p = logs.exp()
        entropy = -torch.special.xlogy(p, p).sum(1)
        row = torch.arange(case["rows"], device="cuda")
        given = s["targets"] >= 0
        chosen = s["targets"].clamp(min=0)
        out = {"logp": logs[row, chosen] * given, "entropy": entropy, "lse": torch.logsumexp(z, 1)}
        if kind == "tokens":
            if case["top"]:
                out["top_logp"] = logs.topk(case["top"], dim=1).values
                out["top_ids"] = None
            return out
        g = s["d_logp"].double() * given
        grad = -p * g[:, None]
        grad[row, chosen] += g
        if s["d_entropy"] is not None:
            grad -= s["d_entropy"].double()[:, None] * (torch.special.xlogy(p, p) + p * entropy[:, None])
        grad *= case["scale"]
        return {"dlogits": grad} if kind == "tokens_backward" else dict(out, dlogits=grad)
    w, d = s["w"].double(), s["d"].double() * s["d_scale"]
    out = {}
    if case["max_norm"]:
        out["norm"] = torch.linalg.vector_norm(d).view(1)
        d *= min(1.0, case["max_norm"] / float(out["norm"]))
    if case["bits"] == 8:
        m = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (s["v"].double() * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m = torch.lerp(d, m, BETA1)
    v = torch.lerp(d * d, v, BETA2)
    rate = s["lr"] / (1.0 - BETA1 ** s["t"])
    out["w"] = w - w * s["lr"] * DECAY * s["decays"].double().repeat_interleave(BLOCK) \
        + rate * m / (torch.sqrt(v / (1.0 - BETA2 ** s["t"])) + ADAM_EPS)
    if case["copies"]:
        out["copy"] = out["w"]
    if case["bits"] == 8:
        # a state in 8 bits has no exact value but the one it is rounded from
        for name, x in (("m", m), ("v", torch.sqrt(v))):
            scale = torch.linalg.vector_norm(x.view(-1, BLOCK), ord=math.inf, dim=1) / E4M3_MAX
            out[name + "_scale"] = scale
            out[name] = (x.view(-1, BLOCK) / scale.clamp(min=LEAST_SCALE)[:, None]).view(-1)
        return out
    return dict(out, m=m, v=v)

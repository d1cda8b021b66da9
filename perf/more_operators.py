"""More operators of token models: what is timed, through `pixienn_amd.ops`, and the same in plain torch operations.

What a network over tokens needs besides its matrix products, and besides the norm, the token log probabilities and the optimiser
that are there.  The products are not part of it: every case starts from synthetic ones.  Kinds of case:

  embedding, embedding_backward
                 rows of a table looked up by token, with a scale; the gradient of the table, overwritten or added to
  layer_norm, layer_norm_backward
                 norm by mean and variance with the residual's addition in front of it; its gradients, with those of weight and bias
  scan, scan_backward, scan_step
                 a gated linear recurrence over sequences, h = h + sigmoid(update) * (x - h), y = h * gate * sigmoid(gate): whole
                 sequences of one length or of ragged ones with states kept in slots, the gradients, one new token of each sequence
  beam           beam search: the best continuations over beams and vocabulary, and the beams' states in their new order

`run` computes in plain torch operations, or, with `own`, by the calls that a user makes.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5                      # of the norm


def listed():
    return [
        # a batch of prompts, or a training step's forward pass: embeddings scaled by the root of the width
        dict(name="embedding_16384x4096_bf16", kind="embedding", rows=16384, width=4096, vocab=50001, type="bf16", scale=64.0, pad=0),
        # a training step's gradient, in the type of the products' gradients; text has few frequent tokens and many rare ones
        dict(name="embedding_backward_16384x2048_bf16", kind="embedding_backward", rows=16384, width=2048, vocab=32768, type="bf16",
             out="same", accumulate=False, scale=1.0, pad=0),
        # a further short batch added to the gradient, full precision, odd sizes
        dict(name="embedding_backward_4099x1025_f32", kind="embedding_backward", rows=4099, width=1025, vocab=10007, type="f32",
             out="f32", accumulate=True, scale=32.0, pad=0),
        # serving: the running sequences' newest tokens
        dict(name="layer_norm_16x4096_bf16", kind="layer_norm", rows=16, width=4096, type="bf16", residual=True, bias=True, pad=0),
        # training in full precision on a slice of wider rows, odd width
        dict(name="layer_norm_2111x5001_f32", kind="layer_norm", rows=2111, width=5001, type="f32", residual=False, bias=True, pad=23),
        # a training step's gradients of one norm
        dict(name="layer_norm_backward_16384x4096_bf16", kind="layer_norm_backward", rows=16384, width=4096, type="bf16", residual=True,
             bias=True, pad=0),
        # training: whole sequences of one length, with an output gate
        dict(name="scan_8x4096x2048_bf16", kind="scan", sequences=8, tokens=32768, width=2048, type="bf16", gate=True, ragged=False),
        # serving: a batch of prompts of ragged lengths, of which some go on from a state
        dict(name="scan_31_prompts_30011x2561_f16", kind="scan", sequences=31, tokens=30011, width=2561, type="f16", gate=False, ragged=True),
        # the gradients of the training pass
        dict(name="scan_backward_8x4096x2048_bf16", kind="scan_backward", sequences=8, tokens=32768, width=2048, type="bf16", gate=True,
             ragged=False),
        # serving: one new token for each running sequence
        dict(name="scan_step_64x4096_bf16", kind="scan_step", sequences=64, tokens=64, width=4096, type="bf16", gate=True, ragged=False),
        # serving: one prompt, four beams of which one has ended, a large vocabulary
        dict(name="beam_1x4x131072_bf16", kind="beam", batch=1, beams=4, vocab=131072, type="bf16", scale=1.0, ended=0.25, layers=8,
             width=2048, history=100),
        # a batch of texts with eight beams each, odd vocabulary
        dict(name="beam_64x8x50001_f16", kind="beam", batch=64, beams=8, vocab=50001, type="f16", scale=0.8, ended=0.1, layers=4, width=1024,
             history=301),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, step):
    """Spread over the logarithm: a power of two, a multiple of `step`, or odd."""
    n = _log_int(rng, lo, hi)
    return rng.choice([max(lo, 1 << n.bit_length() - 1), max(lo, n // step * step), n | 1])


def draw(rng):
    kind = rng.choice(["embedding", "embedding_backward", "embedding_backward", "layer_norm", "layer_norm_backward", "scan", "scan",
                       "scan_backward", "scan_backward", "scan_step", "beam", "beam"])
    value = rng.choice(["bf16", "bf16", "f16", "f32"])
    half = 2 if value == "f32" else 1
    if kind.startswith("embedding"):
        width = _size(rng, 64, 8192, 80)
        vocab = _size(rng, 256, min(160000, 32768 * 2048 // half // width), 80)
        case = dict(kind=kind, rows=_log_int(rng, 1, min(65536, 16384 * 2048 // half // width)), width=width, vocab=vocab, type=value,
                    scale=rng.choice([1.0, 1.0, 0.5, 32.0]), pad=rng.choice([0, 0, 8, 13]))
        if kind == "embedding_backward":
            case.update(out=rng.choice(["same", "f32"]) if 2 * width * vocab <= 32768 * 2048 else "same", accumulate=rng.random() < 0.4)
        return case
    if kind.startswith("layer_norm"):
        width = _size(rng, 64, 16384, 80)
        return dict(kind=kind, rows=_log_int(rng, 1, min(16384, 16384 * 4096 // half // width)), width=width, type=value,
                    residual=rng.random() < 0.6, bias=rng.random() < 0.8, pad=rng.choice([0, 0, 8, 13]))
    if kind.startswith("scan"):
        width = _size(rng, 64, 8192, 80)
        if kind == "scan_step":
            sequences = _log_int(rng, 1, 512)
            return dict(kind=kind, sequences=sequences, tokens=sequences, width=width, type=value, gate=rng.random() < 0.6, ragged=False)
        tokens = _log_int(rng, 16, min(65536, 32768 * 2048 // half // width))
        ragged = rng.random() < 0.5
        sequences = _log_int(rng, 1, max(1, min(64, tokens // 4)))
        if not ragged:
            tokens = tokens // sequences * sequences
        return dict(kind=kind, sequences=sequences, tokens=tokens, width=width, type=value, gate=rng.random() < 0.6, ragged=ragged)
    vocab = _size(rng, 1000, 160000, 80)
    beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
    return dict(kind=kind, batch=_log_int(rng, 1, max(1, min(128, 64 * 8 * 50001 // half // (beams * vocab)))), beams=beams, vocab=vocab,
                type=value, scale=rng.choice([1.0, 1.0, 0.7, 1.3]), ended=rng.choice([0.0, 0.2, 0.6]), layers=rng.randint(1, 6),
                width=_size(rng, 64, 1024, 80), history=rng.randint(1, 300))


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


def _text(g, rows, vocab):
    """Tokens as texts have them, the k-th most frequent one about 1 / k as often as the first; some places have none (-1)."""
    weights = 1.0 / (torch.arange(vocab, device="cuda", dtype=torch.float64) + 2.7)
    ranks = torch.searchsorted(weights.cumsum(0), torch.rand(rows, device="cuda", dtype=torch.float64, generator=g) * weights.sum())
    tokens = torch.randperm(vocab, device="cuda", generator=g)[ranks.clamp(max=vocab - 1)]
    return tokens.masked_fill_(torch.rand(rows, device="cuda", generator=g) < 0.02, -1)


def _lengths(case, seed):
    """Lengths of sequences that add up to the tokens: most short, a few long, with an empty one and one of a single token."""
    sequences, tokens = case["sequences"], case["tokens"]
    if not case["ragged"]:
        return [tokens // sequences] * sequences
    g = torch.Generator()
    g.manual_seed(seed + 1)
    cuts = torch.rand(sequences, generator=g, dtype=torch.float64).pow_(-0.8)
    cuts = (cuts.cumsum(0) / cuts.sum() * tokens).round().long()
    lengths = cuts.diff(prepend=cuts.new_zeros(1)).tolist()
    if sequences > 4:
        lengths[2] += lengths[1] + lengths[3] - 1
        lengths[1], lengths[3] = 0, 1
        if lengths[2] < 0:
            most = lengths.index(max(lengths))
            lengths[most] += lengths[2]
            lengths[2] = 0
    return lengths


def _scan_state(case, seed, g):
    width, value, sequences = case["width"], TYPES[case["type"]], case["sequences"]
    behind = 19 if case["ragged"] else 0                # rows behind the last sequence, as a batch of a fixed size has them
    rows = case["tokens"] + behind
    # some channels forget at once, some remember for thousands of tokens
    bias = torch.rand(width, device="cuda", generator=g).mul_(-8.0)
    tensors = {"x": _normal(g, (rows, width), 1.0, value), "update": _normal(g, (rows, width)).add_(bias).to(value)}
    tensors["gate"] = _normal(g, (rows, width), 1.0, value) if case["gate"] else None
    s = dict(tensors, lengths=_lengths(case, seed), dgate=None)
    lengths = torch.tensor(s["lengths"])
    ends = lengths.cumsum(0)
    full = torch.nonzero(lengths)[:, 0]
    # sequences that are not empty, their first tokens, their last ones
    s["borders"] = full.cuda(), (ends - lengths)[full].cuda(), (ends - 1)[full].cuda()
    if case["ragged"]:
        s["starts"] = torch.tensor([0] + s["lengths"], device="cuda").cumsum(0).to(torch.int32)
    if case["ragged"] or case["kind"] == "scan_step":
        slots = torch.randperm(sequences + 5, device="cuda", generator=g)[:sequences].to(torch.int32)
        if sequences > 6:
            slots[5] = -1                               # a sequence of which no state is kept
        s["slots"] = slots
        s["state"] = _normal(g, (sequences + 5, width), 0.5)
        if case["kind"] == "scan":
            s["final"] = torch.zeros_like(s["state"])
        elif case["kind"] == "scan_backward":
            s["d_final"] = _normal(g, (sequences + 5, width), 1e-2)
            s["d_state"] = torch.zeros_like(s["state"])
    if case["kind"] == "scan_backward":
        s["dy"] = _normal(g, (rows, width), 1e-2, value)
        for name in ("dx", "dupdate") + (("dgate",) if case["gate"] else ()):
            s[name] = torch.zeros(rows, width, device="cuda", dtype=value)
    else:
        s["y"] = torch.zeros(rows, width, device="cuda", dtype=value)
    if own and case["kind"] != "scan_step" and (case["kind"] == "scan_backward" or not case["ragged"]):
        from pixienn_amd import ops
        s["saved"] = ops.gated_scan_saved_like(s["x"])
        if case["kind"] == "scan_backward":
            y = torch.empty_like(s["x"])
            ops.gated_scan_forward(s["x"], s["update"], y, gate=s["gate"], starts=s.get("starts"), sequences=sequences, state=s.get("state"),
                                   slots=s.get("slots"), saved=s["saved"])
    return s


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    state = {"case": dict(case)}
    value = TYPES[case["type"]]
    if kind == "embedding":
        rows, width, pad = case["rows"], case["width"], case["pad"]
        state["table"] = _normal(g, (case["vocab"], width), 0.02, value)
        state["tokens"] = _text(g, rows, case["vocab"])
        state["y"] = torch.empty(rows, width + pad, device="cuda", dtype=value)[:, :width]
    elif kind == "embedding_backward":
        state["dy"] = _rows(g, case, 1e-2)
        state["tokens"] = _text(g, case["rows"], case["vocab"]).to(torch.int32)
        out = value if case["out"] == "same" else torch.float32
        shape = (case["vocab"], case["width"])
        state["d"] = _normal(g, shape, 0.3, out) if case["accumulate"] else torch.empty(shape, device="cuda", dtype=out)
    elif kind.startswith("layer_norm"):
        rows, width = case["rows"], case["width"]
        state["weight"] = (1.0 + _normal(g, width, 0.2)).to(value)
        state["bias"] = _normal(g, width, 0.2).to(value) if case["bias"] else None
        x = _rows(g, case)
        # a few channels of a residual stream are far larger than the others, and a row's mean is not zero
        x[:, torch.randint(0, width, (max(1, width // 200),), device="cuda", generator=g)] *= 15.0
        x += _normal(g, (rows, 1), 0.5).to(value)
        empty = lambda: torch.empty(rows, width, device="cuda", dtype=value)  # noqa: E731
        if kind == "layer_norm":
            state.update(x=x, y=empty(), mean=torch.empty(rows, device="cuda"), rstd=torch.empty(rows, device="cuda"))
            if case["residual"]:
                state.update(residual=_rows(g, case, 2.0), sum=empty())
        else:
            h = x.double()
            mean = h.mean(1)
            state.update(h=x, dy=_rows(g, case, 1e-2), mean=mean.float(), rstd=torch.rsqrt((h - mean[:, None]).square().mean(1) + EPS).float())
            state["dsum"] = _rows(g, case, 1e-2) if case["residual"] else None
            state.update(dx=empty(), dw=torch.empty(width, device="cuda"), db=torch.empty(width, device="cuda") if case["bias"] else None)
    elif kind.startswith("scan"):
        state.update(_scan_state(case, seed, g))
    else:
        batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
        logits = _normal(g, (batch * beams, vocab), 2.5, value)
        # one token is likely, a few more are possible
        likely = torch.randint(0, vocab, (batch * beams, 5), device="cuda", generator=g)
        logits.scatter_add_(1, likely, _normal(g, likely.shape, 2.0).add_(7.0).to(value))
        state["logits"] = logits
        state["scores"] = _normal(g, (batch, beams), 1.0).sub_(12.0)
        state["ended"] = torch.rand(batch, beams, device="cuda", generator=g) < case["ended"] if case["ended"] else None
        state["best"] = torch.empty(batch, beams, device="cuda")
        state["parents"], state["tokens"] = (torch.empty(batch, beams, device="cuda", dtype=torch.int32) for _ in range(2))
        state["states"] = [_normal(g, (batch * beams, case["width"])) for _ in range(case["layers"])]
        state["states"].append(torch.randint(0, vocab, (batch * beams, case["history"]), device="cuda", generator=g).to(torch.int32))
    return state


# ---------------------------------------------------------------- plain forms
def _plain_embedding(s):
    tokens = s["tokens"]
    given = (tokens >= 0) & (tokens < len(s["table"]))
    rows = s["table"][torch.where(given, tokens, 0)].float() * s["case"]["scale"]
    return {"y": (rows * given[:, None]).to(s["table"].dtype)}


def _plain_embedding_backward(s):
    d, tokens = s["d"], s["tokens"].long()
    vocab = len(d)
    total = torch.zeros(vocab + 1, d.shape[1], device="cuda")
    total.index_add_(0, torch.where((tokens >= 0) & (tokens < vocab), tokens, vocab), s["dy"].float())
    total = total[:vocab] * s["case"]["scale"]
    if s["case"]["accumulate"]:
        total = total + d.float()
    d.copy_(total)
    return {"d": d}


def _plain_layer_norm(s):
    h = s["x"]
    out = {}
    if s["case"]["residual"]:
        h = out["sum"] = (h.float() + s["residual"].float()).to(h.dtype)
    h = h.float()
    mean = h.mean(1, keepdim=True)
    centred = h - mean
    rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + EPS)
    y = centred * rstd * s["weight"].float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return dict(out, y=y.to(s["x"].dtype), mean=mean[:, 0], rstd=rstd[:, 0])


def _plain_layer_norm_backward(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["h"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    out = {"dx": dx.to(s["h"].dtype), "dw": (dy * xhat).sum(0)}
    if s["db"] is not None:
        out["db"] = dy.sum(0)
    return out


def _linear(a, b, longest):
    """h[t] = a[t] * h[t - 1] + b[t] from zero, with an a of zero at least every `longest` rows: within parts of the rows at once, then
    from part to part."""
    if longest <= 1:
        return b
    rows, width = b.shape
    part = min(math.isqrt(rows - 1) + 1, longest)
    parts = -(-rows // part)
    a, b = (torch.cat([t, t.new_zeros(parts * part - rows, width)]).view(parts, part, width) for t in (a, b))
    for i in range(1, part):
        b[:, i] += a[:, i] * b[:, i - 1]
        a[:, i] *= a[:, i - 1]
    for k in range(1, parts):
        b[k] += a[k] * b[k - 1, -1]
    return b.view(parts * part, width)[:rows]


def _of_slots(s, states):
    """A row of `states` for each sequence, zeros where none is kept."""
    if s.get(states) is None:
        return torch.zeros(len(s["lengths"]), s["case"]["width"], device="cuda")
    slots = s["slots"].long()
    kept = (slots >= 0) & (slots < len(s[states]))
    return s[states][torch.where(kept, slots, 0)] * kept[:, None]


def _into_slots(s, states, values):
    slots = s["slots"].long()
    kept = (slots >= 0) & (slots < len(states))
    states[slots[kept]] = values[kept]


def _plain_recurrence(s):
    """(h, h of the token before, 1 - z) of the tokens of all sequences."""
    n = s["case"]["tokens"]
    x, update = s["x"][:n].float(), s["update"][:n].float()
    z, keep = torch.sigmoid(update), torch.sigmoid(-update)
    full, first, _ = s["borders"]
    init = _of_slots(s, "state")
    a, b = keep.clone(), z * x
    b[first] += keep[first] * init[full]
    a[first] = 0.0
    h = _linear(a, b, max(s["lengths"]))
    before = torch.cat([h.new_zeros(1, h.shape[1]), h[:-1]])
    before[first] = init[full]
    return h, before, z, keep


def _plain_scan(s):
    n = s["case"]["tokens"]
    h = _plain_recurrence(s)[0]
    y = h
    if s["gate"] is not None:
        gate = s["gate"][:n].float()
        y = h * gate * torch.sigmoid(gate)
    s["y"][:n] = y.to(s["y"].dtype)
    out = {"y": s["y"]}
    target = s["state"] if s["case"]["kind"] == "scan_step" else s.get("final")
    if target is not None:
        full, _, last = s["borders"]
        values = _of_slots(s, "state")
        values[full] = h[last]
        _into_slots(s, target, values)
        out["final"] = target
    return out


def _plain_scan_backward(s):
    n = s["case"]["tokens"]
    h, before, z, keep = _plain_recurrence(s)
    dy, x = s["dy"][:n].float(), s["x"][:n].float()
    grad = dy
    if s["gate"] is not None:
        gate = s["gate"][:n].float()
        open_ = torch.sigmoid(gate)
        grad = dy * gate * open_
        s["dgate"][:n] = (dy * h * open_ * (1.0 + gate * torch.sigmoid(-gate))).to(s["dgate"].dtype)
    full, first, last = s["borders"]
    d_final = _of_slots(s, "d_final")
    grad = grad.clone()
    grad[last] += d_final[full]
    # what reaches a token from the next one of its sequence
    a = torch.cat([keep[1:], keep.new_zeros(1, keep.shape[1])])
    a[last] = 0.0
    total = _linear(a.flip(0), grad.flip(0), max(s["lengths"])).flip(0)
    s["dx"][:n] = (z * total).to(s["dx"].dtype)
    s["dupdate"][:n] = (total * (x - before) * z * keep).to(s["dupdate"].dtype)
    out = {"dx": s["dx"], "dupdate": s["dupdate"]}
    if s["gate"] is not None:
        out["dgate"] = s["dgate"]
    if s.get("d_state") is not None:
        d_final[full] = (keep * total)[first]
        _into_slots(s, s["d_state"], d_final)
        out["d_state"] = s["d_state"]
    return out


def _plain_beam(s):
    case = s["case"]
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    # in 64 bits: which of two continuations is the better one is a matter of the last bits
    z = (s["logits"].float() * case["scale"]).double()
    peak = z.amax(1, keepdim=True)
    scores = z - peak
    scores -= scores.exp().sum(1, keepdim=True).log()
    scores += s["scores"].double().view(-1, 1)
    scores = scores.view(batch, beams, vocab)
    if s["ended"] is not None:
        scores.masked_fill_(s["ended"][:, :, None], -math.inf)
        scores[:, :, 0] = torch.where(s["ended"], s["scores"].double(), scores[:, :, 0])
    best, index = torch.sort(scores.view(batch, -1), dim=1, descending=True, stable=True)
    best, index = best[:, :beams], index[:, :beams]
    none = best == -math.inf
    parents = torch.where(none, -1, index // vocab)
    out = {"scores": best.float(), "parents": parents.to(torch.int32), "tokens": torch.where(none, -1, index % vocab).to(torch.int32)}
    places = torch.arange(beams, device="cuda")
    rows = (torch.arange(batch, device="cuda")[:, None] * beams + torch.where(none, places, parents)).view(-1)
    for t in s["states"]:
        t.copy_(t[rows])
    return dict(out, states=s["states"])


PLAIN = {"embedding": _plain_embedding, "embedding_backward": _plain_embedding_backward, "layer_norm": _plain_layer_norm,
         "layer_norm_backward": _plain_layer_norm_backward, "scan": _plain_scan, "scan_step": _plain_scan, "scan_backward": _plain_scan_backward,
         "beam": _plain_beam}


# ---------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return PLAIN[kind](s)
    from pixienn_amd import ops
    if kind == "embedding":
        ops.embedding_forward(s["table"], s["tokens"], s["y"], scale=case["scale"])
        return {"y": s["y"]}
    if kind == "embedding_backward":
        ops.embedding_backward(s["dy"], s["tokens"], s["d"], scale=case["scale"], accumulate=case["accumulate"])
        return {"d": s["d"]}
    if kind == "layer_norm":
        ops.layer_norm_forward(s["x"], s["y"], s["weight"], bias=s["bias"], residual=s.get("residual"), sum=s.get("sum"), mean=s["mean"],
                               rstd=s["rstd"], eps=EPS)
        return {k: s[k] for k in ("sum", "y", "mean", "rstd") if k in s}
    if kind == "layer_norm_backward":
        ops.layer_norm_backward(s["dy"], s["h"], s["weight"], s["mean"], s["rstd"], s["dx"], s["dw"], db=s["db"], dsum=s["dsum"])
        return {k: s[k] for k in ("dx", "dw", "db") if s[k] is not None}
    if kind == "scan":
        ops.gated_scan_forward(s["x"], s["update"], s["y"], gate=s["gate"], starts=s.get("starts"), sequences=case["sequences"],
                               state=s.get("state"), final=s.get("final"), slots=s.get("slots"), saved=s.get("saved"))
        return {k: s[k] for k in ("y", "final") if k in s}
    if kind == "scan_step":
        ops.gated_scan_step(s["x"], s["update"], s["y"], s["state"], gate=s["gate"], slots=s["slots"])
        return {"y": s["y"], "final": s["state"]}
    if kind == "scan_backward":
        ops.gated_scan_backward(s["dy"], s["x"], s["update"], s["saved"], s["dx"], s["dupdate"], gate=s["gate"], dgate=s["dgate"],
                                starts=s.get("starts"), sequences=case["sequences"], state=s.get("state"), d_final=s.get("d_final"),
                                d_state=s.get("d_state"), slots=s.get("slots"))
        return {k: s[k] for k in ("dx", "dupdate", "dgate", "d_state") if s.get(k) is not None}
    ops.beam_select(s["logits"], s["scores"], s["best"], s["parents"], s["tokens"], ended=s["ended"], end_token=0, scale=case["scale"])
    ops.beam_reorder(s["states"], s["parents"])
    return {"scores": s["best"], "parents": s["parents"], "tokens": s["tokens"], "states": s["states"]}


def work(case):
    kind = case["kind"]
    size = 4 if case["type"] == "f32" else 2
    if kind.startswith("embedding"):
        n = case["rows"] * case["width"]
        if kind == "embedding":
            return {"bytes": 2 * n * size + 8 * case["rows"], "flops": n}
        out = size if case["out"] == "same" else 4
        # a row of the gradient to which nothing is added is not touched
        d = 2 * min(case["rows"], case["vocab"]) * case["width"] * out if case["accumulate"] else case["vocab"] * case["width"] * out
        return {"bytes": n * size + d + 4 * case["rows"], "flops": 2 * n}
    if kind == "layer_norm":
        n = case["rows"] * case["width"]
        return {"bytes": n * size * (4 if case["residual"] else 2) + 8 * case["rows"] + 2 * size * case["width"], "flops": 8.0 * n}
    if kind == "layer_norm_backward":
        n = case["rows"] * case["width"]
        return {"bytes": n * size * (4 if case["residual"] else 3) + 8 * case["rows"] + (size + 8) * case["width"], "flops": 13.0 * n}
    if kind.startswith("scan"):
        n = case["tokens"] * case["width"]
        states = 8 * case["sequences"] * case["width"] if case["ragged"] or kind == "scan_step" else 0
        if kind == "scan_backward":
            return {"bytes": n * size * (7 if case["gate"] else 5) + states, "flops": (40.0 if case["gate"] else 25.0) * n}
        return {"bytes": n * size * (4 if case["gate"] else 3) + states, "flops": (20.0 if case["gate"] else 10.0) * n}
    rows = case["batch"] * case["beams"]
    return {"bytes": rows * (case["vocab"] * size + 17 + 8 * (case["layers"] * case["width"] + case["history"])),
            "flops": 5.0 * rows * case["vocab"]}


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _exact_scan(s):
    case = s["case"]
    kind = case["kind"]
    n, width, lengths = case["tokens"], case["width"], s["lengths"]
    if kind == "scan_backward" and (max(lengths) if not case["ragged"] else n) > 40000:
        return None
    backward = kind == "scan_backward"
    with torch.set_grad_enabled(backward):
        leaves = {k: s[k][:n].double().requires_grad_(backward) for k in ("x", "update", "gate") if s[k] is not None}
        states = None
        if s.get("state") is not None:
            states = leaves["state"] = s["state"].double().requires_grad_(backward)
        slots = s["slots"].tolist() if states is not None else []
        z = 1.0 / (1.0 + torch.exp(-leaves["update"]))
        zx = z * leaves["x"]
        keep = 1.0 / (1.0 + torch.exp(leaves["update"]))
        finals = {}
        if case["ragged"] or states is not None:
            rows, at = [], 0
            for i, length in enumerate(lengths):
                h = states[slots[i]] if slots[i] >= 0 else torch.zeros(width, device="cuda", dtype=torch.float64)
                for t in range(at, at + length):
                    h = torch.addcmul(zx[t], keep[t], h)
                    rows.append(h)
                at += length
                if slots[i] >= 0:
                    finals[slots[i]] = h
            h = torch.stack(rows)
        else:
            keep, zx = (t.view(len(lengths), lengths[0], width) for t in (keep, zx))
            one, rows = torch.zeros(len(lengths), width, device="cuda", dtype=torch.float64), []
            for k, v in zip(keep.unbind(1), zx.unbind(1)):
                one = torch.addcmul(v, k, one)
                rows.append(one)
            h = torch.stack(rows, 1).view(n, width)
        y = h if s["gate"] is None else torch.nn.functional.silu(leaves["gate"]) * h
        if not backward:
            rest = torch.zeros(len(s["y"]) - n, width, device="cuda", dtype=torch.float64)
            out = {"y": torch.cat([y, rest])}
            if states is not None:
                final = states.clone() if kind == "scan_step" else torch.zeros_like(states)
                for slot, value in finals.items():
                    final[slot] = value
                out["final"] = final
            return out
        loss = (y * s["dy"][:n].double()).sum()
        for slot, value in finals.items():
            loss = loss + (value * s["d_final"][slot].double()).sum()
        grads = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
    out = {}
    for name, key in (("dx", "x"), ("dupdate", "update"), ("dgate", "gate")):
        if key in grads:
            out[name] = torch.cat([grads[key], torch.zeros(len(s[name]) - n, width, device="cuda", dtype=torch.float64)])
    if states is not None:
        out["d_state"] = grads["state"]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "embedding":
        tokens = s["tokens"].tolist()
        y = torch.zeros(case["rows"], case["width"], device="cuda", dtype=torch.float64)
        places = [i for i, t in enumerate(tokens) if 0 <= t < case["vocab"]]
        y[places] = s["table"].double()[[tokens[i] for i in places]] * case["scale"]
        return {"y": y}
    if kind == "embedding_backward":
        table = torch.zeros(case["vocab"], case["width"], device="cuda", dtype=torch.float64)
        places = s["tokens"] >= 0
        table.index_put_((s["tokens"][places].long(),), s["dy"][places].double(), accumulate=True)
        table *= case["scale"]
        return {"d": table + s["d"].double() if case["accumulate"] else table}
    if kind == "layer_norm":
        h = s["x"].double()
        out = {}
        if case["residual"]:
            h = out["sum"] = h + s["residual"].double()
            h = h.to(s["x"].dtype).double()            # the norm is that of the sum as it is kept
        deviation, mean = torch.std_mean(h, dim=1, correction=0)
        out.update(mean=mean, rstd=1.0 / torch.sqrt(deviation ** 2 + EPS))
        y = s["weight"].double() * ((h - mean[:, None]) * out["rstd"][:, None])
        return dict(out, y=y if s["bias"] is None else y + s["bias"].double())
    if kind == "layer_norm_backward":
        with torch.enable_grad():
            h, w = s["h"].double().requires_grad_(), s["weight"].double().requires_grad_()
            b = torch.zeros(case["width"], device="cuda", dtype=torch.float64).requires_grad_()
            centre = h - h.sum(1, keepdim=True) / case["width"]
            y = centre / torch.sqrt((centre * centre).sum(1, keepdim=True) / case["width"] + EPS) * w + b
            dx, dw, db = torch.autograd.grad(y, (h, w, b), s["dy"].double())
        out = {"dx": dx if s["dsum"] is None else dx + s["dsum"].double(), "dw": dw}
        return dict(out, db=db) if case["bias"] else out
    if kind.startswith("scan"):
        return _exact_scan(s)
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    best = torch.empty(batch, beams, device="cuda", dtype=torch.float64)
    order = []
    for item in range(batch):
        logs = torch.log_softmax(s["logits"][item * beams:(item + 1) * beams].double() * case["scale"], 1) + s["scores"][item].double()[:, None]
        ended = torch.nonzero(s["ended"][item])[:, 0].tolist() if s["ended"] is not None else []
        for k in ended:
            logs[k] = -math.inf
            logs[k, 0] = s["scores"][item, k].double()
        best[item], index = logs.flatten().topk(beams)
        order.append(index // vocab + item * beams)
    # equal scores may come in either order here: then the states, which follow them, have no one value
    tied = bool((best.diff(dim=1).abs() < 1e-6).any())
    rows = torch.cat(order)
    return {"scores": best, "parents": None, "tokens": None,
            "states": [None if tied or not t.dtype.is_floating_point else t.double()[rows] for t in s["states"]]}

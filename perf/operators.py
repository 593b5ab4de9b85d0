"""Cases of the sequence operators: gated scan over time, gated residual norm, token scores, distillation from a teacher's
top tokens.  ``run`` computes a case in plain 32-bit torch operations, or (``own``) through the package's own calls.

What the operators compute (all sums, states and statistics in 32 bits, outputs rounded once):

* ``GatedScanFunction.apply(x, gate, state, lengths) -> y, last`` and ``GatedScanFunction.step(x, gate, state, slots) -> y``:
  ``h_t = s(gate_t) h_{t-1} + (1 - s(gate_t)) x_t`` per channel, ``s`` the logistic function; ``y_t = h_t``, ``last`` the
  state after the sequence's own length, zeros behind it.  ``step`` advances the rows ``slots`` of a pool in place.
* ``ResidualNormFunction.apply(x, block, gate, scale, post_weight, pre_weight, eps) -> stream, normed``:
  ``stream = x + scale s(gate) rms(block) post_weight``, ``normed = rms(stream) pre_weight``.
* ``TokenScoresFunction.apply(logits, tokens, top, temperature, ignore_index) -> logprob, entropy, top_logprobs, top_tokens``.
* ``DistillTopkFunction.apply(logits, teacher_logprobs, teacher_tokens, temperature, tail) -> loss`` per row:
  ``temperature^2 KL(teacher || student)`` over the teacher's top tokens, all others as one more outcome (``tail``), or
  over the top tokens renormalised.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MOST_CHANNEL_STEPS = 2 * 16384 * 2048          # elements of the largest sequence tensors
MOST_LOGITS = 2047 * 100003                    # elements of the largest logits


def listed():
    return [
        # one new clip feature of 16 live streams through a layer of the sequence head: all latency
        {"name": "step 16x512 f32", "op": "step", "type": "f32", "rows": 16, "channels": 512, "pool": 24},
        # a batch of stored videos of different lengths, features of an earlier part carried in
        {"name": "scan 24x777x1024 bf16 ragged", "op": "scan", "type": "bf16", "batch": 24, "steps": 777, "channels": 1024,
         "ragged": True, "train": False},
        # training on short clips' features, width that no vector divides
        {"name": "scan train 5x131x390 f32", "op": "scan", "type": "f32", "batch": 5, "steps": 131, "channels": 390,
         "ragged": True, "train": True},
        # training on hours of video or token sequences: few rows, a long axis
        {"name": "scan train 2x16384x2048 bf16", "op": "scan", "type": "bf16", "batch": 2, "steps": 16384, "channels": 2048,
         "ragged": False, "train": True},
        # the same 16 live streams between two blocks
        {"name": "norm 16x512 bf16", "op": "norm", "type": "bf16", "rows": 16, "channels": 512, "gate": True, "train": False,
         "weights": "f32"},
        # a small training batch in full precision, odd row count
        {"name": "norm train 4099x1000 f32", "op": "norm", "type": "f32", "rows": 4099, "channels": 1000, "gate": True,
         "train": True, "weights": "f32"},
        # the long training batch between two blocks
        {"name": "norm train 32768x2048 bf16", "op": "norm", "type": "bf16", "rows": 32768, "channels": 2048, "gate": True,
         "train": True, "weights": "f32"},
        # answers for 16 clips over the 400 classes of the video network: label, confidence, five alternatives
        {"name": "scores 16x400 f32 top5", "op": "scores", "type": "f32", "rows": 16, "vocab": 400, "top": 5,
         "temperature": 1.0, "masked": False, "train": False},
        # a decoding step over a large vocabulary, some tokens forbidden
        {"name": "scores 64x131072 bf16 top20", "op": "scores", "type": "bf16", "rows": 64, "vocab": 131072, "top": 20,
         "temperature": 0.8, "masked": True, "train": False},
        # policy-gradient or likelihood training with an entropy term
        {"name": "scores train 4096x32768 bf16", "op": "scores", "type": "bf16", "rows": 4096, "vocab": 32768, "top": 0,
         "temperature": 1.0, "masked": False, "train": True},
        # the video network's classifier trained from a larger one's ten best classes
        {"name": "distill train 32x400 f32 k10", "op": "distill", "type": "f32", "rows": 32, "vocab": 400, "k": 10,
         "temperature": 2.0, "tail": True, "train": True},
        # a large vocabulary of odd size, rows that no vector load starts on
        {"name": "distill train 2047x100003 bf16", "op": "distill", "type": "bf16", "rows": 2047, "vocab": 100003, "k": 64,
         "temperature": 1.0, "tail": True, "train": True},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    def width(lo, hi):
        n = log(lo, hi)                        # half of the widths are ordinary (multiples of 64), the others any number
        return max(lo, n // 64 * 64) if rng.random() < 0.5 else n

    op = rng.choice(["scan", "scan", "step", "norm", "norm", "scores", "scores", "distill", "distill"])
    c = {"op": op, "type": rng.choice(["f32", "bf16", "bf16", "f16"])}
    most = 2 if c["type"] == "f32" else 1
    if op == "step":
        rows = log(1, 2048)
        c.update(rows=rows, channels=width(64, 8192), pool=rows + rng.randrange(0, 16))
    elif op == "scan":
        channels = width(64, 4096)
        steps = log(1, 16384)
        c.update(batch=max(1, min(log(1, 64), MOST_CHANNEL_STEPS // most // (steps * channels))), steps=steps,
                 channels=channels, ragged=rng.random() < 0.5, train=rng.random() < 0.5)
    elif op == "norm":
        channels = width(64, 8192)
        c.update(rows=log(1, min(65536, MOST_CHANNEL_STEPS // most // channels)), channels=channels,
                 gate=rng.random() < 0.7, train=rng.random() < 0.5,
                 weights=rng.choice(["f32", c["type"]]))
    else:
        vocab = width(100, 200000)
        rows = log(1, min(16384, MOST_LOGITS // most // vocab))
        c.update(rows=rows, vocab=vocab, temperature=rng.choice([1.0, 1.0, 0.7, 2.0]), train=rng.random() < 0.5)
        if op == "scores":
            c.update(top=0 if c["train"] else rng.choice([0, 1, 5, 20, 50]), masked=rng.random() < 0.3)
        else:
            c.update(k=rng.choice([1, 8, 32, 64, 100]), tail=rng.random() < 0.6)
    return c


class State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    op = case["op"]

    def normal(*shape, std=1.0, mean=0.0, dtype=t):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")

    s = State(case=case)
    if op == "step":
        n, c = case["rows"], case["channels"]
        both = normal(n, 2 * c)                # value and gate as one projection of the features gives them
        s.x, s.gate = both[:, :c], both[:, c:].add_(2.0)
        s.state = normal(case["pool"], c, dtype=torch.float32)
        s.slots = torch.randperm(case["pool"], generator=g, device="cuda")[:n]
    elif op == "scan":
        b, n, c = case["batch"], case["steps"], case["channels"]
        both = normal(b, n, 2 * c)
        both[..., c:] += 2.0                   # states that last some ten to hundreds of steps
        s.x, s.gate = both[..., :c], both[..., c:]
        s.state = normal(b, c, dtype=torch.float32)
        s.lengths = whole(0, n + 1, b) if case["ragged"] else None
        if case["train"]:
            s.dy = normal(b, n, c)
            s.dlast = normal(b, c, dtype=torch.float32)
            s.x, s.gate, s.state = (v.requires_grad_() for v in (s.x, s.gate, s.state))
    elif op == "norm":
        n, c = case["rows"], case["channels"]
        w = TYPES[case["weights"]]
        s.x, s.block = normal(n, c, std=2.0), normal(n, c, std=0.5)
        s.gate = normal(n, c) if case["gate"] else None
        s.scale = normal(c, std=0.1, mean=0.5, dtype=w)
        s.post, s.pre = normal(c, std=0.1, mean=1.0, dtype=w), normal(c, std=0.1, mean=1.0, dtype=w)
        if case["train"]:
            s.dstream, s.dnormed = normal(n, c), normal(n, c)
            for v in (s.x, s.block, s.gate, s.scale, s.post, s.pre):
                if v is not None:
                    v.requires_grad_()
    elif op == "scores":
        n, v = case["rows"], case["vocab"]
        s.logits = normal(n, v, std=2.5)
        s.tokens = whole(0, v, n)
        s.tokens[whole(0, 16, n) == 0] = -100  # positions of a prompt that are not scored
        if case["masked"]:
            s.logits[:, whole(0, v, max(1, v // 8))] = -math.inf
        if case["train"]:
            s.dlogprob, s.dentropy = normal(n, dtype=torch.float32), normal(n, std=0.01, dtype=torch.float32)
            s.logits.requires_grad_()
    else:
        n, v = case["rows"], case["vocab"]
        k = min(case["k"], v)
        teacher = normal(n, v, std=3.0, dtype=torch.float32)
        s.logits = (0.7 * teacher + normal(n, v, dtype=torch.float32)).to(t)
        best, s.teacher_tokens = teacher.topk(k)
        s.teacher_logprobs = (best - teacher.logsumexp(-1, keepdim=True)).contiguous()
        if case["train"]:
            s.dloss = torch.full((n,), 1.0 / n, device="cuda")
            s.logits.requires_grad_()
    return s


# ---- the operators in plain operations ------------------------------------------------------------------------------------

def _scan(a, b):
    """Inclusive scan of h_t = a_t h_{t-1} + b_t along dim 1, by doubling."""
    d = 1
    while d < a.size(1):
        b = torch.cat((b[:, :d], torch.addcmul(b[:, d:], a[:, d:], b[:, :-d])), 1)
        a = torch.cat((a[:, :d], a[:, d:] * a[:, :-d]), 1)
        d *= 2
    return b


def _plain_scan(s):
    t = s.x.dtype
    x, a, keep = s.x.float(), torch.sigmoid(s.gate.float()), torch.sigmoid(-s.gate.float())
    n = x.size(1)
    inside = None
    if s.lengths is not None:
        inside = torch.arange(n, device="cuda")[None, :, None] < s.lengths[:, None, None]
        a, b = torch.where(inside, a, 1.0), torch.where(inside, keep * x, 0.0)
    else:
        b = keep * x
    b[:, 0] += a[:, 0] * s.state
    h = _scan(a, b)
    y = (h if inside is None else torch.where(inside, h, 0.0)).to(t)
    last = h[:, -1].clone()
    if not s.case["train"]:
        return y, last
    dy = s.dy.float()
    if inside is not None:
        dy = torch.where(inside, dy, 0.0)
    u = a * dy                                 # gradient that a step passes on: p_t = a_t p_{t+1} + a_t dy_t
    u[:, -1] += a[:, -1] * s.dlast
    p = _scan(a.flip(1), u.flip(1)).flip(1)
    dh = dy + torch.cat((p[:, 1:], s.dlast[:, None]), 1)
    before = torch.cat((s.state[:, None], h[:, :-1]), 1)
    dx, dgate = dh * keep, dh * (before - x) * a * keep
    if inside is not None:
        dx, dgate = torch.where(inside, dx, 0.0), torch.where(inside, dgate, 0.0)
    return y, last, dx.to(t), dgate.to(t), p[:, 0].clone()


def _plain_step(s):
    a, keep = torch.sigmoid(s.gate.float()), torch.sigmoid(-s.gate.float())
    h = a * s.state[s.slots] + keep * s.x.float()
    s.state[s.slots] = h
    return h.to(s.x.dtype), s.state


def _plain_norm(s):
    t, eps = s.x.dtype, 1e-6
    x, y = s.x.float(), s.block.float()
    scale, post, pre = s.scale.float(), s.post.float(), s.pre.float()
    g = torch.sigmoid(s.gate.float()) if s.gate is not None else 1.0
    r = torch.rsqrt((y * y).mean(-1, keepdim=True) + eps)
    yn = y * r
    stream = x + scale * post * g * yn
    q = torch.rsqrt((stream * stream).mean(-1, keepdim=True) + eps)
    sn = stream * q
    out = stream.to(t), (sn * pre).to(t)
    if not s.case["train"]:
        return out
    dn = s.dnormed.float()
    dpre = (dn * sn).sum(0)
    dsn = dn * pre
    ds = s.dstream.float() + q * (dsn - sn * (dsn * sn).mean(-1, keepdim=True))
    z = (ds * g * yn).sum(0)
    dyn = ds * scale * post * g
    dy = r * (dyn - yn * (dyn * yn).mean(-1, keepdim=True))
    dgate = (dyn * yn * (1 - g)).to(t) if s.gate is not None else None
    w = s.scale.dtype
    return out + (ds.to(t), dy.to(t), dgate, (z * post).to(w), (z * scale).to(w), dpre.to(w))


def _log_softmax_parts(logits, temperature):
    z = logits.float() / temperature
    m = z.amax(-1, keepdim=True)
    d = z - torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    return d, e, total, torch.log(total)


def _plain_scores(s):
    c = s.case
    d, e, total, lse = _log_softmax_parts(s.logits, c["temperature"])
    scored = s.tokens != -100
    token = torch.where(scored, s.tokens, 0)[:, None]
    logprob = torch.where(scored, (d.gather(1, token) - lse)[:, 0], 0.0)
    entropy = (lse - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / total)[:, 0]
    if c["train"]:
        p = e / total
        log_p = torch.where(e > 0, d - lse, 0.0)
        dz = -p * (s.dentropy[:, None] * (log_p + entropy[:, None]))
        gl = torch.where(scored, s.dlogprob, 0.0)[:, None]
        dz -= p * gl
        dz.scatter_add_(1, token, gl)
        return logprob, entropy, (dz / c["temperature"]).to(s.logits.dtype)
    if c["top"] == 0:
        return logprob, entropy
    v = s.logits.size(1)
    bits = (s.logits.float() + 0.0).view(torch.int32).long()
    rank = torch.where(bits < 0, -(bits & 0x7fffffff), bits)           # the order of the values, ties to the lowest index
    key = rank * 2 ** 20 + (2 ** 20 - 1 - torch.arange(v, device="cuda"))
    top_tokens = 2 ** 20 - 1 - (key.topk(min(c["top"], v), dim=-1).values & (2 ** 20 - 1))
    return logprob, entropy, d.gather(1, top_tokens) - lse, top_tokens


def _plain_distill(s):
    c = s.case
    temperature, tokens = c["temperature"], s.teacher_tokens
    d, e, total, lse = _log_softmax_parts(s.logits, temperature)
    lq = s.teacher_logprobs.float()
    if not c["tail"]:
        lq = lq - lq.logsumexp(-1, keepdim=True)
    q = torch.exp(lq)
    log_p = d.gather(1, tokens) - lse
    loss = torch.where(q > 0, q * (lq - log_p), 0.0).sum(-1)
    rest = None
    if c["tail"]:
        rest = torch.ones_like(e, dtype=torch.bool).scatter_(1, tokens, False)
        e_rest = torch.where(rest, e, 0.0)
        total_rest = e_rest.sum(-1, keepdim=True)
        q_rest = torch.where(total_rest > 0, (1 - q.sum(-1, keepdim=True)).clamp(min=0), 0.0)
        log_p_rest = torch.log(total_rest) - lse
        loss = loss + torch.where(q_rest > 0, q_rest * (torch.log(q_rest) - log_p_rest), 0.0)[:, 0]
    loss = loss * temperature ** 2
    if not c["train"]:
        return loss
    mass = q.sum(-1, keepdim=True)
    if c["tail"]:
        mass = mass + q_rest
    dz = e / total * mass
    if c["tail"]:
        dz -= torch.where(total_rest > 0, q_rest / total_rest * e_rest, 0.0)
    dz.scatter_add_(1, tokens, -q)
    return loss, (dz * (temperature * s.dloss[:, None])).to(s.logits.dtype)


# ---- one pass -------------------------------------------------------------------------------------------------------------

def run(state):
    s = state
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"scan": _plain_scan, "step": _plain_step, "norm": _plain_norm, "scores": _plain_scores,
                "distill": _plain_distill}[s.case["op"]](s)


def _run_own(s):
    import deform_conv3d_pytorch_op_b200 as dcn
    c, op = s.case, s.case["op"]
    grad = torch.autograd.grad
    if op == "step":
        return dcn.GatedScanFunction.step(s.x, s.gate, s.state, s.slots), s.state
    if op == "scan":
        y, last = dcn.GatedScanFunction.apply(s.x, s.gate, s.state, s.lengths)
        if not c["train"]:
            return y, last
        return (y.detach(), last.detach()) + grad((y, last), (s.x, s.gate, s.state), (s.dy, s.dlast))
    if op == "norm":
        out = dcn.ResidualNormFunction.apply(s.x, s.block, s.gate, s.scale, s.post, s.pre, 1e-6)
        if not c["train"]:
            return out
        asked = [v for v in (s.x, s.block, s.gate, s.scale, s.post, s.pre) if v is not None]
        got = grad(out, asked, (s.dstream, s.dnormed))
        if s.gate is None:
            got = got[:2] + (None,) + got[2:]
        return (out[0].detach(), out[1].detach()) + got
    if op == "scores":
        out = dcn.TokenScoresFunction.apply(s.logits, s.tokens, c["top"], c["temperature"], -100)
        if not c["train"]:
            return out if c["top"] else out[:2]
        return (out[0].detach(), out[1].detach()) + grad(out[:2], (s.logits,), (s.dlogprob, s.dentropy))
    loss = dcn.DistillTopkFunction.apply(s.logits, s.teacher_logprobs, s.teacher_tokens, c["temperature"], c["tail"])
    if not c["train"]:
        return loss
    return (loss.detach(),) + grad((loss,), (s.logits,), (s.dloss,))


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

def work(case):
    op, e = case["op"], SIZE[case["type"]]
    if op == "step":
        n = case["rows"] * case["channels"]
        return {"bytes": n * (3 * e + 8) + case["rows"] * 8, "flops": 10 * n}
    if op == "scan":
        n, rows = case["batch"] * case["steps"] * case["channels"], case["batch"] * case["channels"] * 4
        if case["train"]:                      # x, gate, dy in; y, dx, dgate out; state and its gradients
            return {"bytes": n * 6 * e + 4 * rows, "flops": 30 * n}
        return {"bytes": n * 3 * e + 2 * rows, "flops": 10 * n}
    if op == "norm":
        n, c, w = case["rows"] * case["channels"], case["channels"], SIZE[case["weights"]]
        k = 1 if case["gate"] else 0
        if case["train"]:                      # x, block, gate, dstream, dnormed in; stream, normed, dx, dblock, dgate out
            return {"bytes": n * e * (8 + 2 * k) + 6 * c * w, "flops": 45 * n}
        return {"bytes": n * e * (4 + k) + 3 * c * w, "flops": 15 * n}
    n = case["rows"] * case["vocab"]
    more = case["rows"] * (8 + 8 + 12 * case["top"] if op == "scores" else 4 + 12 * case["k"])
    return {"bytes": n * e * (2 if case["train"] else 1) + more, "flops": n * (16 if case["train"] else 7)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    wide = State(case=case)
    for name, v in vars(s).items():
        if name != "case":
            wide.__dict__[name] = v.detach().double() if v is not None and v.is_floating_point() else v
    return {"scan": _exact_scan, "step": _exact_step, "norm": _exact_norm, "scores": _exact_scores,
            "distill": _exact_distill}[case["op"]](case, wide)


def _exact_step(case, s):
    f = 1 / (1 + torch.exp(-s.gate))
    new = s.state.index_select(0, s.slots).mul(f).add((1 - f) * s.x)
    return new, s.state.index_copy(0, s.slots, new)


def _exact_scan(case, s):
    b, n, c = s.x.shape
    lengths = s.lengths if s.lengths is not None else torch.full((b,), n, device="cuda")
    f = 1 / (1 + torch.exp(-s.gate))
    states, h = torch.empty(n + 1, b, c, dtype=torch.float64, device="cuda"), s.state
    states[0] = h
    live = (torch.arange(n, device="cuda")[:, None] < lengths)[..., None]
    for t in range(n):
        h = torch.where(live[t], torch.lerp(s.x[:, t], h, f[:, t]), h)
        states[t + 1] = h
    y = (states[1:] * live).transpose(0, 1)
    if not case["train"]:
        return y, h
    d, dx, df = s.dlast, torch.zeros_like(s.x), torch.zeros_like(s.x)
    for t in range(n - 1, -1, -1):
        here = d + s.dy[:, t]
        dx[:, t] = here * (1 - f[:, t]) * live[t]
        df[:, t] = here * (states[t] - s.x[:, t]) * live[t]
        d = torch.where(live[t], here * f[:, t], d)
    return y, h, dx, df.mul_(f).mul_(1 - f), d


def _exact_norm(case, s):
    ins = [s.x, s.block, s.gate, s.scale, s.post, s.pre]
    with torch.enable_grad():
        for v in ins:
            if v is not None and case["train"]:
                v.requires_grad_()
        n = case["channels"]
        body = s.block / torch.sqrt(s.block.square().sum(1, keepdim=True) / n + 1e-6) * s.post * s.scale
        if s.gate is not None:
            body = body / (1 + torch.exp(-s.gate))
        stream = s.x + body
        normed = stream / torch.sqrt(stream.square().sum(1, keepdim=True) / n + 1e-6) * s.pre
        if not case["train"]:
            return stream, normed
        got = list(torch.autograd.grad((stream, normed), [v for v in ins if v is not None], (s.dstream, s.dnormed)))
    if s.gate is None:
        got.insert(2, None)
    return [stream.detach(), normed.detach()] + got


def _exact_scores(case, s):
    with torch.enable_grad():
        logits = s.logits.requires_grad_(case["train"])
        log_p = logits / case["temperature"]
        log_p = log_p - torch.logsumexp(log_p, 1, keepdim=True)
        picked = log_p[torch.arange(case["rows"], device="cuda"), s.tokens.clamp(min=0)]
        logprob = picked.masked_fill(s.tokens == -100, 0.0)
        entropy = -(torch.exp(log_p) * log_p.masked_fill(log_p == -math.inf, 0.0)).sum(1)
        if case["train"]:
            if case["masked"]:                 # the gradient past forbidden tokens: of the others' softmax alone
                allowed = torch.isfinite(logits[0])
                inner = State(**{**vars(s), "logits": s.logits.detach()[:, allowed]})
                renumber = torch.cumsum(allowed, 0) - 1
                gone = (s.tokens >= 0) & ~allowed[s.tokens.clamp(min=0)]
                inner.tokens = torch.where((s.tokens >= 0) & ~gone, renumber[s.tokens.clamp(min=0)], -100)
                _, _, part = _exact_scores({**case, "masked": False}, inner)
                probs = torch.softmax(inner.logits.detach() / case["temperature"], 1)
                part = part - probs * (s.dlogprob * gone)[:, None] / case["temperature"]
                full = torch.zeros_like(logits)
                full[:, allowed] = part
                full[torch.arange(case["rows"], device="cuda"), s.tokens.clamp(min=0)] += s.dlogprob * gone / case["temperature"]
                return logprob.detach(), entropy.detach(), full
            return (logprob.detach(), entropy.detach()) + torch.autograd.grad((logprob, entropy), logits, (s.dlogprob, s.dentropy))
    if case["top"] == 0:
        return logprob, entropy
    return logprob, entropy, log_p.sort(1, descending=True).values[:, :case["top"]].contiguous(), None


def _exact_distill(case, s):
    with torch.enable_grad():
        logits = s.logits.requires_grad_(case["train"])
        log_p = torch.log_softmax(logits / case["temperature"], 1)
        lq, student = s.teacher_logprobs, log_p.gather(1, s.teacher_tokens)
        if case["tail"]:
            rest = 1 - torch.exp(lq).sum(1, keepdim=True)
            others = log_p.scatter(1, s.teacher_tokens, -math.inf)
            if case["k"] < case["vocab"]:
                lq = torch.cat((lq, torch.log(rest.clamp(min=1e-300))), 1)
                student = torch.cat((student, torch.logsumexp(others, 1, keepdim=True)), 1)
        else:
            lq = torch.log_softmax(lq, 1)
        loss = (torch.exp(lq) * (lq - student)).sum(1) * case["temperature"] ** 2
        if not case["train"]:
            return loss
        return (loss.detach(),) + torch.autograd.grad(loss, logits, s.dloss)

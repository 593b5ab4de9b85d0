"""Cases of decayed linear attention over a sequence, of group norm with an activation over channels-last features, and of drawing
tokens (or classes) from logits.  ``run`` computes a case in plain torch operations, or (``own``) through the package's own calls.

What the operators compute (sums, states and statistics in 32 bits or more, outputs rounded once):

* ``DecayAttentionFunction.apply(q, k, v, log_decay, state, lengths, scale) -> out, last``:
  ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T``, ``out_t = scale S_t^T q_t`` for each head; ``last`` is the state after the sequence's
  own length, zeros behind it.  Several heads may share a key and a value.  ``step`` advances the rows ``slots`` of a pool.
* ``GroupNormActFunction.apply(x, groups, weight, bias, residual, activation, eps) -> y``:
  ``y = act((x - mean) / sqrt(var + eps) weight + bias + residual)`` with the statistics of a sample's group of channels.
* ``TokenSampleFunction.apply(logits, uniform, temperature, top_k, top_p, min_p) -> tokens, logprob``: weights
  ``w = floor(2^40 exp((logits - max) / temperature))``; kept are the top_k largest logits (equal ones by index), of these the
  fewest largest that have top_p of their weight, of these the ones that have min_p of the largest weight.  The token is
  the first, by index, up to which the kept weights are more than ``floor(uniform * sum)``; its logprob is log(w / sum).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MOST_HEAD_STEPS = 2 * 16384 * 16               # rows of q of the largest attention, times heads
MOST_FEATURES = 8 * 50176 * 64                 # elements of the largest features
MOST_LOGITS = 64 * 131072


def listed():
    return [
        # the next clip (or token) of 16 live streams: all latency
        {"name": "step 16x8x64 f32", "op": "step", "type": "f32", "rows": 16, "heads": 8, "kv_heads": 8, "dk": 64, "dv": 64, "pool": 24},
        # the same for a server's batch, heads that share keys and values: the states are read and written
        {"name": "step 256x16x128 bf16 shared", "op": "step", "type": "bf16", "rows": 256, "heads": 16, "kv_heads": 4, "dk": 128,
         "dv": 128, "pool": 300},
        # a batch of stored videos of different lengths, features of an earlier part carried in
        {"name": "attend 24x777x8x64 bf16 ragged", "op": "attend", "type": "bf16", "batch": 24, "steps": 777, "heads": 8, "kv_heads": 8,
         "dk": 64, "dv": 64, "ragged": True, "train": False},
        # training in full precision on short sequences, widths that no tile divides
        {"name": "attend train 5x331x6x(40,72) f32 ragged", "op": "attend", "type": "f32", "batch": 5, "steps": 331, "heads": 6,
         "kv_heads": 3, "dk": 40, "dv": 72, "ragged": True, "train": True},
        # training on hours of video or token sequences
        {"name": "attend train 2x16384x16x128 bf16", "op": "attend", "type": "bf16", "batch": 2, "steps": 16384, "heads": 16,
         "kv_heads": 16, "dk": 128, "dv": 128, "ragged": False, "train": True},
        # the heads' outputs of 16 live streams, normalised head by head
        {"name": "group norm 16x1x512 by 8 f32", "op": "norm", "type": "f32", "samples": 16, "positions": 1, "channels": 512, "groups": 8,
         "act": "silu", "residual": False, "train": False, "weights": "f32"},
        # a late stage of the video network on few clips, as it trains: norm, shortcut, activation; odd position count
        {"name": "group norm train 6x1183x256 by 32 f32", "op": "norm", "type": "f32", "samples": 6, "positions": 1183, "channels": 256,
         "groups": 32, "act": "relu", "residual": True, "train": True, "weights": "f32"},
        # the stem of the video network: 16 frames of 56 x 56 positions
        {"name": "group norm train 8x50176x64 by 32 bf16", "op": "norm", "type": "bf16", "samples": 8, "positions": 50176, "channels": 64,
         "groups": 32, "act": "relu", "residual": False, "train": True, "weights": "f32"},
        # an answer for each of 16 clips over the 400 classes of the video network
        {"name": "sample 16x400 f32", "op": "sample", "type": "f32", "rows": 16, "vocab": 400, "temperature": 1.0, "top_k": 0,
         "top_p": 1.0, "min_p": 0.0, "per_row": False, "masked": False},
        # a decoding step of a server: every request with its own settings, some tokens forbidden
        {"name": "sample 64x131072 bf16 k50 p0.9", "op": "sample", "type": "bf16", "rows": 64, "vocab": 131072, "temperature": 0.8,
         "top_k": 50, "top_p": 0.9, "min_p": 0.0, "per_row": True, "masked": True},
        # a nucleus without a count, odd vocabulary
        {"name": "sample 37x50257 f16 p0.95", "op": "sample", "type": "f16", "rows": 37, "vocab": 50257, "temperature": 1.0,
         "top_k": 0, "top_p": 0.95, "min_p": 0.02, "per_row": False, "masked": False},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["attend", "attend", "attend", "step", "norm", "norm", "norm", "sample", "sample", "sample"])
    c = {"op": op, "type": rng.choice(["f32", "bf16", "bf16", "f16"])}
    most = 2 if c["type"] == "f32" else 1
    if op in ("attend", "step"):
        heads = rng.choice([1, 2, 4, 6, 8, 12, 16])
        even = rng.random() < 0.6              # head widths: multiples of 16 mostly
        c.update(heads=heads, kv_heads=heads // rng.choice([n for n in (1, 1, 1, 2, 4) if heads % n == 0]),
                 dk=16 * rng.randint(2, 8) if even else rng.randint(8, 128), dv=16 * rng.randint(2, 8) if even else rng.randint(8, 128))
        if op == "step":
            rows = log(1, 2048 // heads)
            c.update(rows=rows, pool=rows + rng.randrange(0, 16))
        else:
            steps = log(1, 16384)
            c.update(batch=max(1, min(log(1, 64), MOST_HEAD_STEPS // most // (steps * heads))), steps=steps,
                     ragged=rng.random() < 0.5, train=rng.random() < 0.5)
    elif op == "norm":
        per = log(1, 32)                       # channels of a group
        groups = rng.choice([1, 2, 4, 8, 16, 32, 32, rng.randint(1, 32)])
        channels = per * groups
        positions = rng.choice([1, log(1, 65536), log(1, 65536)])
        samples = max(1, min(log(1, 32768 if positions == 1 else 64), MOST_FEATURES // most // 2 // (positions * channels)))
        c.update(samples=samples, positions=positions, channels=channels, groups=groups, act=rng.choice(["none", "relu", "silu", "silu"]),
                 residual=rng.random() < 0.4, train=rng.random() < 0.5, weights=rng.choice(["f32", c["type"]]))
    else:
        vocab = log(100, 131072)
        c.update(rows=log(1, min(4096, MOST_LOGITS // most // vocab)), vocab=vocab, temperature=rng.choice([0.6, 0.8, 1.0, 1.0, 1.3]),
                 top_k=rng.choice([0, 0, 1, 20, 50, 200]), top_p=rng.choice([1.0, 0.8, 0.9, 0.95]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]),
                 per_row=rng.random() < 0.5, masked=rng.random() < 0.3)
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
    if op in ("attend", "step"):
        h, kv, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
        lead = (case["rows"],) if op == "step" else (case["batch"], case["steps"])
        # q, k and v as one projection of the features gives them
        s.q, s.k, s.v = normal(*lead, h * dk + kv * (dk + dv)).split((h * dk, kv * dk, kv * dv), -1)
        s.q, s.k, s.v = s.q.unflatten(-1, (h, dk)), s.k.unflatten(-1, (kv, dk)), s.v.unflatten(-1, (kv, dv))
        # states that last some ten to some hundred steps
        s.log_decay = torch.log1p(-torch.exp2(-3.0 - torch.rand(h, generator=g, device="cuda", dtype=torch.float64) * 6)).float()
        s.scale = dk ** -0.5
        if op == "step":
            s.state = normal(case["pool"], h, dk, dv, std=2.0, dtype=torch.float32)
            s.slots = torch.randperm(case["pool"], generator=g, device="cuda")[:case["rows"]]
        else:
            s.state = normal(case["batch"], h, dk, dv, std=2.0, dtype=torch.float32)
            s.lengths = whole(0, case["steps"] + 1, case["batch"]) if case["ragged"] else None
            if case["train"]:
                s.dout = normal(*lead, h, dv)
                s.dlast = normal(case["batch"], h, dk, dv, std=0.1, dtype=torch.float32)
                s.q, s.k, s.v, s.state = (v.requires_grad_() for v in (s.q, s.k, s.v, s.state))
    elif op == "norm":
        n, p, c = case["samples"], case["positions"], case["channels"]
        w = TYPES[case["weights"]]
        s.x = (normal(n, p, c, std=1.5, dtype=torch.float32) + normal(c, dtype=torch.float32)).to(t)
        s.residual = normal(n, p, c) if case["residual"] else None
        s.weight, s.bias = normal(c, std=0.1, mean=1.0, dtype=w), normal(c, std=0.1, dtype=w)
        if case["train"]:
            s.dy = normal(n, p, c)
            s.asked = [v.requires_grad_() for v in (s.x, s.weight, s.bias, s.residual) if v is not None]
    else:
        n, v = case["rows"], case["vocab"]
        # some rows are sure of a few tokens, others of hardly any
        sharp = 2.0 + 2.5 * torch.rand(n, 1, generator=g, device="cuda")
        s.logits = (normal(n, v, dtype=torch.float32) * sharp).to(t)
        if case["masked"]:
            s.logits[:, whole(0, v, max(1, v // 8))] = -math.inf
        s.uniform = torch.rand(n, generator=g, device="cuda")
        s.temperature, s.top_k, s.top_p, s.min_p = (case[key] for key in ("temperature", "top_k", "top_p", "min_p"))
        if case["per_row"]:
            s.temperature = s.temperature * (0.75 + 0.5 * torch.rand(n, generator=g, device="cuda"))
            s.top_k = torch.where(whole(0, 4, n) == 0, 0, s.top_k)             # a quarter of the requests has no count
            s.top_p = torch.full((n,), s.top_p, device="cuda")
            s.min_p = torch.full((n,), s.min_p, device="cuda")
    return s


# ---- the operators in plain operations ------------------------------------------------------------------------------------

CHUNK = 128


def _powers(log_decay, exponents):
    """decay^exponents for each head, [heads, ...] in float32, from angles in 64 bits; 0 for negative exponents."""
    e = exponents.double()
    g = log_decay.double().view((-1,) + (1,) * e.dim())
    return torch.where(e < 0, 0.0, torch.exp(g * e.clamp(min=0))).float()


def _run_through(a, b, c, log_decay, first):
    """out_i = sum over j <= i of decay^(i - j) (a_i . b_j) c_j, with [batch, heads, steps, width] of each; chunk by chunk, the states
    between chunks through one product with the powers of a chunk's decay.  first: where the sums run the other way."""
    n = a.size(2)
    if first:
        return _run_through(a.flip(2), b.flip(2), c.flip(2), log_decay, False).flip(2)
    chunks = -(-n // CHUNK)
    a, b, c = (torch.nn.functional.pad(t, (0, 0, 0, chunks * CHUNK - n)).unflatten(2, (chunks, CHUNK)) for t in (a, b, c))
    i = torch.arange(CHUNK, device="cuda")
    inside = _powers(log_decay, i[:, None] - i[None, :])[:, None]              # [heads, 1, i, j]
    out = ((a @ b.transpose(-1, -2)) * inside) @ c
    if chunks > 1:
        ends = (b * _powers(log_decay, CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2) @ c
        m = torch.arange(chunks, device="cuda")
        between = _powers(log_decay, (m[:, None] - 1 - m[None, :]) * CHUNK)    # state before chunk m from each chunk's own
        before = (between @ ends.flatten(-2)).unflatten(-1, ends.shape[-2:])
        out = out + (a * _powers(log_decay, i + 1)[:, None, :, None]) @ before
    return out.flatten(2, 3)[:, :, :n]


def _heads_first(t, heads):
    return t.float().repeat_interleave(heads // t.size(2), 2).transpose(1, 2)


def _plain_attend(s):
    t, h, kv, scale = s.q.dtype, s.q.size(2), s.k.size(2), s.scale
    b, n = s.q.shape[:2]
    lengths = s.lengths if s.lengths is not None else torch.full((b,), n, device="cuda")
    steps = torch.arange(n, device="cuda")
    inside = (steps < lengths[:, None])[:, None, :, None]
    q, k, v = (torch.where(inside, _heads_first(x, h), 0.0) for x in (s.q, s.k, s.v))
    since = _powers(s.log_decay, steps + 1)[:, :, None]                        # of the first state, after each step
    left = _powers(s.log_decay, lengths[:, None] - 1 - steps).transpose(0, 1)[..., None]     # of each step, in the last state
    all_of = _powers(s.log_decay, lengths).transpose(0, 1)[..., None, None]
    out = scale * (_run_through(q, k, v, s.log_decay, False) + (q * since) @ s.state)
    last = all_of * s.state + (k * left).transpose(-1, -2) @ v
    out = out.transpose(1, 2).to(t)
    if not s.case["train"]:
        return out, last
    do = torch.where(inside, scale * s.dout.float().transpose(1, 2), 0.0)
    dq = _run_through(do, v, k, s.log_decay, False) + (do * since) @ s.state.transpose(-1, -2)
    dk = _run_through(v, do, q, s.log_decay, True) + (v * left) @ s.dlast.transpose(-1, -2)
    dv = _run_through(k, q, do, s.log_decay, True) + (k * left) @ s.dlast
    dstate = all_of * s.dlast + (q * since).transpose(-1, -2) @ do

    def shared(x):
        return x.unflatten(1, (kv, h // kv)).sum(2).transpose(1, 2).to(t)

    return out, last, dq.transpose(1, 2).to(t), shared(dk), shared(dv), dstate


def _plain_step(s):
    h = s.q.size(1)
    k, v = (x.float().repeat_interleave(h // x.size(1), 1) for x in (s.k, s.v))
    state = torch.exp(s.log_decay)[:, None, None] * s.state[s.slots] + k[..., None] * v[..., None, :]
    s.state[s.slots] = state
    return (s.scale * (s.q.float()[..., None] * state).sum(-2)).to(s.q.dtype), s.state


def _plain_norm(s):
    c, t = s.case, s.x.dtype
    n, p, channels = s.x.shape
    split = (c["groups"], channels // c["groups"])
    x = s.x.float().unflatten(-1, split)
    mean = x.mean((1, 3), keepdim=True)
    r = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + 1e-5)
    h = ((x - mean) * r).flatten(-2)
    z = h * s.weight.float() + s.bias.float()
    if s.residual is not None:
        z = z + s.residual.float()
    sig = torch.sigmoid(z)
    y = {"none": z, "relu": z.clamp(min=0), "silu": z * sig}[c["act"]].to(t)
    if not c["train"]:
        return y
    dy = s.dy.float()
    dz = {"none": dy, "relu": torch.where(z > 0, dy, 0.0), "silu": dy * (sig * (1 + z * (1 - sig)))}[c["act"]]
    dw, db = (dz * h).sum((0, 1)).to(s.weight.dtype), dz.sum((0, 1)).to(s.bias.dtype)
    dh = (dz * s.weight.float()).unflatten(-1, split)
    h = h.unflatten(-1, split)
    dx = r * (dh - dh.mean((1, 3), keepdim=True) - h * (dh * h).mean((1, 3), keepdim=True))
    return (y, dx.flatten(-2).to(t), dw, db) + ((dz.to(t),) if s.residual is not None else ())


def _column(value, logits, dtype):
    """A setting that is a number or one of each row, as a column."""
    return torch.as_tensor(value, device=logits.device).to(dtype).expand(logits.size(0))[:, None]


def _plain_sample(s):
    x = s.logits.float()
    vocab = x.size(-1)
    inverse = 1.0 / _column(s.temperature, x, torch.float32)
    top_k, top_p, min_p = _column(s.top_k, x, torch.int64), _column(s.top_p, x, torch.float32), _column(s.min_p, x, torch.float32)
    e = torch.exp((x - x.amax(-1, keepdim=True)) * inverse)
    w = (e.double() * 2.0 ** 40).long()
    order = x.sort(dim=-1, descending=True, stable=True).indices
    place = torch.arange(vocab, device="cuda")
    wo = w.gather(-1, order)
    wo = torch.where((top_k <= 0) | (place < top_k), wo, 0)
    up_to = wo.cumsum(-1)
    enough = top_p.double() * up_to[:, -1:].double()
    kept = (wo > 0) & ((top_p >= 1) | ((up_to - wo).double() < enough)) & (e.gather(-1, order) >= min_p) | (place == 0)
    w = w * torch.zeros_like(w, dtype=torch.bool).scatter_(-1, order, kept)
    up_to = w.cumsum(-1)
    total = up_to[:, -1:]
    r = torch.minimum((s.uniform[:, None].double() * total.double()).floor().long(), total - 1)
    token = (up_to <= r).sum(-1, keepdim=True)
    logprob = torch.log(w.gather(-1, token).double()) - torch.log(total.double())
    return token[:, 0], logprob[:, 0].float()


# ---- one pass -------------------------------------------------------------------------------------------------------------

def run(state):
    s = state
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"attend": _plain_attend, "step": _plain_step, "norm": _plain_norm, "sample": _plain_sample}[s.case["op"]](s)


def _run_own(s):
    import deform_conv3d_pytorch_op_b200 as dcn
    c, op = s.case, s.case["op"]
    grad = torch.autograd.grad
    if op == "step":
        return dcn.DecayAttentionFunction.step(s.q, s.k, s.v, s.log_decay, s.state, s.slots, s.scale), s.state
    if op == "attend":
        out, last = dcn.DecayAttentionFunction.apply(s.q, s.k, s.v, s.log_decay, s.state, s.lengths, s.scale)
        if not c["train"]:
            return out, last
        return (out.detach(), last.detach()) + grad((out, last), (s.q, s.k, s.v, s.state), (s.dout, s.dlast))
    if op == "norm":
        y = dcn.GroupNormActFunction.apply(s.x, c["groups"], s.weight, s.bias, s.residual, c["act"], 1e-5)
        if not c["train"]:
            return y
        return (y.detach(),) + grad((y,), s.asked, (s.dy,))
    return dcn.TokenSampleFunction.apply(s.logits, s.uniform, s.temperature, s.top_k, s.top_p, s.min_p)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

def work(case):
    op, e = case["op"], SIZE[case["type"]]
    if op in ("attend", "step"):
        h, kv, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
        once = (h * (dk + dv) + kv * (dk + dv)) * e                            # q, k, v and out of a step
        if op == "step":                       # and the states, in and out
            return {"bytes": case["rows"] * (once + 8 * h * dk * dv), "flops": 5 * case["rows"] * h * dk * dv}
        n = case["batch"] * case["steps"]
        ends = 8 * case["batch"] * h * dk * dv
        if case["train"]:                      # with the gradients of all four, both ways three products with the state
            return {"bytes": 2 * (n * once + ends), "flops": 12 * n * h * dk * dv}
        return {"bytes": n * once + ends, "flops": 4 * n * h * dk * dv}
    if op == "norm":
        n, c, w = case["samples"] * case["positions"] * case["channels"], case["channels"], SIZE[case["weights"]]
        k = 1 if case["residual"] else 0
        if case["train"]:                      # x, residual, dy in; y, dx, dresidual out
            return {"bytes": n * e * (4 + 2 * k) + 4 * c * w, "flops": 25 * n}
        return {"bytes": n * e * (2 + k) + 2 * c * w, "flops": 9 * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * e + 16 * case["rows"], "flops": 6 * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attend": _exact_attend, "step": _exact_step, "norm": _exact_norm, "sample": _exact_sample}[case["op"]](case, s)


def _exact_step(case, s):
    each = case["heads"] // case["kv_heads"]
    key, value = s.k.double().repeat_interleave(each, 1), s.v.double().repeat_interleave(each, 1)
    old = s.state.double()
    new = old[s.slots] * s.log_decay.double().exp()[None, :, None, None] + torch.einsum("rhi,rhj->rhij", key, value)
    return torch.einsum("rhi,rhij->rhj", s.q.double(), new) * s.scale, old.index_copy(0, s.slots, new)


def _exact_attend(case, s):
    each, steps = case["heads"] // case["kv_heads"], case["steps"]
    d = s.log_decay.double().exp()[:, None, None]
    q = s.q.detach().double()
    key, value = s.k.detach().double().repeat_interleave(each, 2), s.v.detach().double().repeat_interleave(each, 2)
    ends = s.lengths.tolist() if s.lengths is not None else [steps] * case["batch"]
    live = torch.tensor([[float(t < e) for e in ends] for t in range(steps)], device="cuda", dtype=torch.float64)[:, :, None, None, None]
    state = s.state.detach().double()
    out = torch.zeros(*s.v.shape[:2], case["heads"], case["dv"], device="cuda", dtype=torch.float64)
    dq = torch.zeros_like(q)
    train = case["train"]
    for t in range(steps):                     # the recurrence as it stands
        grown = state * d + key[:, t, :, :, None] * value[:, t, :, None, :]
        state = torch.lerp(state, grown, live[t])
        out[:, t] = torch.matmul(q[:, t, :, None], state)[:, :, 0] * live[t, :, 0] * s.scale
        if train:
            dq[:, t] = torch.matmul(state, s.dout[:, t].double()[..., None])[..., 0] * live[t, :, 0] * s.scale
    if not train:
        return out, state
    dkey, dvalue, back = torch.zeros_like(key), torch.zeros_like(value), s.dlast.double()
    for t in range(steps - 1, -1, -1):
        here = back + s.scale * q[:, t, :, :, None] * s.dout[:, t].double()[:, :, None, :]
        dkey[:, t] = torch.matmul(here, value[:, t, :, :, None])[..., 0] * live[t, :, 0]
        dvalue[:, t] = torch.matmul(key[:, t, :, None], here)[:, :, 0] * live[t, :, 0]
        back = torch.lerp(back, here * d, live[t])
    kv = case["kv_heads"]
    return out, state, dq, dkey.unflatten(2, (kv, each)).sum(3), dvalue.unflatten(2, (kv, each)).sum(3), back


def _exact_norm(case, s):
    def wide(v):
        return None if v is None else v.detach().double().requires_grad_(case["train"])

    x, weight, bias, residual = wide(s.x), wide(s.weight), wide(s.bias), wide(s.residual)
    with torch.enable_grad():
        n, p, c = x.shape
        g = x.view(n, p, case["groups"], -1).transpose(1, 2).reshape(n, case["groups"], -1)
        g = (g - g.sum(-1, keepdim=True) / g.size(-1))
        g = g / (g.pow(2).sum(-1, keepdim=True) / g.size(-1) + 1e-5).sqrt()
        z = g.view(n, case["groups"], p, -1).transpose(1, 2).reshape(n, p, c) * weight + bias
        z = z if residual is None else z + residual
        y = z if case["act"] == "none" else torch.relu(z) if case["act"] == "relu" else z / (1 + torch.exp(-z))
        if not case["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, [v for v in (x, weight, bias, residual) if v is not None], s.dy.double())


def _exact_sample(case, s):
    n, v = s.logits.shape

    def row(value):
        return value.double() if isinstance(value, torch.Tensor) else torch.full((n,), value, dtype=torch.float64, device="cuda")

    temperature, count, mass, least = row(s.temperature), row(s.top_k), row(s.top_p), row(s.min_p)
    z = s.logits.double()
    p = torch.exp((z - z.max(1).values[:, None]) / temperature[:, None])
    p = torch.floor(p * 2 ** 40) / 2 ** 40
    ranked, who = torch.sort(z, dim=1, descending=True, stable=True)
    q = p.gather(1, who)
    rank = torch.arange(v, device="cuda")[None]
    q = q.masked_fill((count > 0)[:, None] & (rank >= count[:, None]), 0)
    before = torch.cumsum(q, 1) - q
    q = q.masked_fill((mass < 1)[:, None] & (before >= mass[:, None] * q.sum(1, keepdim=True)) & (rank > 0), 0)
    q = q.masked_fill((q < least[:, None]) & (rank > 0), 0)
    by_index = torch.zeros_like(q).scatter(1, who, q)
    sums = torch.cumsum(by_index, 1)
    token = torch.searchsorted(sums, (s.uniform.double() * sums[:, -1])[:, None], right=True).clamp(max=v - 1)
    return None, (by_index.gather(1, token) / sums[:, -1:]).log()[:, 0]

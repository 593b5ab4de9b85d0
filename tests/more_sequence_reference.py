"""Decayed attention, group norm with an activation and token sampling from their definitions.  Bounds: those of
tests/sequence_reference.py, with what the kernels round in between added where a test says so."""
import math

import torch


def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale=None):
    """Differentiable, in the type of its arguments (64 bits), all pairs of steps at once: out, last."""
    b, n, h, dk = q.shape
    scale = dk ** -0.5 if scale is None else scale
    k, v = (x.repeat_interleave(h // x.size(2), 2) for x in (k, v))
    lengths = torch.full((b,), n, device=q.device) if lengths is None else lengths.clamp(0, n)
    t = torch.arange(n, device=q.device)
    live = t < lengths[:, None]                                                  # [b, n]
    q, k, v = (torch.where(live[..., None, None], x, 0.0) for x in (q, k, v))
    g = log_decay.double().clamp(max=0.0).to(q.dtype)

    def power(e):                                                               # decay^e by head, 0 for negative e, 1 for 0
        e = e.to(q.dtype)
        x = torch.where(e > 0, e * g.view((-1,) + (1,) * e.dim()), 0.0)
        return torch.where(e < 0, 0.0, torch.exp(x))

    scores = torch.einsum("bihd,bjhd->bhij", q, k) * power(t[:, None] - t[None, :])
    out = torch.einsum("bhij,bjhe->bihe", scores, v)
    left = power(lengths[:, None] - 1 - t)                                      # [h, b, n]
    last = torch.einsum("hbj,bjhd,bjhe->bhde", left, k, v)
    if state is not None:
        out = out + torch.einsum("hi,bihd,bhde->bihe", power(t + 1), q, state)
        last = last + power(lengths).t()[..., None, None] * state
    return out * scale, last


def decay_attention_steps(q, k, v, log_decay, state=None, scale=None):
    """The recurrence itself"""
    b, n, h, dk = q.shape
    k, v = (x.repeat_interleave(h // x.size(2), 2) for x in (k, v))
    s = q.new_zeros(b, h, dk, v.size(3)) if state is None else state
    out = []
    for t in range(n):
        s = torch.exp(log_decay.to(q.dtype))[:, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append((q[:, t, :, :, None] * s).sum(-2) * (dk ** -0.5 if scale is None else scale))
    return torch.stack(out, 1), s


def group_norm_act(x, groups, weight=None, bias=None, residual=None, activation=None, eps=1e-5):
    n, c = x.size(0), x.size(-1)
    g = x.reshape(n, -1, groups, c // groups)
    d = g - g.mean((1, 3), keepdim=True)
    z = (d / torch.sqrt(d.square().mean((1, 3), keepdim=True) + eps)).reshape(x.shape)
    z = z if weight is None else z * weight
    z = z if bias is None else z + bias
    z = z if residual is None else z + residual
    return z if activation in (None, "none") else z.clamp(min=0) if activation == "relu" else z * torch.sigmoid(z)


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Rows one by one, with whole numbers: token, logprob (64 bits).  The exponential in float32 is what the definition has."""
    rows, v = logits.shape

    def column(x, t):
        return torch.as_tensor(x, device=logits.device).to(t).expand(rows)

    x = logits.float()
    temperature, top_k = column(temperature, torch.float32), column(top_k, torch.int64)
    top_k = torch.where(temperature == 0, 1, top_k)
    temperature = torch.where(temperature == 0, 1.0, temperature.clamp(1e-3, 1e3))
    top_p, min_p = column(top_p, torch.float32), column(min_p, torch.float32)
    largest = x.amax(-1)
    fine = torch.isfinite(largest) & ~torch.isnan(x).any(-1)
    e = torch.exp((x - largest[:, None]) * (1.0 / temperature)[:, None])
    w = (e.double() * 2.0 ** 40).nan_to_num(0.0).long()
    tokens, logprobs = [], []
    for r in range(rows):
        if not bool(fine[r]):
            tokens.append(-1)
            logprobs.append(float("nan"))
            continue
        order = x[r].sort(descending=True, stable=True).indices
        order = order[w[r][order] > 0]
        if 0 < int(top_k[r]) < v:
            order = order[:int(top_k[r])]
        mass = w[r][order].cumsum(0)
        if float(top_p[r]) < 1:
            before, enough = mass - w[r][order], top_p[r].double() * mass[-1].double()
            order = order[(before.double() < enough) | (torch.arange(order.numel(), device=order.device) == 0)]
        best = order[0]
        kept = order[(e[r][order] >= min_p[r]) | (order == best)].sort().values
        mass = w[r][kept].cumsum(0)
        target = min(int(float(uniform[r]) * float(mass[-1])), int(mass[-1]) - 1)
        i = int(kept[int((mass <= target).sum())])
        tokens.append(i)
        logprobs.append(math.log(int(w[r, i])) - math.log(int(mass[-1])))
    return torch.tensor(tokens, device=logits.device), torch.tensor(logprobs, device=logits.device, dtype=torch.float64)


def decay_attention_blocks(q, k, v, log_decay, state=None, lengths=None, scale=None, block=512):
    """decay_attention for long sequences: block by block, each from the state that the one before has left."""
    lengths = torch.full((q.size(0),), q.size(1), device=q.device) if lengths is None else lengths.clamp(0, q.size(1))
    out = []
    for t in range(0, q.size(1), block):
        o, state = decay_attention(q[:, t:t + block], k[:, t:t + block], v[:, t:t + block], log_decay, state, lengths - t, scale)
        out.append(o)
    return torch.cat(out, 1), state

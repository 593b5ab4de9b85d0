"""The sequence operators from their definitions, in 64 bits, and the bounds their results are held to.

Bounds.  A result in float32 is a chain of a few rounded operations and of function values good to about 2 units in the last
place, over sums made as trees; errors of a sum's terms are independent, so that the 2-norm of the error stays within some
tens of roundings of the result's: 64 * 2^-24.  Rounding to a 16-bit type adds at most half its spacing to each element: 2^-8
relative for bfloat16, 2^-11 for float16.  A single element may be off by 40 times the norm's share, of its own size or of the
root mean square where that is more.  Results near zero in exact arithmetic (a loss or a gradient of equal distributions) are
compared on the scale `scale` of the terms they are made of.
"""
import math

import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHAIN = 64 * 2.0 ** -24
ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def close(got, want, what="", scale=0.0, chain=CHAIN):
    """Asserts the bounds above; infinities and NaN have to be the same."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = chain + ROUND[got.dtype]
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0                # float16's smallest spacing
    g, w = got.detach().double().flatten(), want.detach().double().flatten()
    if got.dtype == torch.float16:
        w = torch.where(w.abs() >= 65520, w.sign() * math.inf, w)
    fine = torch.isfinite(w)
    assert torch.equal(fine, torch.isfinite(g)), (what, "infinities or NaN differ")
    assert torch.equal(torch.isnan(w), torch.isnan(g)) and torch.equal(w[torch.isinf(w)], g[torch.isinf(w)]), what
    g, w = g[fine], w[fine]
    if not w.numel():
        return
    d, rms = (g - w).abs(), max(float(w.square().mean().sqrt()), scale)
    assert float(d.square().mean().sqrt()) <= tol * rms + tiny, (what, float(d.square().mean().sqrt()), tol * rms)
    assert bool((d <= 40 * tol * w.abs().clamp(min=rms) + tiny).all()), (what, float((d / w.abs().clamp(min=rms)).max()), 40 * tol)


def scan(x, gate, state=None, lengths=None):
    """Differentiable, step by step: y, last."""
    b, n, c = x.shape
    h = torch.zeros(b, c, dtype=torch.float64, device=x.device) if state is None else state
    out = []
    for t in range(n):
        a = torch.sigmoid(gate[:, t])
        new = a * h + torch.sigmoid(-gate[:, t]) * x[:, t]
        if lengths is not None:
            live = (t < lengths)[:, None]
            h = torch.where(live, new, h)
            out.append(torch.where(live, new, 0.0))
        else:
            h = new
            out.append(new)
    return (torch.stack(out, 1) if out else x * 0), h


def residual_norm(x, block=None, gate=None, scale=None, post=None, pre=None, eps=1e-6):
    def rms(v):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)

    s = x
    if block is not None:
        s = rms(block)
        for factor in (post, scale, None if gate is None else torch.sigmoid(gate)):
            if factor is not None:
                s = s * factor
        s = x + s
    n = rms(s)
    return s, n if pre is None else n * pre


def log_softmax(logits, temperature):
    """-inf where a row has nothing left; differentiable elsewhere."""
    z = logits / temperature
    empty = (logits == -math.inf).all(-1, keepdim=True)
    return torch.where(empty, -math.inf, torch.log_softmax(torch.where(empty, 0.0, z), -1))


def token_scores(logits, tokens, top=0, temperature=1.0, ignore=-100):
    v = logits.size(-1)
    log_p = log_softmax(logits, temperature)
    finite = torch.where(log_p == -math.inf, 0.0, log_p)
    entropy = -(torch.exp(log_p) * finite).sum(-1)
    known = (tokens >= 0) & (tokens < v)
    logprob = log_p.gather(-1, torch.where(known, tokens, 0)[..., None])[..., 0]
    logprob = torch.where(known, logprob, torch.where(tokens == ignore, 0.0, math.nan))
    order = logits.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    return logprob, entropy, log_p.gather(-1, order), order


def distill(logits, teacher_logprobs, teacher_tokens, temperature=1.0, tail=True):
    """Row by row, from the definition.  [rows, vocabulary], [rows, k]."""
    losses = []
    for z, lq, t in zip(log_softmax(logits, temperature), teacher_logprobs, teacher_tokens):
        used = (t >= 0) & (t < z.numel())
        lq, t = lq[used], t[used]
        if not len(t) or (not tail and bool((lq == -math.inf).all())):
            losses.append(z.new_zeros(()) + 0 * torch.where(torch.isfinite(z), z, 0.0).sum())
            continue
        if not tail:
            lq = torch.log_softmax(lq, 0)
        q = torch.exp(lq)
        student = z[t]
        terms = torch.where(q > 0, q * (torch.where(q > 0, lq, 0.0) - torch.where(q > 0, student, 0.0)), 0.0)
        terms = torch.where(torch.isnan(q), q, terms)
        loss = terms.sum()
        others = torch.ones_like(z, dtype=torch.bool)
        others[t] = False
        if tail and bool((z[others] != -math.inf).any()):
            rest = (1 - q.sum()).clamp(min=0)
            if rest > 0:
                loss = loss + rest * (torch.log(rest) - torch.logsumexp(z[others], 0))
        losses.append(loss * temperature ** 2)
    return torch.stack(losses)

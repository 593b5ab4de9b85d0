"""Operators for what comes after the clip features of a video network: a recurrence over time, the norms around its blocks,
the loss against a larger teacher and the scores that it answers with.  (The reference has no counterpart of these.)

* :class:`GatedScanFunction`     -- per-channel gated recurrence over a sequence, its gradient, and its form for one step
* :class:`ResidualNormFunction`  -- norm behind a block, gate, scaled residual and the norm before the next block in one pass
* :class:`TokenScoresFunction`   -- log-probabilities of given tokens (or classes), entropy and the best alternatives
* :class:`DistillTopkFunction`   -- KL divergence from a teacher's best tokens
* :class:`DecayAttentionFunction` -- linear attention whose states decay, head by head, its gradient, and its form for one step
* :class:`GroupNormActFunction`  -- group norm of channels-last features with a residual and an activation
* :class:`TokenSampleFunction`   -- tokens (or classes) drawn by given random numbers after temperature, top-k, top-p and min-p

and the modules :class:`GatedScan`, :class:`ResidualNorm`, :class:`TopkDistillLoss`, :class:`DecayAttention` and :class:`GroupNormAct`
over them.

Tensors are float32, bfloat16 or float16 on a CUDA device; the last axis should be dense (it is copied otherwise), the others may
have any strides, so the parts of one projection's output are taken as they are.  Sums, statistics and states are float32.  Calls
run on the current stream, without synchronising it.  As in :mod:`functions`, the work behind ``.apply`` is C++
(``csrc/seq_torch.cpp`` over the C ABI of ``include/dcn_seq.h``); traces, function transforms and forward-mode derivatives go through
the ``_...Function`` of the same arguments.  Gradients of gradients are refused.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib


def _function(name, differentiable):
    """A torch.autograd.Function over the same forward and backward calls, for the cases named above."""

    class SequenceFunction(Function):
        @staticmethod
        def forward(ctx, *args):
            native = _lib.native()
            out, kept = getattr(native, name + "_forward")(*args)
            ctx.save_for_backward(*kept)
            ctx.args, ctx.inputs = args, len(args)
            ctx.set_materialize_grads(False)
            ctx.mark_non_differentiable(*[t for t in out if t is not None and not t.is_floating_point()])
            return out if len(out) > 1 else out[0]

        @staticmethod
        @once_differentiable
        def backward(ctx, *grads):
            if all(g is None for g in grads):
                return (None,) * ctx.inputs
            asked = [i < differentiable and isinstance(a, torch.Tensor) and need
                     for i, (a, need) in enumerate(zip(ctx.args, ctx.needs_input_grad))][:differentiable]
            want = tuple(asked) + (False,) * (differentiable - len(asked))
            got = getattr(_lib.native(), name + "_backward")(ctx.saved_tensors, grads, want, ctx.args)
            got = got[:ctx.inputs]
            return got + (None,) * (ctx.inputs - len(got))

    SequenceFunction.__name__ = SequenceFunction.__qualname__ = "_" + name
    return SequenceFunction


_GatedScanFunction = _function("gated_scan", 3)
_ResidualNormFunction = _function("residual_norm", 6)
_TokenScoresFunction = _function("token_scores", 1)
_DistillTopkFunction = _function("distill_topk", 1)


_DecayAttentionFunction = _function("decay_attention", 5)
_GroupNormActFunction = _function("group_norm_act", 4)


class _DecayAttentionStepFunction(Function):
    """As _GatedScanStepFunction."""

    @staticmethod
    def forward(ctx, *args):
        return _lib.native().decay_attention_step_forward(*args)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        raise RuntimeError("step has no gradient: take apply")


class _TokenSampleFunction(Function):
    """As _GatedScanStepFunction."""

    @staticmethod
    def forward(ctx, *args):
        out = _lib.native().token_sample_forward(*args)
        ctx.mark_non_differentiable(*out)
        return out

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("sampling has no gradient")


class _GatedScanStepFunction(Function):
    """A step that traces record; it has no derivative of any kind (and no transform: there is no setup_context)."""

    @staticmethod
    def forward(ctx, x, gate, state, slots):
        return _lib.native().gated_scan_step_forward(x, gate, state, slots)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        raise RuntimeError("step has no gradient: take apply")


class GatedScanFunction:
    """Per-channel recurrence over time: ``h_t = a_t h_{t-1} + (1 - a_t) x_t``, ``a_t = sigmoid(gate_t)``."""

    @staticmethod
    def apply(x, gate, state=None, lengths=None):
        """``(y, last)``: the states [batch, steps, channels] in x's type and the last ones [batch, channels] in float32.

        ``x``, ``gate`` [batch, steps, channels]; ``state`` [batch, channels] float32: the state before the first step (zeros);
        ``lengths`` [batch] int64 or int32: steps of each sequence.  Behind them y is zero, x and gate are not read, and last is
        the state after the sequence's own steps (``state`` where it has none).  Gradients: x, gate, state."""
        out = _lib.native().gated_scan(x, gate, state, lengths)
        return _GatedScanFunction.apply(x, gate, state, lengths) if out is NotImplemented else out

    @staticmethod
    def step(x, gate, state, slots=None):
        """One step of running sequences, without gradients: ``x``, ``gate`` [rows, channels]; ``state`` [pool, channels]
        float32, contiguous, advanced in place at the rows ``slots`` [rows] (0, 1, ... if None), each of which occurs once; a
        slot outside the pool is skipped, and its row is zero.  Returns the new states [rows, channels] in x's type."""
        out = _lib.native().gated_scan_step(x, gate, state, slots)
        return _GatedScanStepFunction.apply(x, gate, state, slots) if out is NotImplemented else out


class ResidualNormFunction:
    """``stream = x + scale * sigmoid(gate) * rms(block) * post_weight``; ``normed = rms(stream) * pre_weight``, with
    ``rms(v) = v / sqrt(mean(v^2) + eps)`` over the last axis (1 to 8192 channels)."""

    @staticmethod
    def apply(x, block=None, gate=None, scale=None, post_weight=None, pre_weight=None, eps=1e-6):
        """``(stream, normed)``, both in x's type; normed comes from the unrounded stream.

        ``x``, ``block``, ``gate`` [..., channels]; ``scale``, ``post_weight``, ``pre_weight`` [channels], all float32 or all of
        x's type.  What is None is left out (a factor of one).  Without a block, stream is x itself.  Gradients: all tensors; the
        weights' are summed over the rows in a fixed order."""
        args = (x, block, gate, scale, post_weight, pre_weight, eps)
        out = _lib.native().residual_norm(*args)
        if out is NotImplemented:
            out = _ResidualNormFunction.apply(*args)
            out = out if isinstance(out, tuple) else (out,)
        return (x,) + out if block is None else out


class TokenScoresFunction:
    """Scores of rows of logits [..., vocabulary], ``log p = log_softmax(logits / temperature)``.  Logits may be any finite values
    (masks of -1e9 or of the type's lowest value among them) and -inf."""

    @staticmethod
    def apply(logits, tokens=None, top=0, temperature=1.0, ignore_index=-100):
        """``(logprob, entropy, top_logprobs, top_tokens)``, float32 and int64: log p of ``tokens`` [...] (None without tokens),
        the rows' entropy, and the ``top`` (up to 128) largest logits' log p and tokens [..., top] (None for top = 0), equal ones
        by their index.  A token ``ignore_index`` has log p 0, any other outside the vocabulary has NaN.  Logits of -inf stand
        for tokens that cannot come; a row of nothing else has log p = -inf, entropy 0 and no gradient.  Gradient: logits, from
        the three float outputs."""
        args = (logits, tokens, top, temperature, ignore_index)
        out = _lib.native().token_scores(*args)
        return _TokenScoresFunction.apply(*args) if out is NotImplemented else out


class DistillTopkFunction:
    """``temperature^2 KL(teacher || student)`` by row, from the teacher's best tokens alone."""

    @staticmethod
    def apply(logits, teacher_logprobs, teacher_tokens, temperature=1.0, tail=True):
        """``loss`` [...] in float32 for the student's logits [..., vocabulary] (up to 2^20).

        ``teacher_logprobs``, ``teacher_tokens`` [..., k], k up to 128: log-probabilities at this temperature and their tokens, as
        :class:`TokenScoresFunction` gives them for a teacher's logits.  ``tail``: all other tokens together are one more
        outcome, with the teacher's remaining probability; it is left out where the student has masked all of them (-inf).  Without
        ``tail`` the teacher's are renormalised over the k tokens.  A token outside the vocabulary (-1) marks an unused place; a row
        without any has loss 0.  Gradient: logits."""
        args = (logits, teacher_logprobs, teacher_tokens, temperature, tail)
        out = _lib.native().distill_topk(*args)
        return _DistillTopkFunction.apply(*args) if out is NotImplemented else out


class DecayAttentionFunction:
    """Linear attention over time whose states decay, for each head: ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T``,
    ``out_t = scale S_t^T q_t``."""

    @staticmethod
    def apply(q, k, v, log_decay, state=None, lengths=None, scale=None):
        """``(out, last)``: [batch, steps, heads, dv] in q's type, and the last states [batch, heads, dk, dv] in float32.

        ``q`` [batch, steps, heads, dk], ``k`` and ``v`` [batch, steps, kv_heads, dk or dv] (1 to 128 each), where kv_heads divides
        heads: neighbouring heads share a key and a value.  ``log_decay`` [heads] float32, taken as 0 where it is above: no gradient.
        ``state`` [batch, heads, dk, dv] float32: the states before the first step (zeros); ``lengths`` [batch] int64 or int32: steps
        of each sequence.  Behind them out is zero, q, k and v are not read, and last is the state after the sequence's own steps.
        ``scale``: 1 / sqrt(dk) if None.  Gradients: q, k, v, state.

        In 16-bit types a step's weight on each of the steps of its block (of 64 or 128), and the state that it meets from before, are rounded
        to the type (the states themselves are float32).  In all types NaN or infinity at a step may reach steps of its block before it."""
        args = (q, k, v, log_decay, state, lengths, scale)
        out = _lib.native().decay_attention(*args)
        return _DecayAttentionFunction.apply(*args) if out is NotImplemented else out

    @staticmethod
    def step(q, k, v, log_decay, state, slots=None, scale=None):
        """One step of running sequences, without gradients: ``q`` [rows, heads, dk], ``k``, ``v`` [rows, kv_heads, dk or dv];
        ``state`` [pool, heads, dk, dv] float32, contiguous, advanced in place at the rows ``slots`` [rows] (0, 1, ... if None),
        each of which occurs once; a slot outside the pool is skipped, and its row is zero.  Returns [rows, heads, dv]."""
        args = (q, k, v, log_decay, state, slots, scale)
        out = _lib.native().decay_attention_step(*args)
        return _DecayAttentionStepFunction.apply(*args) if out is NotImplemented else out


_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2}


class GroupNormActFunction:
    """``act((x - mean) / sqrt(var + eps) * weight + bias + residual)``, mean and variance over the positions and channels of each
    sample's groups."""

    @staticmethod
    def apply(x, groups, weight=None, bias=None, residual=None, activation=None, eps=1e-5):
        """``y`` in x's type and shape [samples, ..., channels] (1 to 8192 channels, copied where it is not contiguous).

        ``weight``, ``bias`` [channels], both float32 or both of x's type; ``residual`` as x; ``activation``: None, "relu" or "silu".
        Gradients: x, weight, bias, residual; sums over samples are made in a fixed order."""
        act = _ACTIVATIONS.get(activation)
        if act is None:
            raise _lib.DcnError("activation is %r: None, 'relu' and 'silu' are supported" % (activation,))
        args = (x, weight, bias, residual, groups, act, eps)
        out = _lib.native().group_norm_act(*args)
        return _GroupNormActFunction.apply(*args) if out is NotImplemented else out


class TokenSampleFunction:
    """Tokens drawn from rows of logits [..., vocabulary] (up to 2^20) by given random numbers."""

    @staticmethod
    def apply(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """``(tokens, logprob)``, int64 and float32 [...], from ``uniform`` [...] float32 in [0, 1).

        A row keeps its ``top_k`` largest logits (all for 0), equal ones by index; of these the fewest that have ``top_p`` of the
        probability; of these the ones with ``min_p`` of the largest probability.  The token is where the kept probabilities,
        added by index, pass ``uniform`` of their sum, and logprob its logarithm among them.  Each setting is a number or a tensor
        [...] with one for each row.  ``temperature`` lies between 1e-3 and 1e3 (a tensor's is taken into it), or is 0 for the best token.
        Probabilities are whole numbers of 2^-40 of the largest, so that a draw does not depend on how sums are split.  Logits of -inf
        stand for tokens that cannot come; rows of nothing else, with NaN or with +inf give token -1 and NaN.  No gradient."""
        args = (logits, uniform, temperature, top_k, top_p, min_p)
        out = _lib.native().token_sample(*args)
        return _TokenSampleFunction.apply(*args) if out is NotImplemented else out


class GatedScan(nn.Module):
    """Projection of features to value and gate, and the recurrence over them: [batch, steps, features] -> [batch, steps,
    channels].  The gate's bias starts where a state lasts ``memory`` steps."""

    def __init__(self, features, channels, memory=16.0, device=None, dtype=None):
        super().__init__()
        self.features, self.channels = features, channels
        self.proj = nn.Linear(features, 2 * channels, device=device, dtype=dtype)
        with torch.no_grad():
            self.proj.bias[channels:] = float(torch.tensor(max(memory, 1.001) - 1.0).log())

    def forward(self, input, state=None, lengths=None):
        x, gate = self.proj(input).chunk(2, -1)
        return GatedScanFunction.apply(x, gate, state, lengths)

    def step(self, input, state, slots=None):
        x, gate = self.proj(input).chunk(2, -1)
        return GatedScanFunction.step(x, gate, state, slots)

    def new_states(self, rows):
        """Zeros for a pool of ``rows`` sequences' states."""
        return torch.zeros(rows, self.channels, device=self.proj.weight.device)

    def extra_repr(self):
        return "{features}, {channels}".format(**self.__dict__)


class GroupNormAct(nn.Module):
    """Weights of a group norm, and the activation behind it: ``forward(x, residual)``.  The channels are axis ``dim`` of x: 1 as in
    ``nn.GroupNorm`` (stored channels last, x is read as it is), or -1, where all axes but the first and the last are positions."""

    def __init__(self, groups, channels, activation=None, dim=1, eps=1e-5, device=None, dtype=None):
        super().__init__()
        if groups < 1 or channels % groups:
            raise _lib.DcnError("%d groups do not divide the %d channels" % (groups, channels))
        if not 1 <= channels <= 8192:
            raise _lib.DcnError("%d channels: 1 to 8192 are supported" % channels)
        self.groups, self.channels, self.activation, self.dim, self.eps = groups, channels, activation, dim, eps
        self.weight = nn.Parameter(torch.ones(channels, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(channels, device=device, dtype=dtype))

    def forward(self, x, residual=None):
        if self.dim not in (-1, x.dim() - 1):
            x = x.movedim(self.dim, -1)
            residual = residual if residual is None else residual.movedim(self.dim, -1)
            return GroupNormActFunction.apply(x, self.groups, self.weight, self.bias, residual, self.activation, self.eps).movedim(-1, self.dim)
        return GroupNormActFunction.apply(x, self.groups, self.weight, self.bias, residual, self.activation, self.eps)

    def extra_repr(self):
        return "{groups}, {channels}, activation={activation}, dim={dim}, eps={eps}".format(**self.__dict__)


class DecayAttention(nn.Module):
    """Projection of features to queries, keys and values, decayed attention over time, and a group norm with SiLU over each head's
    outputs: [batch, steps, features] -> [batch, steps, heads * dv] (up to 8192).  The first head's states last about ``memory`` steps, the last
    one's sixteen times as long."""

    def __init__(self, features, heads, dk, dv=None, kv_heads=None, memory=8.0, device=None, dtype=None):
        super().__init__()
        dv, kv_heads = dk if dv is None else dv, heads if kv_heads is None else kv_heads
        if not (1 <= dk <= 128 and 1 <= dv <= 128) or heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise _lib.DcnError("%d heads of %d and %d elements and %d of keys: 1 to 128 elements, and heads that the keys' divide"
                                % (heads, dk, dv, kv_heads))
        if heads * dv > 8192:
            raise _lib.DcnError("%d heads of %d elements: their norm takes up to 8192 channels" % (heads, dv))
        self.features, self.heads, self.kv_heads, self.dk, self.dv = features, heads, kv_heads, dk, dv
        self.proj = nn.Linear(features, heads * dk + kv_heads * (dk + dv), device=device, dtype=dtype)
        self.norm = GroupNormAct(heads, heads * dv, "silu", dim=-1, device=device, dtype=dtype)
        last = memory * 16.0 ** (torch.arange(heads, dtype=torch.float64) / max(heads - 1, 1))
        self.register_buffer("log_decay", torch.log1p(-1.0 / last.clamp(min=1.001)).float().to(device))

    def _apply(self, fn, recurse=True):
        decay = self.log_decay
        super()._apply(fn, recurse)
        if self.log_decay.dtype != torch.float32:            # decays stay float32 in modules of 16 bits
            self.log_decay = decay.to(self.log_decay.device)
        return self

    def _parts(self, input):
        h, kv, dk, dv = self.heads, self.kv_heads, self.dk, self.dv
        q, k, v = self.proj(input).split((h * dk, kv * dk, kv * dv), -1)
        return q.unflatten(-1, (h, dk)), k.unflatten(-1, (kv, dk)), v.unflatten(-1, (kv, dv)), self.log_decay

    def forward(self, input, state=None, lengths=None):
        out, last = DecayAttentionFunction.apply(*self._parts(input), state, lengths)
        return self.norm(out.flatten(0, 1).flatten(1)).unflatten(0, out.shape[:2]), last

    def step(self, input, state, slots=None):
        return self.norm(DecayAttentionFunction.step(*self._parts(input), state, slots).flatten(1))

    def new_states(self, rows):
        """Zeros for a pool of ``rows`` sequences' states."""
        return torch.zeros(rows, self.heads, self.dk, self.dv, device=self.proj.weight.device)

    def extra_repr(self):
        return "{features}, heads={heads}, kv_heads={kv_heads}, dk={dk}, dv={dv}".format(**self.__dict__)


class ResidualNorm(nn.Module):
    """Weights of one place between two blocks: ``forward(x, block, gate) -> stream, normed``; ``first=True``: the place before
    the first block, ``forward(x) -> x, normed``."""

    def __init__(self, channels, first=False, scale=1.0, eps=1e-6, device=None, dtype=None):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        self.channels, self.eps = channels, eps
        self.pre_weight = nn.Parameter(torch.ones(channels, **kw))
        if first:
            self.register_parameter("scale", None)
            self.register_parameter("post_weight", None)
        else:
            self.scale = nn.Parameter(torch.full((channels,), float(scale), **kw))
            self.post_weight = nn.Parameter(torch.ones(channels, **kw))

    def forward(self, x, block=None, gate=None):
        return ResidualNormFunction.apply(x, block, gate, self.scale, self.post_weight, self.pre_weight, self.eps)

    def extra_repr(self):
        return "{channels}, eps={eps}".format(**self.__dict__)


class TopkDistillLoss(nn.Module):
    """Mean of :class:`DistillTopkFunction` over all rows, those without a used place among them (whose loss is 0).
    :meth:`teacher` makes its targets from a teacher's logits."""

    def __init__(self, k, temperature=1.0, tail=True):
        super().__init__()
        self.k, self.temperature, self.tail = k, temperature, tail

    def teacher(self, logits):
        with torch.no_grad():
            return TokenScoresFunction.apply(logits, None, self.k, self.temperature)[2:]

    def forward(self, logits, teacher_logprobs, teacher_tokens):
        return DistillTopkFunction.apply(logits, teacher_logprobs, teacher_tokens, self.temperature, self.tail).mean()

    def extra_repr(self):
        return "{k}, temperature={temperature}, tail={tail}".format(**self.__dict__)

"""Operators for what comes after the clip features of a video network: a recurrence over time, the norms around its blocks,
the loss against a larger teacher and the scores that it answers with.  (The reference has no counterpart of these.)

* :class:`GatedScanFunction`     -- per-channel gated recurrence over a sequence, its gradient, and its form for one step
* :class:`ResidualNormFunction`  -- norm behind a block, gate, scaled residual and the norm before the next block in one pass
* :class:`TokenScoresFunction`   -- log-probabilities of given tokens (or classes), entropy and the best alternatives
* :class:`DistillTopkFunction`   -- KL divergence from a teacher's best tokens

and the modules :class:`GatedScan`, :class:`ResidualNorm` and :class:`TopkDistillLoss` over them.

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

    def extra_repr(self):
        return "{features}, {channels}".format(**self.__dict__)


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

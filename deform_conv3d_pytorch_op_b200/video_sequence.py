"""Long videos: a recurrent head over the features of consecutive clips, trained from a larger teacher's best classes, answering
clip by clip.  The operators of :mod:`sequence` as they are used together; everything else is stock PyTorch.

    features of each clip (R3D18Deform.features, or any others)
      -> norm -> [ value and gate -> gated scan over the clips -> projection -> gated residual norm ] x blocks -> classes

or, with ``mixer="attention"``, queries, keys and values -> decayed attention over the clips -> group norm of each head with SiLU in the
place of value and gate -> gated scan.  :class:`SequenceHead` runs over whole sequences (training, stored videos; sequences of different lengths in one batch) and, with
:meth:`SequenceHead.step`, over live streams one clip at a time, whose states live in a pool with a row for each stream.

``python -m deform_conv3d_pytorch_op_b200.video_sequence [scan|attention]`` trains a small head on synthetic features and lets it answer.
"""
from __future__ import annotations

import sys
from typing import List, Optional

import torch
import torch.nn as nn

from ._lib import DcnError
from .sequence import DecayAttention, GatedScan, ResidualNorm, TokenSampleFunction, TokenScoresFunction, TopkDistillLoss


class SequenceBlock(nn.Module):
    """Gated scan or decayed attention, projection, and the gate and norms that join it to the stream."""

    def __init__(self, width, memory, device=None, dtype=None, mixer="scan", heads=8):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        if mixer == "scan":
            self.scan = GatedScan(width, width, memory=memory, **kw)
        elif mixer == "attention" and width % heads == 0:
            self.scan = DecayAttention(width, heads, width // heads, memory=memory, **kw)
        else:
            raise DcnError("mixer is %r of %d heads for width %d: 'scan' or 'attention', of heads that divide the width" % (mixer, heads, width))
        self.out = nn.Linear(width, width, bias=False, **kw)
        self.gate = nn.Linear(width, width, **kw)
        self.norm = ResidualNorm(width, scale=0.5, **kw)

    def forward(self, stream, normed, state=None, lengths=None):
        y, last = self.scan(normed, state, lengths)
        return self.norm(stream, self.out(y), self.gate(normed)) + (last,)

    def step(self, stream, normed, state, slots=None):
        return self.norm(stream, self.out(self.scan.step(normed, state, slots)), self.gate(normed))


class SequenceHead(nn.Module):
    """[batch, clips, features] -> logits [batch, clips, classes].  The blocks' states last about ``memory`` clips at first, four
    times as long from block to block."""

    def __init__(self, features=512, width=512, num_classes=400, blocks=2, memory=8.0, device=None, dtype=None, mixer="scan", heads=8):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        self.width = width
        self.embed = nn.Linear(features, width, **kw)
        self.first = ResidualNorm(width, first=True, **kw)
        self.blocks = nn.ModuleList([SequenceBlock(width, memory * 4 ** i, mixer=mixer, heads=heads, **kw) for i in range(blocks)])
        self.fc = nn.Linear(width, num_classes, **kw)

    def forward(self, features, states: Optional[List[torch.Tensor]] = None, lengths=None):
        """``(logits, states)``: states of each block in float32 ([batch, width], or [batch, heads, width / heads, width / heads] of
        attention), to go on from in a later call."""
        stream, normed = self.first(self.embed(features))
        out = []
        for i, block in enumerate(self.blocks):
            stream, normed, last = block(stream, normed, None if states is None else states[i], lengths)
            out.append(last)
        return self.fc(normed), out

    def new_pool(self, streams):
        """States for :meth:`step`: a row for each of ``streams`` live streams, in each block."""
        return [block.scan.new_states(streams) for block in self.blocks]

    @torch.no_grad()
    def step(self, features, pool, slots=None):
        """Logits [rows, classes] of one more clip of the streams ``slots``, whose rows of the pool advance in place."""
        stream, normed = self.first(self.embed(features))
        for block, state in zip(self.blocks, pool):
            stream, normed = block.step(stream, normed, state, slots)
        return self.fc(normed)

    @torch.no_grad()
    def answer(self, logits, top=5):
        """(classes [..., top], their probabilities, entropy) of logits; all classes where there are fewer."""
        _, entropy, best, classes = TokenScoresFunction.apply(logits, None, min(top, logits.size(-1)))
        return classes, best.exp(), entropy


    @torch.no_grad()
    def sample(self, logits, uniform=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """(classes [...], log-probabilities [...]) drawn from logits by the random numbers ``uniform`` [...] (fresh ones if None),
        as :class:`TokenSampleFunction` does."""
        if uniform is None:
            uniform = torch.rand(logits.shape[:-1], device=logits.device)
        return TokenSampleFunction.apply(logits, uniform, temperature, top_k, top_p, min_p)


def train_step(head, loss, opt, features, teacher, lengths=None):
    """One step from the teacher's best classes (``loss.teacher(logits)``).  Padding behind a sequence's clips is left out: the
    loss is the mean over the clips, however long the batch's longest sequence is (0 without any)."""
    logits, _ = head(features, lengths=lengths)
    logprobs, classes = teacher
    if lengths is not None:
        behind = torch.arange(features.size(1), device=features.device)[None, :] >= lengths[:, None]
        classes = torch.where(behind[..., None], -1, classes)
    value = loss(logits, logprobs, classes)
    if lengths is not None:                        # (the mean over all rows, of which those behind a sequence's end have 0)
        value = value * (behind.numel() / (~behind).sum().clamp(min=1))
    opt.zero_grad(set_to_none=True)
    value.backward()
    opt.step()
    return value.detach()


def main(mixer="scan"):
    torch.manual_seed(0)
    batch, clips, features, classes = 32, 64, 64, 400
    head = SequenceHead(features, 256, classes, device="cuda", mixer=mixer)
    opt = torch.optim.AdamW(head.parameters(), lr=2e-3)
    loss = TopkDistillLoss(10, temperature=2.0)
    basis = torch.randn(features, classes, device="cuda") / features ** 0.5

    def videos():                                  # the teacher judges a clip by what the last few showed
        x = torch.randn(batch, clips, features, device="cuda")
        seen = x.cumsum(1)
        seen[:, 8:] = seen[:, 8:] - x.cumsum(1)[:, :-8]
        return x, loss.teacher(seen @ basis), torch.randint(clips // 2, clips + 1, (batch,), device="cuda")

    for i in range(201):
        x, teacher, lengths = videos()
        value = train_step(head, loss, opt, x, teacher, lengths)
        if i % 40 == 0:
            print("step %3d  loss %.4f" % (i, float(value)))
    x, _, _ = videos()
    pool = head.new_pool(batch)
    for t in range(clips):                         # the same videos, live
        logits = head.step(x[:, t], pool)
    with torch.no_grad():
        whole = head(x)[0][:, -1]
    best, p, entropy = head.answer(logits)
    print("live and stored answers differ by at most %.1e" % float((logits - whole).abs().max()))
    drawn, _ = head.sample(logits, temperature=0.8, top_p=0.9)
    print("drawn answers: " + ", ".join("class %d" % c for c in drawn[:3].tolist()))
    for r in range(3):
        print("video %d: %s  entropy %.2f" % (r, ", ".join("class %d %.2f" % v for v in zip(best[r].tolist(), p[r].tolist())), float(entropy[r])))


if __name__ == "__main__":
    main(*sys.argv[1:2])

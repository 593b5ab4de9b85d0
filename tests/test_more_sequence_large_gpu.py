"""Decayed attention, group norm and token sampling on tensors of more than 2^31 elements: offsets past 32 bits.  What lies at their
ends is compared."""
import pytest
import torch

from tests import more_sequence_reference as more
from tests import sequence_reference as ref
from tests.test_decay_attention_gpu import EXTRA

pytestmark = pytest.mark.gpu
dcn = pytest.importorskip("deform_conv3d_pytorch_op_b200")


def fill(*shape):
    return torch.empty(shape, device="cuda", dtype=torch.bfloat16).normal_()


def wide(t):
    return t.detach().double().requires_grad_()


@pytest.mark.parametrize("heads,width", [(128, 128), (130, 127)], ids=["whole", "odd"])
def test_attention(heads, width):
    n, k, seen = 2 ** 17 + 70, 220, 100
    q, key, v = (fill(1, n, heads, width).requires_grad_() for _ in range(3))
    decay = torch.full((heads,), -1.0, device="cuda")         # what lies 120 steps back counts e^-120 of itself
    do = fill(1, n, heads, width)
    out, last = dcn.DecayAttentionFunction.apply(q, key, v, decay)
    got = torch.autograd.grad(out, (q, key, v), do)
    leaves = [wide(x[:, -k:]) for x in (q, key, v)]
    want, end = more.decay_attention(*leaves, decay.double())
    expected = torch.autograd.grad(want, leaves, do[:, -k:].double())
    chain = ref.CHAIN + EXTRA[torch.bfloat16]
    ref.close(last, end, "last", chain=ref.CHAIN + 2.0 ** -17)
    for a, b in zip((out,) + got, (want,) + expected):
        ref.close(a[:, -seen:], b[:, -seen:], chain=chain)


def test_steps():
    pool = torch.randn(8200, 16, 128, 128, device="cuda")
    slots = torch.tensor([8199, 0, 8195, 5], device="cuda")
    q, k, v = (fill(4, 16, 128) for _ in range(3))
    decay = -torch.rand(16, device="cuda")
    first = pool[slots]
    out = dcn.DecayAttentionFunction.step(q, k, v, decay, pool, slots)
    want, end = more.decay_attention_steps(*(x[:, None].double() for x in (q, k, v)), decay.double(), first.double())
    ref.close(out, want[:, 0])
    ref.close(pool[slots], end)


@pytest.mark.parametrize("samples,positions,channels,groups", [(9, 120001, 2000, 20), (35001, 30, 2048, 32)], ids=["long", "many"])
def test_group_norm(samples, positions, channels, groups):
    x, dy = fill(samples, positions, channels).requires_grad_(), fill(samples, positions, channels)
    weight = torch.randn(channels, device="cuda")
    y = dcn.GroupNormActFunction.apply(x, groups, weight, None, None, "silu")
    (dx,) = torch.autograd.grad(y, x, dy)
    w = wide(x[-1:])
    want = more.group_norm_act(w, groups, weight.double(), None, None, "silu")
    ref.close(y[-1:], want)
    ref.close(dx[-1:], torch.autograd.grad(want, w, dy[-1:].double())[0])


def test_tokens():
    n, v = 65600, 32771
    logits = fill(n, v)
    uniform = torch.rand(n, device="cuda")
    token, logprob = dcn.TokenSampleFunction.apply(logits, uniform, 0.9, 50, 0.9, 0.0)
    want, score = more.sample(logits[-3:], uniform[-3:], 0.9, 50, 0.9, 0.0)
    assert torch.equal(token[-3:], want)
    ref.close(logprob[-3:], score)


@pytest.mark.parametrize("vocab,skew", [(1 << 20, 0), (1 << 20, 3), ((1 << 20) - 100, 5), ((1 << 20) - 127, 1), ((1 << 20) - 4000, 0)])
def test_neighbouring_tokens_of_the_largest_vocabularies(vocab, skew):
    """So many rows that a CTA has one, and a thousand likely tokens side by side, where a CTA looks for the token among neighbours"""
    n, likely = 160, 1000
    g = torch.Generator(device="cuda").manual_seed(vocab + skew)
    logits = torch.full((n * (vocab + 8) + skew,), -60.0, device="cuda", dtype=torch.bfloat16)[skew:].view(n, vocab + 8)[:, :vocab]
    begins = torch.randint(0, vocab - likely, (n,), generator=g, device="cuda")
    begins[:4] = torch.tensor([0, vocab - likely, 1024, 512], device="cuda")
    places = begins[:, None] + torch.arange(likely, device="cuda")
    close = (torch.randn(n, likely, generator=g, device="cuda") * 0.3).bfloat16()
    logits.scatter_(1, places, close)
    uniform = torch.rand(n, generator=g, device="cuda")
    for settings in ((1.0, 0, 0.99, 0.0), (1.0, 900, 1.0, 0.0), (0.9, 700, 0.95, 0.0), (1.0, 0, 0.7, 0.0)):
        token, logprob = dcn.TokenSampleFunction.apply(logits, uniform, *settings)
        # (the others' weights are below 2^-40 of the largest: 0)
        want, score = more.sample(close, uniform, *settings)
        assert torch.equal(token, begins + want), settings
        ref.close(logprob, score)

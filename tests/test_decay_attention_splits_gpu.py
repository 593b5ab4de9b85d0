"""Decayed attention whose time axis is split: every gradient, of widths that are and are not multiples of 8, against the definition in
64 bits, and the same bits each time."""
import pytest
import torch

from tests import more_sequence_reference as more
from tests import sequence_reference as ref
from tests.test_decay_attention_gpu import EXTRA, STATE, make

pytestmark = pytest.mark.gpu
dcn = pytest.importorskip("deform_conv3d_pytorch_op_b200")

NAMES = ("q", "k", "v", "state")


def results(args, decay, lengths, dout, dlast, asked=NAMES):
    leaves = [x.detach().requires_grad_(n in asked) for n, x in zip(NAMES, args)]
    out, last = dcn.DecayAttentionFunction.apply(*leaves[:3], decay, leaves[3], lengths)
    return [out.detach(), last.detach()] + list(torch.autograd.grad((out, last), [x for x in leaves if x.requires_grad], (dout, dlast)))


def check(t, args, decay, lengths, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, _, v, state = args
    dout = torch.randn(q.shape[:3] + v.shape[3:], generator=g, device="cuda").to(t)
    dlast = torch.randn(state.shape, generator=g, device="cuda")
    got = results(args, decay, lengths, dout, dlast)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got, results(args, decay, lengths, dout, dlast)))
    wide = [x.detach().double().requires_grad_() for x in args]
    want, end = more.decay_attention_blocks(*wide[:3], decay.double(), wide[3], lengths)
    expected = [want, end] + list(torch.autograd.grad((want, end), wide, (dout.double(), dlast.double())))
    for name, a, b in zip(("out", "last", "dq", "dk", "dv", "dstate"), got, expected):
        ref.close(a, b, name, chain=ref.CHAIN + (STATE if name in ("last", "dstate") else EXTRA)[t])


@pytest.mark.parametrize("batch,steps,heads,dk,dv", [(1, 2050, 4, 33, 64), (1, 8192, 8, 20, 64), (1, 4096, 2, 100, 128), (2, 16384, 2, 107, 71),
                                                     (1, 4096, 4, 64, 33), (1, 3000, 4, 9, 121)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_parts_of_each_gradient(t, batch, steps, heads, dk, dv):
    """The parts' states are dk x dv in one gradient and dv x dk in others, with rows rounded up to 8: each gradient has its own place"""
    q, k, v, decay, state = make(t, batch, steps, heads, heads, dk, dv, seed=dk)
    check(t, (q, k, v, state), decay, None)
    lengths = torch.tensor([steps - 129, steps // 2 + 3], device="cuda")[:batch]
    check(t, (q, k, v, state), decay, lengths)
    if heads % 2 == 0:                              # heads that share keys and values: float32 gradients, summed
        q, k, v, decay, state = make(t, batch, steps, heads, heads // 2, dk, dv, seed=dv)
        check(t, (q, k, v, state), decay, lengths)


@pytest.mark.parametrize("dk,dv", [(40, 72), (33, 64), (128, 20)])
def test_parts_of_each_gradient_in_float32(dk, dv):
    q, k, v, decay, state = make(torch.float32, 1, 2050, 4, 2, dk, dv, seed=dk)
    check(torch.float32, (q, k, v, state), decay, torch.tensor([2000], device="cuda"))


@pytest.mark.parametrize("t,batch,steps,heads,dk,dv", [
    (torch.float32, 16, 331, 5, 40, 72), (torch.float32, 16, 777, 6, 128, 64), (torch.float32, 30, 400, 5, 33, 65),
    (torch.bfloat16, 6, 2100, 16, 64, 128), (torch.bfloat16, 6, 2100, 16, 128, 64), (torch.float16, 10, 1500, 10, 121, 50),
    (torch.bfloat16, 25, 1200, 6, 24, 104)])
def test_some_gradients_alone(t, batch, steps, heads, dk, dv):
    """Gradients whose own columns are 64 or fewer where the other width is more: as many heads as fill the GPU only with the wider one"""
    q, k, v, decay, state = make(t, batch, steps, heads, heads, dk, dv, seed=steps)
    g = torch.Generator(device="cuda").manual_seed(2)
    dout = torch.randn(batch, steps, heads, dv, generator=g, device="cuda").to(t)
    dlast = torch.randn(state.shape, generator=g, device="cuda")
    wide = [x.detach().double().requires_grad_() for x in (q, k, v, state)]
    want, end = more.decay_attention_blocks(*wide[:3], decay.double(), wide[3])
    expected = dict(zip(NAMES, torch.autograd.grad((want, end), wide, (dout.double(), dlast.double()))))
    for asked in (("q",), ("k",), ("q", "k"), ("v",), ("state",), ("v", "state"), ("k", "v"), NAMES):
        got = results((q, k, v, state), decay, None, dout, dlast, asked)[2:]
        for name, a in zip(asked, got):
            ref.close(a, expected[name], (asked, name), chain=ref.CHAIN + (STATE if name == "state" else EXTRA)[t])

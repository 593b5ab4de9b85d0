"""The sequence operators on tensors of more than 2^31 elements: offsets past 32 bits.  The last rows are compared."""
import pytest
import torch

from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu
dcn = pytest.importorskip("deform_conv3d_pytorch_op_b200")


def fill(*shape):
    return torch.empty(shape, device="cuda", dtype=torch.bfloat16).normal_()


def wide(t):
    return t.detach().double().requires_grad_()


def test_norm():
    n, c = 2 ** 18 + 5, 8192
    x, block, ds = fill(n, c).requires_grad_(), fill(n, c).requires_grad_(), fill(n, c)
    stream, normed = dcn.ResidualNormFunction.apply(x, block)
    got = torch.autograd.grad((stream, normed), (x, block), (ds, ds))
    wx, wb = wide(x[-3:]), wide(block[-3:])
    wants = ref.residual_norm(wx, wb)
    want = torch.autograd.grad(wants, (wx, wb), (ds[-3:].double(),) * 2)
    for a, b in zip((stream, normed) + got, wants + want):
        ref.close(a[-3:], b)


def test_logits():
    n, v = 65600, 32771
    logits = fill(n, v).requires_grad_()
    tokens = torch.full((n,), v - 1, device="cuda")
    outs = dcn.TokenScoresFunction.apply(logits, tokens, 3)
    (got,) = torch.autograd.grad(outs[0].sum() + outs[1].sum(), logits)
    w = wide(logits[-3:])
    wants = ref.token_scores(w, tokens[-3:], 3)
    (want,) = torch.autograd.grad(wants[0].sum() + wants[1].sum(), w)
    for a, b in zip(outs[:3], wants):
        ref.close(a[-3:], b)
    assert torch.equal(outs[3][-3:], wants[3])
    ref.close(got[-3:], want)
    del got, outs
    places = torch.arange(5, device="cuda").expand(n, 5).contiguous()
    lq = torch.full((n, 5), -2.0, device="cuda")
    loss = dcn.DistillTopkFunction.apply(logits, lq, places)
    (got,) = torch.autograd.grad(loss.sum(), logits)
    want = ref.distill(w, lq[-3:].double(), places[-3:])
    ref.close(loss[-3:], want)
    (want,) = torch.autograd.grad(want.sum(), w)
    ref.close(got[-3:], want)


def test_scan():
    n, c, k = 2 ** 20 + 70, 2050, 150
    x, gate, dy = fill(1, n, c), fill(1, n, c), fill(1, n, c)
    gate[:, -k] = -100.0                                      # what follows owes nothing to the steps before
    x.requires_grad_(), gate.requires_grad_()
    y, last = dcn.GatedScanFunction.apply(x, gate)
    dx, dgate = torch.autograd.grad(y, (x, gate), dy)
    wx, wg = wide(x[:, -k:]), wide(gate[:, -k:])
    wy, wl = ref.scan(wx, wg)
    ref.close(y[:, -k:], wy)
    ref.close(last, wl)
    for a, b in zip((dx, dgate), torch.autograd.grad(wy, (wx, wg), dy[:, -k:].double())):
        ref.close(a[:, -k + 1:], b[:, 1:])

"""Decayed attention in float16 where numbers lie far from one: scores and gradients' products above its largest number, states, values
and gradients below its normal ones.  What is rounded is rounded relative to its row, its head's state or its block, by powers of two."""
import ctypes

import pytest
import torch

from tests import more_sequence_reference as more
from tests import sequence_reference as ref
from tests.test_decay_attention_gpu import EXTRA, STATE, make

pytestmark = pytest.mark.gpu
dcn = pytest.importorskip("deform_conv3d_pytorch_op_b200")
from deform_conv3d_pytorch_op_b200 import _lib  # noqa: E402

F16 = torch.float16
NAMES = ("out", "last", "dq", "dk", "dv", "dstate")
# steps, offset of the results in memory: the small kernel (part of a block of steps, one, several: results off 16 bytes), tensor cores
WAYS = [(40, 0), (64, 0), (300, 1), (200, 0), (700, 0)]


def off_16_bytes(args, decay, lengths, do, dl):
    """All results by the C calls, each 2 (4) bytes behind 16: so the kernel without tensor memory runs through several blocks"""
    q, k, v, state = args
    p = _lib.dcn_attn(dtype=2, batch=q.size(0), steps=q.size(1), heads=q.size(2), kv_heads=k.size(2), dk=q.size(3), dv=v.size(3), scale=q.size(3) ** -0.5)
    for n, x in (("q", q), ("k", k), ("v", v), ("dout", do)):
        for i, a in enumerate(("batch", "step", "head")):
            setattr(p, "%s_%s" % (n, a), x.stride(i))
    L, at = _lib.lib(), ctypes.byref(p)
    ws = [torch.empty(max(L.dcn_attn_workspace_bytes(at, i), 16), dtype=torch.uint8, device="cuda") for i in range(2)]
    dense = [do, state, q, k, v, state]                     # the results' shapes
    got = [torch.empty(x.numel() + 8, dtype=x.dtype, device="cuda")[1:1 + x.numel()].view(x.shape) for x in dense]
    lengths = 0 if lengths is None else lengths.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    ins = [x.data_ptr() for x in (q, k, v, decay, state)] + [lengths]
    outs = [x.data_ptr() for x in got]
    assert all(x % 16 for x in outs)
    assert L.dcn_attn_forward(at, *ins, *outs[:2], ws[0].data_ptr(), ws[0].numel(), stream) == 0
    assert L.dcn_attn_backward(at, *ins, do.data_ptr(), dl.data_ptr(), *outs[2:], ws[1].data_ptr(), ws[1].numel(), stream) == 0
    torch.cuda.synchronize()
    return got


def run(steps, offset, dk, dv, q=1.0, k=1.0, v=1.0, state=1.0, dout=1.0, dlast=1.0, only=NAMES, lengths=None, kv=2):
    """All results with operands of these sizes.  Bounds: those of the operator's other tests, which count roundings relative to what is
    rounded, and so hold at any size that the types have."""
    a = make(F16, 2, steps, 2, kv, dk, dv, seed=steps + dk)
    g = torch.Generator(device="cuda").manual_seed(3)
    args = [x * s for x, s in zip((a[0], a[1], a[2], a[4]), (q, k, v, state))]
    wide = [x.detach().double().requires_grad_() for x in args]
    do = torch.randn(2, steps, 2, dv, generator=g, device="cuda").mul_(dout).to(F16)
    dl = torch.randn(2, 2, dk, dv, generator=g, device="cuda") * dlast
    want, end = more.decay_attention(*wide[:3], a[3].double(), wide[3], lengths)
    if offset:
        got = off_16_bytes(args, a[3], lengths, do, dl)
    else:
        leaves = [x.detach().requires_grad_() for x in args]
        out, last = dcn.DecayAttentionFunction.apply(*leaves[:3], a[3], leaves[3], lengths)
        got = [out, last] + list(torch.autograd.grad((out, last), leaves, (do, dl)))
    expected = [want, end] + list(torch.autograd.grad((want, end), wide, (do.double(), dl.double())))
    for name, x, y in zip(NAMES, got, expected):
        if name in only:
            ref.close(x, y, name, chain=ref.CHAIN + (STATE if name in ("last", "dstate") else EXTRA)[F16])
    return expected


@pytest.mark.parametrize("steps,offset", WAYS)
@pytest.mark.parametrize("dk,dv", [(128, 64), (64, 64), (128, 128)])
def test_scores_above_the_largest_number(steps, offset, dk, dv):
    # q . k of some 64^2 * sqrt(dk) and more, where scale q . k v is some thousand times v
    e = run(steps, offset, dk, dv, q=64.0, k=64.0, v=0.1, state=10.0, dout=0.01, only=("out", "last"))
    assert 1000 < float(e[0].detach().abs().max()) < 65504


@pytest.mark.parametrize("steps,offset", WAYS)
@pytest.mark.parametrize("kv", [1, 2])
def test_gradients_of_a_scaled_loss(steps, offset, kv):
    # dout . v of 200 * 30 * sqrt(128) = 68000 in a third of all pairs, up to 300000.  Their sums stay in range: dk is 68000 / 8 * 0.05 times
    # the root of the steps that a state lasts, 125 (and of two heads): 6700, and five times that in the largest of 10^5 elements
    e = run(steps, offset, 64, 128, q=0.05, k=0.02, v=30.0, dout=200.0, dlast=10.0, kv=kv, state=0.1)
    assert all(float(x.abs().max()) < 65504 for x in e[2:5])


def test_scores_of_equal_rows():
    """q = k = 32 in 128 columns: the score is 131072, and out 11585 v"""
    for steps in (1, 20, 70):
        q = torch.full((1, steps, 1, 128), 32.0, device="cuda", dtype=F16)
        v = torch.randn(1, steps, 1, 64, device="cuda").to(F16)
        out, _ = dcn.DecayAttentionFunction.apply(q, q, v, torch.full((1,), -20.0, device="cuda"))
        ref.close(out, 131072 / 128 ** 0.5 * v.double(), chain=ref.CHAIN + EXTRA[F16] + 2 * 2.0 ** -28)


@pytest.mark.parametrize("steps,offset", WAYS)
@pytest.mark.parametrize("size", [0.02, 1e-3, 1e-4, 4e-6])
def test_states_of_small_values(steps, offset, size):
    """last and dstate are float32: as exact for small values, keys, queries and gradients as for large ones"""
    run(steps, offset, 48, 72, v=size, state=size, dout=size, dlast=size, only=("last", "dstate"))
    run(steps, offset, 48, 72, q=size, k=size, state=size, dlast=size, only=("last", "dstate"))
    run(steps, offset, 48, 72, v=size, dout=size, only=("last", "dstate"), lengths=torch.tensor([steps, steps // 2 + 1], device="cuda"))


@pytest.mark.parametrize("steps,offset", WAYS)
def test_results_of_small_products(steps, offset):
    """Scores, and products dout . v, below the type's normal numbers, that large operands bring back"""
    run(steps, offset, 64, 64, q=3e-3, k=3e-3, v=300.0, state=1e-3, only=("out",))
    run(steps, offset, 64, 64, q=100.0, k=100.0, v=1e-3, dout=1e-4, dlast=1e-4, state=1e-3, only=("dq", "dk"))
    # and states
    run(steps, offset, 64, 64, q=200.0, k=1e-3, v=1e-3, state=1e-5, only=("out",))


@pytest.mark.parametrize("steps,offset", WAYS)
def test_columns_beside_infinite_ones(steps, offset):
    """An infinite column of the state leaves the others as they are"""
    q, k, v, decay, state = make(F16, 1, steps, 1, 1, 32, 40, seed=steps)
    bad = state.clone()
    bad[..., 7] = float("inf")
    want, end = dcn.DecayAttentionFunction.apply(q, k, v, decay, state)
    out, last = dcn.DecayAttentionFunction.apply(q, k, v, decay, bad)
    others = [c for c in range(40) if c != 7]
    assert torch.equal(out[..., others], want[..., others]) and torch.equal(last[..., others], end[..., others])
    assert not bool(torch.isfinite(last[..., 7]).any())


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_parts_of_wider_rows(t):
    """Operands that begin off 16 bytes with strides that are on them: the values of dense ones, bit for bit"""
    row = torch.randn(2, 300, 2, 136, device="cuda").to(t)
    q, k, v = (row[..., i:i + 40] for i in (1, 42, 91))
    decay, state = torch.tensor([-0.01, -0.2], device="cuda"), torch.randn(2, 2, 40, 40, device="cuda")
    leaves, dense = ([x.detach().requires_grad_() for x in y] for y in ((q, k, v), (x.contiguous() for x in (q, k, v))))
    wide = torch.randn(2, 300, 2, 48, device="cuda").to(t)
    do = wide[..., 3:43]
    got, want = ((lambda o: [o[0], o[1]] + list(torch.autograd.grad(o, x, (g, torch.ones_like(state)))))(
        dcn.DecayAttentionFunction.apply(*x, decay, state)) for x, g in ((leaves, do), (dense, do.contiguous())))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("heads", [6, 300])
@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_states_that_last(t, heads):
    """What is left of a first state and of a last one's gradient after 40000 steps, block by block: the decay of a block is rounded to
    float32, but its roundings do not add up from block to block"""
    steps, w = 40003, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    decay = -torch.logspace(-6, -3.7, heads, device="cuda")
    q, k, v = (torch.zeros(1, steps, heads, w, device="cuda", dtype=t).requires_grad_() for _ in range(3))
    state = torch.randn(1, heads, w, w, generator=g, device="cuda").requires_grad_()
    dl = torch.randn(1, heads, w, w, generator=g, device="cuda")
    left = torch.exp(decay.double() * steps).view(1, heads, 1, 1)
    out, last = dcn.DecayAttentionFunction.apply(q, k, v, decay, state)
    (dstate,) = torch.autograd.grad(last, state, dl)
    assert float(out.detach().abs().max()) == 0
    # each head by itself: 626 blocks' (313 on tensor cores) products, each rounded to half a step: 2^-25 sqrt(626) and less
    for h in range(heads):
        ref.close(last[:, h], (left * state.double())[:, h], ("last", h))
        ref.close(dstate[:, h], (left * dl.double())[:, h], ("dstate", h))


def test_states_that_last_step_by_step():
    """The same of 4000 single steps: half a step of float32 each, not the decay's rounding 4000 times"""
    heads, steps = 200, 4000
    decay = -torch.logspace(-5, -3, heads, device="cuda")
    zero = torch.zeros(1, heads, 4, device="cuda")
    pool = torch.randn(1, heads, 4, 4, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    want = torch.exp(decay.double() * steps).view(1, heads, 1, 1) * pool.double()
    for _ in range(steps):
        dcn.DecayAttentionFunction.step(zero, zero, zero, decay, pool)
    for h in range(heads):
        ref.close(pool[:, h], want[:, h], h)


@pytest.mark.parametrize("steps,offset", WAYS + [(1, 0)])
def test_strong_decays(steps, offset):
    """Back in time even the first step's weight is the decay itself: what little of it reaches the first state is exact"""
    a = make(F16, 2, steps, 4, 4, 40, 64, seed=steps)
    decay = torch.tensor([-4.0, -12.0, -25.0, -60.0], device="cuda")
    do = torch.randn(2, steps, 4, 64, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(F16)
    args = (a[0], a[1], a[2], a[4])
    wide = [x.detach().double().requires_grad_() for x in args]
    want, end = more.decay_attention(*wide[:3], decay.double(), wide[3])
    expected = torch.autograd.grad(want, wide[3], do.double())[0]
    if offset:
        got = off_16_bytes(args, decay, None, do, torch.zeros_like(a[4]))[5]
    else:
        leaf = a[4].detach().requires_grad_()
        out, _ = dcn.DecayAttentionFunction.apply(*args[:3], decay, leaf)
        got = torch.autograd.grad(out, leaf, do)[0]
    for h in range(4):
        ref.close(got[:, h], expected[:, h], h, chain=ref.CHAIN + STATE[F16])


def test_infinite_states_step_by_step():
    pool = torch.randn(3, 2, 8, 8, device="cuda")
    pool[1, 0, 3, 4], pool[2, 1, 0, 0], pool[0, 0, 7, 7] = float("inf"), float("-inf"), 3.4e38
    q, k, v = (torch.randn(3, 2, 8, device="cuda") for _ in range(3))
    for log_decay in (0.0, -0.3, -1e-4):
        want = torch.exp(torch.tensor(log_decay).double()) * pool.double() + k.double()[..., None] * v.double()[..., None, :]
        dcn.DecayAttentionFunction.step(q, k, v, torch.full((2,), log_decay, device="cuda"), pool)
        ref.close(pool, want, log_decay)
    zero, large = torch.zeros(1, 1, 4, device="cuda"), torch.full((1, 1, 4, 4), 3e35, device="cuda")
    dcn.DecayAttentionFunction.step(zero, zero, zero, torch.full((1,), -float("inf"), device="cuda"), large)
    assert float(large.abs().max()) == 0                    # none of the past at all

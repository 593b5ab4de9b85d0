"""Decayed attention against its definition in 64 bits."""
import math

import pytest
import torch

from tests import more_sequence_reference as more
from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu

# What is rounded to a 16-bit type on the way: the weights of a block's steps and the state that a step meets, each by at most half a
# step of the type and independently of one another, so that the error's 2-norm stays below two of them.  Float32 results (states and
# their gradients) come from products of a rounded factor and of what its rounding left: 2^-9 of 2^-9 remains in bfloat16.
EXTRA = {torch.float32: 0.0, torch.bfloat16: 2 * 2.0 ** -8, torch.float16: 2 * 2.0 ** -11}
STATE = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -17, torch.float16: 2.0 ** -22}


def make(t, batch, steps, heads, kv, dk, dv, seed=0, offset=0, std=1.0):
    """q, k, v as parts of one projection that starts `offset` elements into its memory."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = heads * dk + kv * (dk + dv)
    flat = torch.randn(batch * steps * width + offset, generator=g, device="cuda").mul_(std).to(t)[offset:]
    q, k, v = flat.view(batch, steps, width).split((heads * dk, kv * dk, kv * dv), -1)
    decay = -torch.rand(heads, generator=g, device="cuda") * 0.3
    decay[0] = -0.004
    state = torch.randn(batch, heads, dk, dv, generator=g, device="cuda")
    return q.unflatten(-1, (heads, dk)), k.unflatten(-1, (kv, dk)), v.unflatten(-1, (kv, dv)), decay, state


def check(t, q, k, v, decay, state, lengths, scale=None, grads=True, seed=1):
    import deform_conv3d_pytorch_op_b200 as dcn
    leaves = [x.detach().requires_grad_(grads) if x is not None else None for x in (q, k, v, state)]
    out, last = dcn.DecayAttentionFunction.apply(*leaves[:3], decay, leaves[3], lengths, scale)
    wide = [x.detach().double().requires_grad_() if x is not None else None for x in (q, k, v, state)]
    want, end = more.decay_attention(*wide[:3], decay.double(), wide[3], lengths, scale)
    ref.close(out, want, "out", chain=ref.CHAIN + EXTRA[t])
    ref.close(last, end, "last", chain=ref.CHAIN + STATE[t])
    if not grads:
        return
    g = torch.Generator(device="cuda").manual_seed(seed)
    do = torch.randn(out.shape, generator=g, device="cuda").to(t)
    dl = torch.randn(last.shape, generator=g, device="cuda")
    asked = [x for x in leaves if x is not None]
    got = torch.autograd.grad((out, last), asked, (do, dl))
    expected = torch.autograd.grad((want, end), [x for x in wide if x is not None], (do.double(), dl.double()))
    for name, a, b in zip(("dq", "dk", "dv", "dstate"), got, expected):
        extra = STATE[t] if name == "dstate" else EXTRA[t]
        ref.close(a, b, name, chain=ref.CHAIN + extra)


@pytest.mark.parametrize("steps", [1, 2, 15, 16, 17, 63, 64, 65, 130, 331])
@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_lengths_of_time(t, steps):
    q, k, v, decay, state = make(t, 2, steps, 3, 3, 32, 48, seed=steps)
    check(t, q, k, v, decay, state, None)


@pytest.mark.parametrize("dk,dv", [(1, 1), (7, 5), (8, 64), (40, 72), (64, 64), (65, 33), (100, 20), (128, 128), (33, 127)])
@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_widths(t, dk, dv):
    q, k, v, decay, state = make(t, 2, 150, 2, 1, dk, dv, seed=dk)
    check(t, q, k, v, decay, state, torch.tensor([150, 77], device="cuda"))


@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_alignments(t, offset):
    q, k, v, decay, state = make(t, 2, 70, 2, 2, 24, 20, seed=offset, offset=offset)
    check(t, q, k, v, decay, state, None)


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (6, 2), (8, 8), (5, 5)])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_heads_that_share(t, heads, kv):
    q, k, v, decay, state = make(t, 2, 100, heads, kv, 32, 32, seed=heads)
    check(t, q, k, v, decay, state, None)


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_parts_of_a_long_axis(t):
    """Few heads: the time axis is split, sequences end before, at and behind the parts' borders"""
    for steps in (1000, 1024, 2050):
        q, k, v, decay, state = make(t, 3, steps, 1, 1, 64, 40, seed=steps)
        check(t, q, k, v, decay, state, torch.tensor([steps, 512, steps - 65], device="cuda"))
    q, k, v, decay, state = make(t, 1, 1025, 1, 1, 128, 128, seed=9)
    check(t, q, k, v, decay, state, None)


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_padded_batches(t):
    """What lies behind a sequence is not read; lengths beyond the axis are cut, of any whole type"""
    q, k, v, decay, state = make(t, 6, 130, 2, 2, 32, 32, seed=5)
    lengths = torch.tensor([0, 1, 64, 129, 500, -3], device="cuda", dtype=torch.int32)
    check(t, q, k, v, decay, state, lengths)
    import deform_conv3d_pytorch_op_b200 as dcn
    behind = torch.arange(130, device="cuda")[None, :] >= lengths[:, None]
    clean = dcn.DecayAttentionFunction.apply(q, k, v, decay, state, lengths)
    bad = [torch.where(behind[..., None, None], float("nan"), x) for x in (q, k, v)]
    leaves = [x.requires_grad_() for x in bad]
    out, last = dcn.DecayAttentionFunction.apply(*leaves, decay, state, lengths)
    assert torch.equal(out, clean[0]) and torch.equal(last, clean[1])
    assert bool((out[behind] == 0).all())
    dout = torch.where(behind[..., None, None], float("nan"), torch.randn_like(out.float())).to(t)
    for name, x in zip("qkv", torch.autograd.grad(out, leaves, dout)):
        assert bool(torch.isfinite(x).all()) and bool((x[behind] == 0).all()), name


@pytest.mark.parametrize("heads,kv,dk,dv", [(4, 4, 107, 71), (4, 2, 33, 64), (3, 1, 64, 33), (2, 2, 12, 20)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_rows_that_are_laid_out_anew(t, heads, kv, dk, dv):
    """Odd widths, strides and places in memory, operands that are broadcast: with padding that is not read, whatever memory holds"""
    import deform_conv3d_pytorch_op_b200 as dcn
    q, k, v, decay, state = make(t, 5, 300, heads, kv, dk, dv, seed=dv, offset=1)
    lengths = torch.tensor([300, 0, 129, 1, 128], device="cuda")
    check(t, q, k, v, decay, state, lengths)
    check(t, q, k[:1].expand(5, -1, -1, -1), v[:, :, :1].expand(-1, -1, kv, -1), decay, state, lengths)
    want = dcn.DecayAttentionFunction.apply(q, k, v, decay, state, lengths)
    behind = torch.arange(300, device="cuda")[None, :] >= lengths[:, None]
    bad = [torch.where(behind[..., None, None], float("nan"), x).requires_grad_() for x in (q, k, v)]
    trash = torch.full((1 << 24,), float("nan"), device="cuda")       # what the allocator gives next
    del trash
    out, last = dcn.DecayAttentionFunction.apply(*bad, decay, state, lengths)
    assert torch.equal(out, want[0]) and torch.equal(last, want[1])
    for x in torch.autograd.grad((out, last), bad, (torch.ones_like(out), torch.ones_like(last))):
        assert bool(torch.isfinite(x).all()) and bool((x[behind] == 0).all())
    # any order of axes, and steps that lie on one another's
    turned = [x.permute(0, 3, 2, 1).contiguous().permute(0, 3, 2, 1) for x in (q, k, v)]
    again = dcn.DecayAttentionFunction.apply(*turned, decay, state, lengths)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_no_state_and_single_gradients():
    import deform_conv3d_pytorch_op_b200 as dcn
    q, k, v, decay, state = make(torch.float32, 2, 90, 2, 2, 16, 24, seed=3)
    check(torch.float32, q, k, v, decay, None, None)
    wide = [x.detach().double().requires_grad_() for x in (q, k, v, state)]
    want, end = more.decay_attention(*wide[:3], decay.double(), wide[3])
    do, dl = torch.randn_like(want), torch.randn_like(end)
    for which in range(4):                          # one gradient at a time, from one output at a time
        for out_of in range(2):
            leaves = [x.detach().requires_grad_(i == which) for i, x in enumerate((q, k, v, state))]
            got = dcn.DecayAttentionFunction.apply(*leaves[:3], decay, leaves[3])[out_of]
            if which == 0 and out_of == 1:
                assert float(torch.autograd.grad(got, leaves[0], dl.float())[0].abs().max()) == 0
                continue
            a = torch.autograd.grad(got, leaves[which], (do, dl)[out_of].float())[0]
            b = torch.autograd.grad((want, end)[out_of], wide[which], (do, dl)[out_of], retain_graph=True)[0]
            ref.close(a, b, (which, out_of))


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_decays(t):
    """No decay at all, numbers above 0 (taken as 0), decays that leave nothing, and none of the past at all"""
    import deform_conv3d_pytorch_op_b200 as dcn
    q, k, v, decay, state = make(t, 1, 200, 6, 6, 16, 16, seed=8)
    decay = torch.tensor([0.0, 0.5, -1e-6, -8.0, -300.0, -math.inf], device="cuda")
    check(t, q, k, v, decay, state, None)
    out, last = dcn.DecayAttentionFunction.apply(q, k, v, torch.full_like(decay, math.nan), state)
    assert bool(torch.isnan(last).all())


def test_differences():
    """The gradient against differences of the operator's own loss"""
    import deform_conv3d_pytorch_op_b200 as dcn
    q, k, v, decay, state = make(torch.float32, 1, 40, 2, 1, 8, 6, seed=2)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v, state)]
    weight = torch.randn(1, 40, 2, 6, device="cuda", dtype=torch.float64)

    def loss(args):
        out, last = dcn.DecayAttentionFunction.apply(*args[:3], decay, args[3], torch.tensor([33], device="cuda"))
        return (out.double() * weight).sum() + last.double().square().sum() / 2

    grads = torch.autograd.grad(loss(leaves), leaves)
    for i, x in enumerate(leaves):
        way = torch.randn_like(x)
        h = 1e-2
        with torch.no_grad():
            up, down = (loss([y + s * h * way if j == i else y for j, y in enumerate(leaves)]) for s in (1, -1))
        # quadratic in each argument but for k and v in last, where the third difference is zero too: what is left are roundings,
        # 2^-24 of the loss's terms over the step
        size = float((weight.abs().sum() + leaves[3].detach().square().sum()) * 40)
        assert abs(float((up - down) / (2 * h)) - float((grads[i] * way).sum())) <= 64 * 2.0 ** -24 * size / h


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
@pytest.mark.parametrize("heads,kv,dk,dv", [(2, 2, 64, 64), (4, 2, 128, 128), (3, 1, 40, 72), (1, 1, 5, 7), (2, 2, 128, 1)])
def test_single_steps(t, heads, kv, dk, dv):
    import deform_conv3d_pytorch_op_b200 as dcn
    q, k, v, decay, _ = make(t, 5, 9, heads, kv, dk, dv, seed=dk + dv)
    pool = torch.randn(8, heads, dk, dv, device="cuda")
    slots = torch.tensor([6, 0, 3, 7, 2], device="cuda")
    first = pool.clone()
    out = torch.stack([dcn.DecayAttentionFunction.step(q[:, i], k[:, i], v[:, i], decay, pool, slots) for i in range(9)], 1)
    want, end = more.decay_attention_steps(q.double(), k.double(), v.double(), decay, first[slots].double())
    ref.close(out, want, "out")
    ref.close(pool[slots], end, "states")
    others = [1, 4, 5]
    assert torch.equal(pool[others], first[others])
    whole, last = dcn.DecayAttentionFunction.apply(q, k, v, decay, first[slots])
    ref.close(whole, want, "whole", chain=ref.CHAIN + EXTRA[t])
    ref.close(last, end, "last", chain=ref.CHAIN + STATE[t])


def test_slots_outside_the_pool():
    import deform_conv3d_pytorch_op_b200 as dcn
    q, k, v, decay, _ = make(torch.float32, 3, 1, 2, 2, 16, 16, seed=1)
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    pool = torch.randn(4, 2, 16, 16, device="cuda")
    first = pool.clone()
    out = dcn.DecayAttentionFunction.step(q, k, v, decay, pool, torch.tensor([9, 2, -1], device="cuda", dtype=torch.int32))
    assert float(out[[0, 2]].abs().max()) == 0 and torch.equal(pool[[0, 1, 3]], first[[0, 1, 3]])
    assert not torch.equal(pool[2], first[2])
    dcn.DecayAttentionFunction.step(q, k, v, decay, pool)          # rows 0, 1, 2
    assert torch.equal(pool[3], first[3]) and not torch.equal(pool[0], first[0])


def test_float16_states_beyond_its_range():
    """A state of which float16 holds no copy meets small queries: it is scaled by a power of two on the way"""
    import deform_conv3d_pytorch_op_b200 as dcn
    t = torch.float16
    q, k, v, decay, state = make(t, 1, 200, 2, 2, 32, 32, seed=4)
    q, state = q * 1e-3, state * 3e5
    check(t, q, k, v, decay, state, None, grads=False)
    huge = state * 1e32
    out, last = dcn.DecayAttentionFunction.apply(q, k, v, decay, huge)
    assert not bool(torch.isnan(out).any()) and bool(torch.isfinite(last).all())


def test_heads_before_steps():
    """[batch, heads, steps, width] in memory, and axes of one stride"""
    q, k, v, decay, state = make(torch.bfloat16, 2, 80, 4, 4, 32, 32, seed=6)
    check(torch.bfloat16, *(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)), decay, state, None)
    one = k[:, :1].expand(-1, 80, -1, -1)
    check(torch.bfloat16, q, one, v.transpose(2, 3).contiguous().transpose(2, 3), decay, state, None)


def test_empty():
    import deform_conv3d_pytorch_op_b200 as dcn
    q, k, v, decay, state = make(torch.float32, 2, 4, 2, 2, 8, 8)
    leaves = [x[:, :0].detach().requires_grad_() for x in (q, k, v)] + [state.detach().requires_grad_()]
    out, last = dcn.DecayAttentionFunction.apply(*leaves[:3], decay, leaves[3])
    assert out.shape == (2, 0, 2, 8) and torch.equal(last, state)
    dl = torch.randn_like(last)
    ref.close(torch.autograd.grad(last, leaves[3], dl)[0], dl.double(), "dstate")
    out, last = dcn.DecayAttentionFunction.apply(q[:0], k[:0], v[:0], decay)
    assert out.shape == (0, 4, 2, 8) and last.shape == (0, 2, 8, 8)
    assert dcn.DecayAttentionFunction.step(q[:0, 0], k[:0, 0], v[:0, 0], decay, state).shape == (0, 2, 8)


def test_refusals():
    import deform_conv3d_pytorch_op_b200 as dcn
    apply, step = dcn.DecayAttentionFunction.apply, dcn.DecayAttentionFunction.step
    q, k, v, decay, state = make(torch.float32, 2, 4, 4, 2, 8, 8)
    for args, text in [((q[0], k, v, decay), "expected \\(batch, steps"), ((q, k[:, :3], v, decay), "k has shape"),
                       ((q, k, v.half(), decay), "v has dtype"), ((q, k, v, decay.double()), "log_decay has dtype"),
                       ((q, k, v, decay[:2]), "log_decay has shape"), ((q[:, :, :3], k, v, decay[:3]), "do not divide"),
                       ((q, k, v, decay, state[:1]), "state has shape"), ((q, k, v, decay, state.half()), "state has dtype"),
                       ((q, k, v, decay, None, torch.zeros(3, device="cuda", dtype=torch.long)), "lengths has shape"),
                       ((q, k, v, decay, None, torch.zeros(2, device="cuda")), "int64 or int32"),
                       ((q, k, v, decay, None, None, 0.0), "scale"), ((q, k, v, decay, None, None, math.nan), "scale"),
                       ((q, k, v, decay.clone().requires_grad_()), "no gradient"), ((q.cpu(), k, v, decay), "CUDA"),
                       ((q, k, v, decay.cpu()), "CUDA")]:
        with pytest.raises(dcn.DcnError, match=text):
            apply(*args)
    wide = torch.zeros(1, 2, 1, 129, device="cuda")
    with pytest.raises(dcn.DcnError, match="1 to 128"):
        apply(wide, wide, wide, decay[:1])
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    for args, text in [((q, k, v, decay, state[:, :, :, :4]), "state has shape"), ((q, k, v, decay, state[:1]), "fewer rows"),
                       ((q, k, v, decay, state.clone().requires_grad_()), "no gradient"),
                       ((q, k, v, decay, state, torch.zeros(3, device="cuda", dtype=torch.long)), "slots has shape")]:
        with pytest.raises(dcn.DcnError, match=text):
            step(*args)
    x = torch.randn(1, 3, 1, 4, device="cuda", requires_grad=True)
    out, _ = apply(x, x, x, decay[:1])
    got = torch.autograd.grad(out, x, torch.ones_like(out).requires_grad_(), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got.sum().backward()


def test_captured_and_on_other_streams():
    import deform_conv3d_pytorch_op_b200 as dcn
    q, k, v, decay, state = make(torch.bfloat16, 1, 700, 2, 1, 64, 64, seed=7)
    do = torch.randn(1, 700, 2, 64, device="cuda").bfloat16()

    def run(q, k, v, state):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, state)]
        out, last = dcn.DecayAttentionFunction.apply(*leaves[:3], decay, leaves[3])
        return (out.detach(), last.detach()) + torch.autograd.grad((out, last), leaves, (do, torch.ones_like(last)))

    want = run(q, k, v, state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(q, k, v, state)
        run(q, k, v, state)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    held = [x.clone() for x in (q, k, v, state)]
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(run(*held))
    for x in held[:3]:
        x.mul_(0.5)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = run(*held)
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))

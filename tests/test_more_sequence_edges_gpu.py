"""Decayed attention, group norm and token sampling in autograd, traces, transforms, threads and modules of 16 bits."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from tests.test_decay_attention_gpu import make

pytestmark = pytest.mark.gpu
dcn = pytest.importorskip("deform_conv3d_pytorch_op_b200")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def attention():
    q, k, v, decay, state = make(torch.bfloat16, 2, 90, 4, 2, 24, 17, seed=3)
    lengths = torch.tensor([90, 71], device="cuda")
    return lambda q, k, v, state: dcn.DecayAttentionFunction.apply(q, k, v, decay, state, lengths), [q, k, v, state]


def group_norm():
    g = gen(4)
    x, res, w, b = randn(g, 3, 50, 24), randn(g, 3, 50, 24), randn(g, 24), randn(g, 24)
    return lambda x, w, b, res: (dcn.GroupNormActFunction.apply(x, 4, w, b, res, "silu"),), [x, w, b, res]


CALLS = {"attention": attention, "group norm": group_norm}


@pytest.mark.parametrize("name", list(CALLS))
def test_place_in_autograd(name):
    fn, args = CALLS[name]()
    leaves = [a.detach().clone().requires_grad_() for a in args]
    total = sum(o.sum() for o in fn(*leaves))
    first = torch.autograd.grad(total, leaves, retain_graph=True)
    for i, leaf in enumerate(leaves):                         # some gradients only
        (one,) = torch.autograd.grad(total, leaf, retain_graph=True)
        assert torch.equal(one, first[i])
    again = torch.autograd.grad(total, leaves)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(total, leaves)
    outs = fn(*leaves)
    with torch.no_grad():
        leaves[0].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(sum(o.sum() for o in outs), leaves)
    traced = torch.jit.trace(lambda *a: tuple(fn(*a)), tuple(a.detach() for a in args), check_trace=False)
    other = [(a.detach() * 0.5).requires_grad_() for a in args]
    t, w = traced(*other), fn(*other)
    t = t if isinstance(t, tuple) else (t,)
    assert all(torch.equal(a, b) for a, b in zip(t, w))
    for a, b in zip(torch.autograd.grad(sum(o.sum() for o in t), other), torch.autograd.grad(sum(o.sum() for o in w), other)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: sum(o.sum() for o in fn(v, *[a.detach() for a in args[1:]])))(args[0].detach())


def test_traced_steps_and_draws():
    q, k, v, decay, _ = make(torch.float32, 3, 1, 2, 2, 12, 20, seed=5)
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    slots = torch.tensor([3, 0, 5], device="cuda")
    step = lambda *a: dcn.DecayAttentionFunction.step(*a)     # noqa: E731
    traced = torch.jit.trace(step, (q, k, v, decay, torch.zeros(6, 2, 12, 20, device="cuda"), slots), check_trace=False)
    here, there = (torch.zeros(6, 2, 12, 20, device="cuda") for _ in range(2))
    for i in range(3):
        assert torch.equal(traced(q * i, k, v, decay, here, slots), step(q * i, k, v, decay, there, slots)) and torch.equal(here, there)
    assert bool(here[slots].any())
    draw = lambda x, u, t: dcn.TokenSampleFunction.apply(x, u, t, 5, 0.9)     # noqa: E731
    x, u, t = randn(gen(1), 7, 300), torch.rand(7, device="cuda"), torch.rand(7, device="cuda") + 0.5
    traced = torch.jit.trace(draw, (x, u, t), check_trace=False)
    for a, b in zip(traced(x * 2, u * 0.5, t), draw(x * 2, u * 0.5, t)):
        assert torch.equal(a, b)


def test_steps_and_draws_refuse_derivatives_and_transforms():
    import torch.autograd.forward_ad as fwad
    q, k, v, decay, _ = make(torch.float32, 3, 1, 2, 2, 12, 20, seed=6)
    args = [q[:, 0], k[:, 0], v[:, 0], decay, torch.randn(3, 2, 12, 20, device="cuda")]
    before = args[4].clone()
    with fwad.dual_level():
        for i in (0, 1, 2, 4):
            dual = list(args)
            dual[i] = fwad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError), torch.no_grad():
                dcn.DecayAttentionFunction.step(*dual)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q, k, v, s: dcn.DecayAttentionFunction.step(q[None], k[None], v[None], decay, s[None]))(*args[:3], args[4])
    assert torch.equal(args[4], before)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x, u: dcn.TokenSampleFunction.apply(x[None], u[None])[0])(torch.randn(3, 50, device="cuda"), torch.rand(3, device="cuda"))


def test_several_host_threads():
    """Each with its own stream and sizes, all at once"""
    def once(i):
        q, k, v, decay, state = make(torch.bfloat16, 1, 200 + 64 * i, 2, 1, 32 + i, 40, seed=i)
        q = q.detach().requires_grad_()
        out, last = dcn.DecayAttentionFunction.apply(q, k, v, decay, state)
        y = dcn.GroupNormActFunction.apply(out.flatten(2), 2, None, None, None, "silu")
        token, score = dcn.TokenSampleFunction.apply(y[0].detach().float(), torch.full((y.size(1),), 0.3, device="cuda"), 0.8, 7, 0.9)
        (dq,) = torch.autograd.grad(y, q, torch.ones_like(y))
        return [x.detach().clone() for x in (out, last, y, token, score, dq)]

    want = [once(i) for i in range(4)]
    torch.cuda.synchronize()
    start, bad = threading.Barrier(4), []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            start.wait(60)
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = once(i)
            stream.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append(i)
        except Exception as e:                   # reported by the test's own thread
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not bad


FIRST = """
import threading, torch
import deform_conv3d_pytorch_op_b200 as dcn
torch.manual_seed(0)
q, k, v = (torch.randn(1, 300, 1, w, device="cuda").bfloat16().requires_grad_() for w in (21, 21, 115))
decay = torch.full((1,), -0.1, device="cuda")

def run():
    out, last = dcn.DecayAttentionFunction.apply(q, k, v, decay)
    return [out, last] + list(torch.autograd.grad((out, last), (q, k, v), (torch.ones_like(out), torch.ones_like(last))))

torch.cuda.synchronize()
got = []
threads = [threading.Thread(target=lambda: got.append(run())) for _ in range(2)]
for t in threads:
    t.start()
    t.join()
torch.cuda.synchronize()
want = run()
assert len(got) == 2 and all(torch.equal(a, b) for g in got for a, b in zip(g, want))
print("same")
"""


def test_first_calls_of_threads():
    """The first thing that a thread does, and the first backward pass of a process, which autograd's own thread runs"""
    done = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300, cwd=Path(__file__).parent.parent)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_modules_of_16_bits(t):
    """Decays stay float32: rounded to 16 bits, one that lasts 512 steps would be another"""
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    torch.manual_seed(0)
    block = dcn.DecayAttention(24, 4, 16, 8, kv_heads=2, memory=32.0, device="cuda")
    decay = block.log_decay.clone()
    block = block.to(t)
    assert torch.equal(block.log_decay, decay) and torch.equal(block.cpu().log_decay.cuda(), decay)
    block = block.cuda()
    x = torch.randn(2, 90, 24, device="cuda", dtype=t)
    y, last = block(x)
    assert y.dtype == t and last.dtype == torch.float32 and bool(torch.isfinite(y).all())
    block.load_state_dict(dcn.DecayAttention(24, 4, 16, 8, kv_heads=2, memory=8.0).state_dict())
    assert block.log_decay.dtype == torch.float32 and not torch.equal(block.log_decay, decay)
    head = SequenceHead(12, 24, 9, mixer="attention", heads=3, device="cuda").to(t)
    logits, _ = head(torch.randn(2, 30, 12, device="cuda", dtype=t))
    assert bool(torch.isfinite(logits).all())

"""Decayed attention, group norm and token sampling in autograd, traces, transforms, threads and modules of 16 bits."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from tests.test_decay_attention_gpu import EXTRA, STATE, make

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


def _between_guards(elements, dtype, offset):
    """A buffer of bytes, and the part of it that starts `offset` elements behind 256 bytes"""
    size = torch.empty(0, dtype=dtype).element_size()
    raw = torch.full((512 + (elements + offset) * size + 16,), 0x5A, dtype=torch.uint8, device="cuda")
    begin = 256 + offset * size
    return raw, begin, begin + elements * size


def _untouched(raw, begin, end):
    return bool((raw[:begin] == 0x5A).all()) and bool((raw[end:] == 0x5A).all())


@pytest.mark.parametrize("steps,heads,kv,dk,dv", [(1, 1, 1, 1, 1), (1, 2, 1, 3, 1), (3, 2, 1, 5, 7), (60, 4, 2, 16, 24), (100, 2, 2, 16, 24),
                                                  (100, 4, 2, 33, 9), (300, 1, 1, 21, 115)])
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_results_that_start_anywhere(t, offset, steps, heads, kv, dk, dv):
    """The C calls with results in the middle of 16 bytes, between guards: right, and nothing written beside"""
    import ctypes
    from deform_conv3d_pytorch_op_b200 import _lib
    from tests import more_sequence_reference as more
    from tests import sequence_reference as ref
    L, b = _lib.lib(), 2
    q, k, v, decay, state = make(t, b, steps, heads, kv, dk, dv, seed=steps + dk)
    do = randn(gen(9), b, steps, heads, dv).to(t)
    leaves = [x.double().requires_grad_() for x in (q, k, v, state)]
    want, end = more.decay_attention(*leaves[:3], decay.double(), leaves[3])
    expected = torch.autograd.grad((want, end), leaves, (do.double(), torch.ones_like(end)))
    p = _lib.dcn_attn(dtype=0 if t == torch.float32 else 1, batch=b, steps=steps, heads=heads, kv_heads=kv, dk=dk, dv=dv, scale=dk ** -0.5)
    for n, x in (("q", q), ("k", k), ("v", v), ("dout", do)):
        for i, a in enumerate(("batch", "step", "head")):
            setattr(p, "%s_%s" % (n, a), x.stride(i))
    ws = [torch.empty(max(L.dcn_attn_workspace_bytes(ctypes.byref(p), i), 16), dtype=torch.uint8, device="cuda") for i in range(2)]
    sizes = [("out", want, t), ("last", end, torch.float32), ("dq", expected[0], t), ("dk", expected[1], t), ("dv", expected[2], t),
             ("dstate", expected[3], torch.float32)]
    bufs = {n: _between_guards(x.numel(), d, offset) for n, x, d in sizes}
    at = {n: raw.data_ptr() + begin for n, (raw, begin, _) in bufs.items()}
    stream = torch.cuda.current_stream().cuda_stream
    ones = torch.ones_like(state)
    assert L.dcn_attn_forward(ctypes.byref(p), q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), state.data_ptr(), 0, at["out"],
                              at["last"], ws[0].data_ptr(), ws[0].numel(), stream) == 0
    assert L.dcn_attn_backward(ctypes.byref(p), q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), state.data_ptr(), 0,
                               do.data_ptr(), ones.data_ptr(), at["dq"], at["dk"], at["dv"], at["dstate"], ws[1].data_ptr(),
                               ws[1].numel(), stream) == 0
    torch.cuda.synchronize()
    for n, x, d in sizes:
        raw, begin, stop = bufs[n]
        assert _untouched(raw, begin, stop), n
        got = raw[begin:stop].clone().view(d).view(x.shape)
        ref.close(got, x, n, chain=ref.CHAIN + (EXTRA[t] if d == t else STATE[t]))


@pytest.mark.parametrize("shape,groups", [((1, 1, 3), 1), ((4, 1, 20), 4), ((3, 40, 24), 3), ((2, 3000, 40), 5)])
@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("t", [torch.float32, torch.float16], ids=["f32", "f16"])
def test_norms_that_start_anywhere(t, offset, shape, groups):
    import ctypes
    from deform_conv3d_pytorch_op_b200 import _lib
    from tests import more_sequence_reference as more
    from tests import sequence_reference as ref
    L, g, c = _lib.lib(), gen(sum(shape)), shape[-1]
    x, dy, w = randn(g, *shape).to(t), randn(g, *shape).to(t), randn(g, c)
    wx, ww = x.double().requires_grad_(), w.double().requires_grad_()
    want = more.group_norm_act(wx, groups, ww, None, None, "silu")
    dx, dw = torch.autograd.grad(want, (wx, ww), dy.double())
    p = _lib.dcn_gnorm(dtype=0 if t == torch.float32 else 2, weight_dtype=0, act=2, samples=shape[0], positions=shape[1], channels=c, groups=groups, eps=1e-5)
    ws = [torch.empty(max(L.dcn_gnorm_workspace_bytes(ctypes.byref(p), i), 16), dtype=torch.uint8, device="cuda") for i in range(2)]
    sizes = [("y", want, t), ("stats", torch.empty(shape[0] * groups * 2), torch.float32), ("dx", dx, t), ("dw", dw, torch.float32)]
    bufs = {n: _between_guards(v.numel(), d, offset) for n, v, d in sizes}
    at = {n: raw.data_ptr() + begin for n, (raw, begin, _) in bufs.items()}
    stream = torch.cuda.current_stream().cuda_stream
    assert L.dcn_gnorm_forward(ctypes.byref(p), x.data_ptr(), w.data_ptr(), 0, 0, at["y"], at["stats"], ws[0].data_ptr(), ws[0].numel(), stream) == 0
    assert L.dcn_gnorm_backward(ctypes.byref(p), x.data_ptr(), w.data_ptr(), 0, 0, at["stats"], dy.data_ptr(), at["dx"], at["dw"], 0, 0,
                                ws[1].data_ptr(), ws[1].numel(), stream) == 0
    torch.cuda.synchronize()
    for n, v, d in sizes:
        raw, begin, stop = bufs[n]
        assert _untouched(raw, begin, stop), n
        if n != "stats":
            ref.close(raw[begin:stop].clone().view(d).view(v.shape), v, n, scale=(x.numel() / c) ** 0.5 if n == "dw" else 1.0)


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


CAPTURED = """
import torch
import deform_conv3d_pytorch_op_b200 as dcn
g = torch.Generator(device="cuda").manual_seed(0)
logits = torch.randn(20, 50257, generator=g, device="cuda").bfloat16()
uniform = torch.rand(20, generator=g, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    token, score = dcn.TokenSampleFunction.apply(logits, uniform, 0.9, 40, 0.9)
graph.replay()
torch.cuda.synchronize()
want, other = dcn.TokenSampleFunction.apply(logits, uniform, 0.9, 40, 0.9)
assert torch.equal(token, want) and torch.equal(score, other)
print("same")
"""


def test_first_draw_of_a_process_is_captured():
    """How many clusters the GPU holds is asked while a graph records"""
    done = subprocess.run([sys.executable, "-c", CAPTURED], capture_output=True, text=True, timeout=300, cwd=Path(__file__).parent.parent)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr

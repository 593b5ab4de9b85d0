"""CPU checks of the C ABI of decayed attention, group norm and token sampling: arguments are refused before anything is launched."""
import ctypes

import pytest
import torch

import deform_conv3d_pytorch_op_b200 as dcn
from deform_conv3d_pytorch_op_b200 import _lib, build

NULL, SHAPE, UNSUPPORTED, WORKSPACE, ALIGN, LIMIT = -1, -2, -3, -4, -7, -8
P = 0x1000                                       # an address that nothing reads: the calls below stop before a launch


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


def _attn(**kw):
    base = dict(dtype=1, batch=2, steps=70, heads=4, kv_heads=2, dk=16, dv=24, scale=0.25)
    for n, w in (("q", 64), ("k", 32), ("v", 48), ("dout", 96)):
        base.update({n + "_batch": 70 * w, n + "_step": w, n + "_head": w // (2 if n in "kv" else 4)})
    return _lib.dcn_attn(**{**base, **kw})


def test_attention_arguments(L):
    def bytes_of(p, backward):
        return L.dcn_attn_workspace_bytes(ctypes.byref(p), backward)

    def fwd(p, q=P, k=P, v=P, decay=P, state=0, lengths=0, out=P, last=P, ws=P, nbytes=1 << 40):
        return L.dcn_attn_forward(ctypes.byref(p), q, k, v, decay, state, lengths, out, last, ws, nbytes, None)

    def bwd(p, q=P, k=P, v=P, decay=P, state=0, lengths=0, dout=P, dlast=0, dq=P, dk=P, dv=P, dstate=0, ws=P, nbytes=1 << 40):
        return L.dcn_attn_backward(ctypes.byref(p), q, k, v, decay, state, lengths, dout, dlast, dq, dk, dv, dstate, ws, nbytes, None)

    for call in (fwd, bwd):
        assert call(_attn(dtype=3)) == UNSUPPORTED and call(_attn(batch=-1)) == SHAPE and call(_attn(kv_heads=3)) == SHAPE
        assert call(_attn(dk=0)) == SHAPE and call(_attn(scale=0.0)) == SHAPE and call(_attn(scale=float("nan"))) == SHAPE
        assert call(_attn(scale=1e-45)) == SHAPE                                     # (its reciprocal is not finite)
        assert call(_attn(dk=129)) == LIMIT and call(_attn(dv=200)) == LIMIT and call(_attn(steps=1 << 31)) == LIMIT
        assert call(_attn(batch=1 << 27)) == LIMIT and call(_attn(heads=1 << 16, kv_heads=1)) == LIMIT
        assert call(_attn(), q=0) == NULL and call(_attn(), decay=0) == NULL and call(_attn(), v=P + 1) == ALIGN
        assert call(_attn(), state=P + 2) == ALIGN and call(_attn(), lengths=P + 4) == ALIGN and call(_attn(batch=0)) == 0
    assert fwd(_attn(), last=0) == NULL and fwd(_attn(), out=0) == NULL
    assert bwd(_attn(), dout=0) == NULL and bwd(_attn(), dv=0, dstate=P) == NULL
    assert bwd(_attn(), dq=0, dk=0, dv=0) == 0                                       # nothing is asked for
    # heads that share a key or a value: their own gradients are summed up from float32
    assert bytes_of(_attn(), 1) >= 2 * 70 * 4 * (16 + 24) * 4 and bwd(_attn(), ws=0) == WORKSPACE
    assert bwd(_attn(), nbytes=bytes_of(_attn(), 1) - 1) == WORKSPACE
    long = _attn(batch=1, steps=16384, heads=1, kv_heads=1)
    assert bytes_of(long, 0) > 0 and bytes_of(long, 0) % (16 * 24 * 4) == 0 and fwd(long, ws=0) == WORKSPACE
    assert bytes_of(_attn(heads=2048, kv_heads=2048), 0) == 0 and bytes_of(_attn(dtype=9), 0) == 0

    def step(p, q=P, state=P, pool=4, slots=0, out=P):
        return L.dcn_attn_step(ctypes.byref(p), q, P, P, P, state, pool, slots, out, None)

    one = _attn(steps=1)
    assert step(_attn()) == SHAPE and step(one, pool=1) == SHAPE and step(one, pool=-1) == SHAPE and step(one, q=0) == NULL
    assert step(one, state=0) == NULL and step(one, slots=P + 4) == ALIGN and step(one, state=P + 2) == ALIGN
    assert step(_attn(steps=1, batch=0)) == 0 and step(_attn(steps=1, dv=129)) == LIMIT


def _gnorm(**kw):
    return _lib.dcn_gnorm(**{**dict(dtype=1, weight_dtype=0, act=2, samples=4, positions=900, channels=48, groups=6, eps=1e-5), **kw})


def test_group_norm_arguments(L):
    def fwd(p, x=P, w=P, b=P, res=0, y=P, stats=0, ws=P, nbytes=1 << 40):
        return L.dcn_gnorm_forward(ctypes.byref(p), x, w, b, res, y, stats, ws, nbytes, None)

    def bwd(p, x=P, w=P, b=P, res=0, stats=P, dy=P, dx=P, dw=0, db=0, dres=0, ws=P, nbytes=1 << 40):
        return L.dcn_gnorm_backward(ctypes.byref(p), x, w, b, res, stats, dy, dx, dw, db, dres, ws, nbytes, None)

    for call in (fwd, bwd):
        assert call(_gnorm(dtype=4)) == UNSUPPORTED and call(_gnorm(weight_dtype=2)) == UNSUPPORTED and call(_gnorm(act=3)) == UNSUPPORTED
        assert call(_gnorm(groups=5)) == SHAPE and call(_gnorm(samples=-1)) == SHAPE and call(_gnorm(eps=-1.0)) == SHAPE
        assert call(_gnorm(channels=8256, groups=1)) == LIMIT and call(_gnorm(positions=1 << 31)) == LIMIT
        assert call(_gnorm(samples=(1 << 31) - 1, positions=(1 << 31) - 1)) == LIMIT
        assert call(_gnorm(), x=0) == NULL and call(_gnorm(), x=P + 1) == ALIGN and call(_gnorm(), w=P + 2) == ALIGN
        assert call(_gnorm(samples=0)) == 0 and call(_gnorm(positions=0)) == 0
    assert fwd(_gnorm(), y=0) == NULL and bwd(_gnorm(), dy=0) == NULL and bwd(_gnorm(), stats=0) == NULL
    large = _gnorm(positions=50000)
    for backward, call in ((0, fwd), (1, bwd)):
        need = L.dcn_gnorm_workspace_bytes(ctypes.byref(large), backward)
        assert need > 0 and call(large, ws=0) == WORKSPACE and call(large, nbytes=need - 1) == WORKSPACE and call(large, ws=P + 4) == WORKSPACE
    assert L.dcn_gnorm_workspace_bytes(ctypes.byref(_gnorm(positions=1)), 0) == 0
    assert L.dcn_gnorm_workspace_bytes(ctypes.byref(_gnorm(groups=7)), 0) == 0


def _sample(**kw):
    return _lib.dcn_sample(**{**dict(dtype=1, rows=5, vocab=640, row_stride=640, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0), **kw})


def test_sampling_arguments(L):
    def call(p, logits=P, uniforms=P, tokens=P, logprobs=P):
        return L.dcn_sample_tokens(ctypes.byref(p), logits, uniforms, tokens, logprobs, None, 0, None)

    assert call(_sample(dtype=7)) == UNSUPPORTED and call(_sample(rows=-1)) == SHAPE and call(_sample(vocab=0)) == SHAPE
    for bad in (dict(temperature=-1.0), dict(temperature=1e-4), dict(temperature=float("nan")), dict(top_p=1.5), dict(top_p=-0.1),
                dict(min_p=2.0), dict(min_p=float("nan"))):
        assert call(_sample(**bad)) == SHAPE
    assert call(_sample(temperature=0.0, rows=0)) == 0 and call(_sample(vocab=(1 << 20) + 1)) == LIMIT and call(_sample(rows=1 << 27)) == LIMIT
    assert call(_sample(), logits=0) == NULL and call(_sample(), uniforms=0) == NULL and call(_sample(), logprobs=0) == NULL
    assert call(_sample(), logits=P + 1) == ALIGN and call(_sample(), tokens=P + 4) == ALIGN and call(_sample(), uniforms=P + 2) == ALIGN
    assert call(_sample(temperatures=P + 2)) == ALIGN and call(_sample(top_ks=P + 4)) == ALIGN
    assert L.dcn_sample_tokens(None, P, P, P, P, None, 0, None) == NULL


def test_modules_hold_their_parameters_and_refuse_the_cpu():
    attn, norm = dcn.DecayAttention(12, 4, 6, dv=10, kv_heads=2), dcn.GroupNormAct(4, 20, "silu", dim=-1)
    assert attn.proj.weight.shape == (4 * 6 + 2 * 16, 12) and attn.norm.channels == 40
    assert attn.log_decay.shape == (4,) and bool((attn.log_decay < 0).all()) and not attn.log_decay.requires_grad
    assert bool((attn.log_decay.diff() > 0).all()) and attn.new_states(3).shape == (3, 4, 6, 10)
    assert "log_decay" in attn.state_dict()
    for f in (lambda: attn(torch.zeros(1, 3, 12)), lambda: norm(torch.zeros(4, 20)),
              lambda: dcn.TokenSampleFunction.apply(torch.zeros(2, 5), torch.zeros(2))):
        with pytest.raises(dcn.DcnError, match="CUDA"):
            f()
    with pytest.raises(dcn.DcnError, match="activation"):
        dcn.GroupNormActFunction.apply(torch.zeros(4, 20), 4, None, None, None, "gelu")


def test_attention_modules_that_are_refused():
    for kw in (dict(heads=2, dk=129), dict(heads=2, dk=8, dv=0), dict(heads=4, dk=8, kv_heads=3), dict(heads=0, dk=8)):
        with pytest.raises(dcn.DcnError, match="heads"):
            dcn.DecayAttention(16, **kw)
    block = dcn.DecayAttention(16, 4, 8, 12, kv_heads=2)
    assert block.proj.out_features == 4 * 8 + 2 * (8 + 12) and tuple(block.new_states(3).shape) == (3, 4, 8, 12)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_attention_keeps_the_parts_of_split_heads_alone(L, dtype):
    """Heads that do not fill the GPU a whole number of times are split in time, into 32 parts at most: the parts' sums of those few, 64
    columns each, are all that a call without other scratch needs, however many heads there are"""
    for heads in (1, 5, 150, 2962, 5930, 65535):
        for dk, dv in ((128, 128), (64, 128), (128, 8), (16, 24)):
            strides = {n + a: w for n, d in (("q", dk), ("k", dk), ("v", dv), ("dout", dv))
                       for a, w in (("_batch", 16384 * heads * d), ("_step", heads * d), ("_head", d))}
            p = _attn(dtype=dtype, batch=1, steps=16384, heads=heads, kv_heads=heads, dk=dk, dv=dv, **strides)
            most = 2 * 160 * 32 * max(dk, dv) * 64 * 4         # (two CTAs an SM or fewer, on a GPU of up to 160)
            for backward in (0, 1):
                assert L.dcn_attn_workspace_bytes(ctypes.byref(p), backward) <= most, (heads, dk, dv, backward)


def test_modules_of_more_channels_than_their_norm_takes_are_refused():
    for make in (lambda: dcn.DecayAttention(16, 128, 128), lambda: dcn.DecayAttention(16, 65, 8, 127), lambda: dcn.GroupNormAct(2, 8194),
                 lambda: dcn.GroupNormAct(1, 0)):
        with pytest.raises(dcn.DcnError, match="8192"):
            make()
    with pytest.raises(dcn.DcnError, match="8192"):
        from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
        SequenceHead(features=8, width=8320, mixer="attention", heads=65, num_classes=3, blocks=1, device="meta")
    assert dcn.DecayAttention(16, 64, 1, 128).norm.channels == 8192 and dcn.GroupNormAct(8192, 8192).weight.numel() == 8192

"""CPU checks of the sequence operators' C ABI: the header and the binding list the same symbols, and arguments are refused
before anything is launched."""
import ctypes
import os
import re

import pytest
import torch

import deform_conv3d_pytorch_op_b200 as dcn
from deform_conv3d_pytorch_op_b200 import _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NULL, SHAPE, UNSUPPORTED, WORKSPACE, ALIGN, LIMIT = -1, -2, -3, -4, -7, -8
P = 0x1000                                       # an address that nothing reads: the calls below stop before a launch


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


def test_header_symbols_are_exported(L):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "dcn_seq.h")).read(), flags=re.S)
    assert set(re.findall(r"\b(dcn_[a-z0-9_]+)\s*\(", text)) == set(_lib.SEQUENCE_SYMBOLS)
    for sym in _lib.SEQUENCE_SYMBOLS:
        assert hasattr(L, sym), sym


def _scan(**kw):
    return _lib.dcn_scan(**{**dict(dtype=1, batch=2, steps=70, channels=6, x_batch=420, x_step=6, gate_batch=420, gate_step=6,
                                   dy_batch=420, dy_step=6), **kw})


def test_scan_arguments(L):
    def fwd(p, x=P, gate=P, state=0, lengths=0, y=P, last=P, ckpt=0):
        return L.dcn_scan_forward(ctypes.byref(p), x, gate, state, lengths, y, last, ckpt, None)

    def bwd(p, x=P, gate=P, ckpt=P, dy=P, dlast=0, dx=P, dgate=P, dstate=0):
        return L.dcn_scan_backward(ctypes.byref(p), x, gate, 0, ckpt, dy, dlast, dx, dgate, dstate, None)

    assert L.dcn_scan_checkpoint_bytes(ctypes.byref(_scan())) == 2 * 2 * 6 * 4
    assert L.dcn_scan_checkpoint_bytes(ctypes.byref(_scan(steps=0))) == 0
    for call in (fwd, bwd):
        assert call(_scan(dtype=3)) == UNSUPPORTED and call(_scan(batch=-1)) == SHAPE
        assert call(_scan(steps=1 << 31)) == LIMIT and call(_scan(batch=1 << 27)) == LIMIT
        assert call(_scan(), x=0) == NULL and call(_scan(), gate=0) == NULL
        assert call(_scan(), x=P + 1) == ALIGN and call(_scan(dtype=0), gate=P + 2) == ALIGN
        assert call(_scan(batch=0)) == 0 and call(_scan(channels=0)) == 0
    assert fwd(_scan(), last=0) == NULL and fwd(_scan(), y=0) == NULL and fwd(_scan(), state=P + 2) == ALIGN
    assert bwd(_scan(), ckpt=0) == NULL and bwd(_scan(), dx=0) == NULL and bwd(_scan(), dlast=P + 2) == ALIGN
    assert L.dcn_scan_forward(None, P, P, 0, 0, P, P, 0, None) == NULL

    def step(dtype=0, rows=3, channels=8, x=P, state=P, pool=4, slots=0):
        return L.dcn_scan_step(dtype, rows, channels, x, 8, P, 8, state, pool, slots, P, None)

    assert step(dtype=7) == UNSUPPORTED and step(rows=-1) == SHAPE and step(pool=2) == SHAPE and step(x=0) == NULL
    assert step(state=0) == NULL and step(slots=P + 4) == ALIGN and step(rows=0) == 0 and step(channels=1 << 31) == LIMIT


def _norm(**kw):
    return _lib.dcn_norm(**{**dict(dtype=1, weight_dtype=0, rows=5, channels=64, x_row=64, block_row=64, gate_row=64,
                                   dstream_row=64, dnormed_row=64, eps=1e-6), **kw})


def test_norm_arguments(L):
    def fwd(p, x=P, block=P, gate=0, scale=0, stream=P, normed=P, stats=0):
        return L.dcn_norm_forward(ctypes.byref(p), x, block, gate, scale, 0, 0, stream, normed, stats, None)

    def bwd(p, x=P, block=P, gate=0, scale=0, stats=P, dblock=P, dgate=0, dscale=0, ws=0, nbytes=0):
        return L.dcn_norm_backward(ctypes.byref(p), x, block, gate, scale, 0, 0, stats, P, P, P, dblock, dgate, dscale, 0, 0, ws,
                                   nbytes, None)

    for call in (fwd, bwd):
        assert call(_norm(dtype=3)) == UNSUPPORTED and call(_norm(weight_dtype=2)) == UNSUPPORTED
        assert call(_norm(rows=-1)) == SHAPE and call(_norm(channels=0)) == SHAPE and call(_norm(channels=8193)) == LIMIT
        assert call(_norm(), x=0) == NULL and call(_norm(), x=P + 1) == ALIGN and call(_norm(), scale=P + 2) == ALIGN
        assert call(_norm(rows=0)) == 0
    assert fwd(_norm(), stream=0) == NULL and fwd(_norm(), block=0) == NULL and fwd(_norm(), stats=P + 2) == ALIGN
    assert bwd(_norm(), stats=0) == NULL and bwd(_norm(), block=0) == NULL and bwd(_norm(), dgate=P) == NULL
    need = L.dcn_norm_workspace_bytes(ctypes.byref(_norm()))
    assert need > 0 and need % (2 * 64 * 4) == 0
    assert bwd(_norm(), dscale=P) == WORKSPACE and bwd(_norm(), dscale=P, ws=P, nbytes=need - 1) == WORKSPACE


def _logits(**kw):
    return _lib.dcn_logits(**{**dict(dtype=1, rows=5, vocab=640, row_stride=640, temperature=1.0), **kw})


def test_logits_arguments(L):
    def scores(p, logits=P, tokens=P, top=0, logprob=P, best=0, best_tokens=0):
        return L.dcn_scores_forward(ctypes.byref(p), logits, tokens, -100, top, logprob, P, best, best_tokens, 0, None)

    def dscores(p, logits=P, top=0, stats=P):
        return L.dcn_scores_backward(ctypes.byref(p), logits, P, -100, top, P, stats, P, P, P, P, None)

    def distill(p, logits=P, k=8, teacher_type=0, tail=1):
        return L.dcn_distill_forward(ctypes.byref(p), logits, k, P, teacher_type, P, tail, P, 0, None)

    def ddistill(p, logits=P, k=8, teacher_type=0, tail=1):
        return L.dcn_distill_backward(ctypes.byref(p), logits, k, P, teacher_type, P, tail, P, P, P, None)

    for call in (scores, dscores, distill, ddistill):
        assert call(_logits(dtype=5)) == UNSUPPORTED and call(_logits(vocab=0)) == SHAPE and call(_logits(rows=-2)) == SHAPE
        for t in (0.0, -1.0, 1e-4, 1e4, float("nan")):
            assert call(_logits(temperature=t)) == SHAPE
        assert call(_logits(rows=1 << 27)) == LIMIT and call(_logits(vocab=1 << 31)) == LIMIT
        assert call(_logits(), logits=0) == NULL and call(_logits(), logits=P + 1) == ALIGN and call(_logits(rows=0)) == 0
    for call in (scores, dscores):
        assert call(_logits(), top=-1) == SHAPE and call(_logits(vocab=3), top=4) == SHAPE and call(_logits(), top=129) == LIMIT
    assert scores(_logits(), tokens=0) == NULL and scores(_logits(), top=3, best=P) == NULL and dscores(_logits(), stats=0) == NULL
    for call in (distill, ddistill):
        assert call(_logits(), k=0) == SHAPE and call(_logits(), k=129) == LIMIT and call(_logits(), tail=2) == UNSUPPORTED
        assert call(_logits(), teacher_type=2) == UNSUPPORTED and call(_logits(vocab=(1 << 20) + 1)) == LIMIT


def test_modules_hold_their_parameters_and_refuse_the_cpu():
    scan, norm, first = dcn.GatedScan(12, 20), dcn.ResidualNorm(20, scale=0.5), dcn.ResidualNorm(20, first=True)
    assert scan.proj.weight.shape == (40, 12)
    assert sorted(n for n, _ in norm.named_parameters()) == ["post_weight", "pre_weight", "scale"]
    assert [n for n, _ in first.named_parameters()] == ["pre_weight"]
    with pytest.raises(dcn.DcnError, match="CUDA"):
        scan(torch.zeros(1, 3, 12))
    with pytest.raises(dcn.DcnError, match="CUDA"):
        first(torch.zeros(4, 20))
    with pytest.raises(dcn.DcnError, match="CUDA"):
        dcn.TopkDistillLoss(3).teacher(torch.zeros(4, 20))

"""Token sampling against its definition in whole numbers: tokens have to be the same ones."""
import math

import pytest
import torch

from tests import more_sequence_reference as more
from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu


def check(logits, uniform, *settings):
    import deform_conv3d_pytorch_op_b200 as dcn
    tokens, logprob = dcn.TokenSampleFunction.apply(logits, uniform, *settings)
    want, lp = more.sample(logits, uniform, *settings)
    assert tokens.dtype == torch.int64 and logprob.dtype == torch.float32
    wrong = (tokens != want).nonzero().flatten().tolist()
    assert not wrong, (wrong[:5], tokens[wrong[:5]].tolist(), want[wrong[:5]].tolist())
    assert torch.equal(torch.isnan(logprob), torch.isnan(lp))
    fine = ~torch.isnan(lp)
    # rounded once from 64 bits
    assert bool(((logprob.double() - lp).abs()[fine] <= 2.0 ** -23 * lp.abs()[fine].clamp(min=2.0 ** -20)).all())
    return tokens


def make(t, rows, vocab, sharp=3.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=g, device="cuda") * sharp).to(t)
    return logits, torch.rand(rows, generator=g, device="cuda")


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 50, 0.8, 0.02), (2.0, 1, 0.5, 0.0),
            (1.0, 10 ** 6, 0.999, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 3, 1e-6, 1.0)]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
@pytest.mark.parametrize("vocab", [1, 2, 33, 400, 5003])
def test_settings(t, vocab, settings):
    logits, uniform = make(t, 37, vocab, seed=vocab)
    check(logits, uniform, *settings)


@pytest.mark.parametrize("rows,vocab,sharp", [(1, 131072, 3.0), (5, 100003, 1.0), (3, 50257, 0.05), (300, 9001, 2.0), (2, 1 << 20, 2.5)])
@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_large_vocabularies(t, rows, vocab, sharp):
    if vocab == 1 << 20 and t != torch.bfloat16:
        pytest.skip("once is enough")
    logits, uniform = make(t, rows, vocab, sharp, seed=rows)
    for settings in ((1.0, 0, 1.0, 0.0), (0.9, 50, 0.9, 0.0), (1.0, 0, 0.7, 0.001), (1.0, 20000, 0.99, 0.0)):
        check(logits[:4], uniform[:4], *settings) if rows == 300 else check(logits, uniform, *settings)


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_equal_logits(t):
    """Ties at the limits count by their index, wherever they lie"""
    g = torch.Generator(device="cuda").manual_seed(1)
    for vocab in (50, 40000):
        logits = torch.randint(-3, 4, (9, vocab), generator=g, device="cuda").to(t)
        uniform = torch.rand(9, generator=g, device="cuda")
        for settings in ((1.0, 7, 1.0, 0.0), (1.0, vocab // 3, 1.0, 0.0), (1.0, 0, 0.35, 0.0), (0.5, vocab // 2, 0.9, 0.01)):
            check(logits, uniform, *settings)
    same = torch.zeros(4, 30001, device="cuda", dtype=t)
    same[:, ::2] = -0.0
    uniform = torch.tensor([0.0, 0.25, 0.5, 0.99999994], device="cuda")
    for settings in ((1.0, 1000, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.0)):
        check(same, uniform, *settings)


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_forbidden_tokens_and_odd_rows(t):
    import deform_conv3d_pytorch_op_b200 as dcn
    logits, uniform = make(t, 12, 3000, seed=2)
    logits[:, ::3] = -math.inf
    logits[1] = -math.inf
    logits[2, 17] = math.nan
    logits[3, 5] = math.inf
    logits[4] = -math.inf
    logits[4, 2999] = -5.0
    logits[5] = torch.finfo(t).min                                   # masked by the lowest value, all of them
    logits[6] = torch.finfo(t).min
    logits[6, 1234] = torch.finfo(t).max
    logits[7, 1:] = torch.finfo(t).min
    for settings in SETTINGS:
        tokens = check(logits, uniform, *settings)
        assert tokens[[1, 2, 3]].tolist() == [-1, -1, -1] and int(tokens[4]) == 2999 and int(tokens[6]) == 1234
    nan = torch.tensor([math.nan] * 12, device="cuda")
    for i in range(4):
        args = [uniform, 1.0, 0, 1.0, 0.0]
        args[i if i == 0 else (1, 3, 4)[i - 1]] = nan
        tokens, logprob = dcn.TokenSampleFunction.apply(logits, *args)
        assert bool((tokens == -1).all()) and bool(torch.isnan(logprob).all())


def test_numbers_at_the_ends():
    logits, _ = make(torch.float32, 6, 999, seed=3)
    for u in ([0.0] * 6, [1.0 - 2.0 ** -24] * 6, [1.0, 2.0, -1.0, -0.0, 1e-30, 0.5]):
        uniform = torch.tensor(u, device="cuda")
        check(logits, uniform.clamp(0, 1), 1.0, 0, 0.9)
    import deform_conv3d_pytorch_op_b200 as dcn
    a = dcn.TokenSampleFunction.apply(logits, torch.tensor([2.0, -3.0] * 3, device="cuda"))
    b = dcn.TokenSampleFunction.apply(logits, torch.tensor([1.0, 0.0] * 3, device="cuda"))
    assert torch.equal(a[0], b[0])


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_settings_of_each_row(t):
    rows = 40
    logits, uniform = make(t, rows, 2501, seed=4)
    g = torch.Generator(device="cuda").manual_seed(5)
    temperature = torch.rand(rows, generator=g, device="cuda") * 2
    temperature[::7] = 0
    top_k = torch.randint(-1, 60, (rows,), generator=g, device="cuda", dtype=torch.int32)
    top_p = torch.rand(rows, generator=g, device="cuda") * 1.2
    min_p = torch.rand(rows, generator=g, device="cuda") * 0.1
    check(logits, uniform, temperature, top_k, top_p, min_p)
    check(logits, uniform, temperature, 0, top_p, 0.0)
    check(logits, uniform, 1.0, top_k.long(), 1.0, min_p)


def test_views_and_shapes():
    import deform_conv3d_pytorch_op_b200 as dcn
    base = torch.randn(3, 5, 1010, device="cuda").half()
    part = base[:, :, 3:1004]
    uniform = torch.rand(3, 5, device="cuda")
    tokens, logprob = dcn.TokenSampleFunction.apply(part, uniform, 0.9, 20, 0.95)
    assert tokens.shape == (3, 5) and logprob.shape == (3, 5)
    want, _ = more.sample(part.reshape(15, 1001), uniform.flatten(), 0.9, 20, 0.95)
    assert torch.equal(tokens.flatten(), want)
    t, lp = dcn.TokenSampleFunction.apply(base[0, 0], torch.tensor(0.3, device="cuda"))
    assert t.shape == () and lp.shape == ()
    assert dcn.TokenSampleFunction.apply(base[:0, 0], uniform[:0, 0])[0].shape == (0,)


def test_probabilities():
    """How often tokens come, and their log p, against the softmax"""
    import deform_conv3d_pytorch_op_b200 as dcn
    n = 200000
    logits = torch.tensor([1.0, 0.0, 2.0, -1.0, 0.5], device="cuda").expand(n, 5)
    uniform = (torch.arange(n, device="cuda") + 0.5) / n
    tokens, logprob = dcn.TokenSampleFunction.apply(logits, uniform, 0.7)
    p = torch.softmax(logits[0].double() / 0.7, 0)
    assert float((torch.bincount(tokens, minlength=5) / n - p).abs().max()) <= 2 / n + 1e-6
    # the argument of the exponential is rounded to float32 (of up to 5): 2^-23, its value by two units
    assert float((logprob.double() - p.log()[tokens]).abs().max()) <= 4e-7 + 2.0 ** -22
    kept = dcn.TokenSampleFunction.apply(logits, uniform, 0.7, 2)
    assert set(kept[0].tolist()) == {0, 2}
    scores = dcn.TokenScoresFunction.apply(logits[:, [0, 2]], (kept[0] // 2), 0, 0.7)[0]
    assert float((kept[1] - scores).abs().max()) <= 2e-6


def test_captured():
    import deform_conv3d_pytorch_op_b200 as dcn
    logits, uniform = make(torch.bfloat16, 16, 32000, seed=6)
    held = logits.clone()
    dcn.TokenSampleFunction.apply(held, uniform, 0.8, 40, 0.9)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = dcn.TokenSampleFunction.apply(held, uniform, 0.8, 40, 0.9)
    held.copy_(logits.flip(1))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], dcn.TokenSampleFunction.apply(held, uniform, 0.8, 40, 0.9)[0])


def test_refusals():
    import deform_conv3d_pytorch_op_b200 as dcn
    apply = dcn.TokenSampleFunction.apply
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    for args, text in [((x.cpu(), u), "CUDA"), ((x.double(), u), "float32"), ((x, u[:2]), "uniform has shape"), ((x, u.half()), "uniform has dtype"),
                       ((x, u.cpu()), "CUDA"), ((x, u, -1.0), "temperature"), ((x, u, 1e-4), "temperature"), ((x, u, math.nan), "temperature"),
                       ((x, u, 1.0, 0, 1.1), "top_p"), ((x, u, 1.0, 0, -0.1), "top_p"), ((x, u, 1.0, 0, 1.0, 2.0), "min_p"),
                       ((x, u, 1.0, u), "int64 or int32"), ((x, u, u[:1]), "temperature has shape"), ((x, u, u.long()), "temperature must be"),
                       ((torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1]), "2\\^20"), ((x[:, :0], u), "vocabulary"),
                       ((x.clone().requires_grad_(), u), "no gradient")]:
        with pytest.raises(dcn.DcnError, match=text):
            apply(*args)
    with pytest.raises(TypeError):
        apply(x, u, 1.0, 2.5)

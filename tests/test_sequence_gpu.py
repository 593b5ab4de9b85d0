"""The sequence operators against their definitions in 64 bits: sizes, types, layouts and masks where they can go wrong."""
import math

import pytest
import torch

from tests import sequence_reference as ref
from tests.sequence_reference import TYPES, close

pytestmark = pytest.mark.gpu
dcn = pytest.importorskip("deform_conv3d_pytorch_op_b200")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def wide(*ts):
    """float64 leaves of the same values"""
    return [None if t is None else t.detach().double().requires_grad_() for t in ts]


def grads(outs, ins, gouts):
    """Gradients by input (None where there is no input)"""
    pairs = [(o, g) for o, g in zip(outs, gouts) if o is not None and g is not None]
    asked = [t for t in ins if t is not None]
    got = torch.autograd.grad([o for o, _ in pairs], asked, [g for _, g in pairs], allow_unused=True)
    it = iter(got)
    return [None if t is None else next(it) for t in ins]


# ---- gated scan -----------------------------------------------------------------------------------------------------------
SCANS = [(1, 1, 1), (2, 3, 5), (3, 8, 32), (1, 9, 64), (2, 63, 33), (2, 64, 66), (2, 65, 34), (1, 129, 100), (3, 513, 96),
         (1, 1200, 34), (2, 2050, 130), (150, 70, 64), (5, 300, 2048), (1, 700, 5000), (3, 1000, 1601)]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", SCANS)
def test_scan(shape, kind, ragged):
    g, t = gen(shape[1] + 7 * shape[2]), TYPES[kind]
    b, n, c = shape
    x, gate = randn(g, b, n, c, dtype=t), randn(g, b, n, c, mean=1.5, std=2.0, dtype=t)
    state = randn(g, b, c) if n % 2 else None
    lengths = torch.randint(0, n + 1, (b,), generator=g, device="cuda") if ragged else None
    if ragged:
        lengths[0] = 0 if b > 1 else n
        behind = torch.arange(n, device="cuda")[None, :] >= lengths[:, None]
        x[behind], gate[behind] = math.nan, math.inf          # whatever stands there
    dy, dlast = randn(g, b, n, c, dtype=t), randn(g, b, c)
    xs, gs, ss = x.requires_grad_(), gate.requires_grad_(), None if state is None else state.requires_grad_()
    y, last = dcn.GatedScanFunction.apply(xs, gs, ss, lengths)
    got = grads((y, last), (xs, gs, ss), (dy, dlast))
    wx, wg, ws = wide(x, gate, state)
    if ragged:
        with torch.no_grad():
            wx[behind], wg[behind] = 0.0, 0.0
    wy, wl = ref.scan(wx, wg, ws, lengths)
    want = grads((wy, wl), (wx, wg, ws), (dy.double(), dlast.double()))
    assert y.dtype == t and last.dtype == torch.float32
    close(y, wy, "y")
    close(last, wl, "last")
    for name, a, w in zip(("dx", "dgate", "dstate"), got, want):
        if w is not None:
            close(a, w, name)
    with torch.no_grad():                                     # no checkpoints are made: the same values
        again = dcn.GatedScanFunction.apply(x, gate, state, lengths)
    assert torch.equal(again[0], y) and torch.equal(again[1], last)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["projection", "time_major", "odd_offset", "last_axis_strided", "expanded"])
def test_scan_layouts(kind, layout):
    g, t = gen(3), TYPES[kind]
    b, n, c = 3, 77, 40
    if layout == "projection":
        both = randn(g, b, n, 2 * c, dtype=t)
        x, gate = both[..., :c], both[..., c:]
    elif layout == "time_major":
        x, gate = randn(g, n, b, c, dtype=t).transpose(0, 1), randn(g, n, b, c, dtype=t).transpose(0, 1)
    elif layout == "odd_offset":
        flat = randn(g, b * n * c + 1, dtype=t)
        x, gate = flat[1:].view(b, n, c), randn(g, b, n, c + 1, dtype=t)[..., 1:]
    elif layout == "last_axis_strided":
        x, gate = randn(g, b, n, 2 * c, dtype=t)[..., ::2], randn(g, b, c, n, dtype=t).transpose(1, 2)
    else:
        x, gate = randn(g, 1, n, c, dtype=t).expand(b, n, c), randn(g, b, 1, c, dtype=t).expand(b, n, c)
    x, gate = x.detach().requires_grad_(), gate.detach().requires_grad_()
    y, last = dcn.GatedScanFunction.apply(x, gate)
    wx, wg = wide(x, gate)
    wy, wl = ref.scan(wx, wg)
    close(y, wy)
    close(last, wl)
    for a, w in zip(grads((y.sum(),), (x, gate), (torch.ones((), device="cuda", dtype=t),)), grads((wy.sum(),), (wx, wg), (torch.ones((), device="cuda").double(),))):
        close(a, w)                                           # dy is an expanded scalar
    y, last = dcn.GatedScanFunction.apply(x, gate)
    wy, wl = ref.scan(wx, wg)
    for a, w in zip(grads((last,), (x, gate), (torch.ones_like(last),)), grads((wl,), (wx, wg), (torch.ones_like(wl),))):
        close(a, w)                                           # and no dy at all


def test_scan_keeps_long_memories():
    """Gates near one: 1 - a is not formed as a difference, and a state lasts through thousands of steps."""
    g = gen(4)
    x, gate = randn(g, 2, 3000, 48), torch.full((2, 3000, 48), 11.0, device="cuda")
    state = randn(g, 2, 48)
    y, last = dcn.GatedScanFunction.apply(x, gate, state)
    wy, wl = ref.scan(x.double(), gate.double(), state.double())
    close(y, wy)
    close(last, wl)
    x, gate = randn(g, 1, 70, 3), randn(g, 1, 70, 3)
    gate[:, 5], gate[:, 9] = math.inf, -math.inf              # kept whole, and replaced whole
    gate[:, 20, 1] = math.nan
    y, _ = dcn.GatedScanFunction.apply(x, gate)
    close(y, ref.scan(x.double(), gate.double())[0])
    assert torch.equal(y[:, 5], y[:, 4]) and torch.equal(y[:, 9], x[:, 9]) and bool(y[0, 20:, 1].isnan().all())


def test_scan_of_nothing():
    x = torch.zeros(2, 0, 5, device="cuda", requires_grad=True)
    state = torch.ones(2, 5, device="cuda", requires_grad=True)
    y, last = dcn.GatedScanFunction.apply(x, x, state)
    assert y.shape == (2, 0, 5) and torch.equal(last, state)
    (d,) = torch.autograd.grad(last.sum(), state)
    assert torch.equal(d, torch.ones_like(state))
    for shape in ((0, 4, 5), (3, 4, 0)):
        y, last = dcn.GatedScanFunction.apply(torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda"))
        assert y.shape == shape and last.shape == (shape[0], shape[2])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("channels", [1, 33, 64, 1000])
def test_steps_are_the_scan(kind, channels):
    g, t = gen(channels), TYPES[kind]
    both = randn(g, 5, 12, 2 * channels, dtype=t)
    x, gate = both[..., :channels], both[..., channels:]
    pool = randn(g, 9, channels)
    before = pool.clone()
    slots = torch.tensor([7, 2, -1, 0, 9], device="cuda")     # the third and the last have no place
    live = torch.tensor([0, 1, 3], device="cuda")
    y, last = dcn.GatedScanFunction.apply(x[live], gate[live], before[slots[live]])
    for i in range(12):
        out = dcn.GatedScanFunction.step(x[:, i], gate[:, i], pool, slots)
        close(out[live], y[:, i].double(), chain=2 * ref.CHAIN)
        assert not out[2].any() and not out[4].any()
    close(pool[slots[live]], last.double(), chain=2 * ref.CHAIN)
    others = [1, 3, 4, 5, 6, 8]
    assert torch.equal(pool[others], before[others])
    state = before.clone()
    out = dcn.GatedScanFunction.step(x[:, 0], gate[:, 0], state, None)
    close(out, ref.scan(x[:, :1].double(), gate[:, :1].double(), before[:5].double())[1])
    assert torch.equal(state[5:], before[5:])


# ---- gated residual norm --------------------------------------------------------------------------------------------------
NORMS = [(1, 1), (3, 7), (5, 32), (17, 256), (4, 257), (9, 512), (33, 1000), (6, 2048), (3, 4099), (5, 8192), (3000, 64), (700, 520),
         (40, 1022), (9, 4098), (71, 34), (1025, 16), (33, 130), (2001, 100), (2, 6002)]


@pytest.mark.parametrize("kind,weights", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("shape", NORMS)
def test_norm(shape, kind, weights):
    g, t, wt = gen(sum(shape)), TYPES[kind], TYPES[weights]
    n, c = shape
    x, block, gate = randn(g, n, c, dtype=t), randn(g, n, c, std=3.0, dtype=t), randn(g, n, c, dtype=t)
    scale, post, pre = [randn(g, c, std=0.2, mean=1.0, dtype=wt) for _ in range(3)]
    ins = [v.requires_grad_() for v in (x, block, gate, scale, post, pre)]
    gouts = randn(g, n, c, dtype=t), randn(g, n, c, dtype=t)
    outs = dcn.ResidualNormFunction.apply(*ins, 1e-5)
    got = grads(outs, ins, gouts)
    w = wide(*ins)
    wants = ref.residual_norm(*w, 1e-5)
    want = grads(wants, w, [v.double() for v in gouts])
    for name, a, b in zip(("stream", "normed"), outs, wants):
        close(a, b, name)
    terms = 1.0 if c == 1 else 0.0                            # one channel: its norm is +-1 and has no gradient
    for name, a, b in zip(("dx", "dblock", "dgate", "dscale", "dpost", "dpre"), got, want):
        assert a.dtype == (wt if name in ("dscale", "dpost", "dpre") else t)
        close(a, b, name, scale=terms)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("parts", ["x", "x,pre", "x,block", "x,block,gate", "x,block,scale,pre", "x,block,post", "x,block,gate,scale,post"])
def test_norm_without_some_parts(kind, parts):
    g, t, parts = gen(9), TYPES[kind], parts.split(",")
    for c in (24, 600):
        full = {"x": randn(g, 2, 11, c, dtype=t), "block": randn(g, 2, 11, c, dtype=t), "gate": randn(g, 2, 11, c, dtype=t)}
        full.update({k: randn(g, c, std=0.3, mean=1.0) for k in ("scale", "post", "pre")})
        ins = [full[k].requires_grad_() if k in parts else None for k in ("x", "block", "gate", "scale", "post", "pre")]
        outs = dcn.ResidualNormFunction.apply(*ins)
        if "block" not in parts:
            assert outs[0] is ins[0]
        w = wide(*ins)
        wants = ref.residual_norm(*w)
        gouts = [randn(g, 2, 11, c, dtype=t) for _ in range(2)]
        for which in ((0, 1), (0,), (1,)):                    # gradients of both outputs, or of one
            pick = [v if i in which else None for i, v in enumerate(gouts)]
            if "block" not in parts and which == (0,):
                continue
            outs, wants = dcn.ResidualNormFunction.apply(*ins), ref.residual_norm(*w)
            got = grads(outs, ins, pick)
            want = grads(wants, w, [None if v is None else v.double() for v in pick])
            for o, b in zip(outs, wants):
                close(o, b)
            for k, a, b in zip(full, got, want):
                if a is not None:
                    close(a, torch.zeros_like(a).double() if b is None else b, k)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_norm_layouts(kind):
    g, t = gen(10), TYPES[kind]
    c = 72
    fused = randn(g, 4, 9, 3 * c, dtype=t)
    odd = randn(g, 4 * 9 * c + 1, dtype=t)[1:].view(4, 9, c)
    moved = randn(g, 9, 4, c, dtype=t).transpose(0, 1)        # rows without one stride: copied
    strided = randn(g, 4, 9, 2 * c, dtype=t)[..., ::2]
    for x, block, gate in ((fused[..., :c], fused[..., c:2 * c], fused[..., 2 * c:]), (odd, moved, strided), (moved, odd, odd)):
        ins = [v.detach().requires_grad_() for v in (x, block, gate)]
        outs = dcn.ResidualNormFunction.apply(*ins)
        w = wide(*ins)
        wants = ref.residual_norm(*w)
        for o, b in zip(outs, wants):
            close(o, b)
        ones = torch.ones((), device="cuda")
        for a, b in zip(grads([o.float().sum() for o in outs], ins, (ones, ones)), grads([o.sum() for o in wants], w, (ones.double(), ones.double()))):
            close(a, b)


def test_norm_of_odd_rows():
    empty = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    outs = dcn.ResidualNormFunction.apply(empty, empty, None, w, w, w)
    assert outs[0].shape == outs[1].shape == (0, 16)
    assert not torch.autograd.grad(outs[1].sum(), w)[0].any()
    x = torch.zeros(3, 40, device="cuda")
    x[1, 3], x[2, 5] = math.nan, math.inf
    stream, normed = dcn.ResidualNormFunction.apply(x, torch.zeros_like(x))
    assert not normed[0].any() and bool(normed[1].isnan().all()) and bool(normed[2, 5].isnan())


# ---- token scores ---------------------------------------------------------------------------------------------------------
VOCABS = [(1, 1), (3, 2), (5, 7), (4, 31), (16, 400), (9, 1023), (3, 2048), (3, 2049), (2, 4100), (700, 517), (1, 20011), (2, 70001), (40, 33000)]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", VOCABS)
def test_scores(shape, kind):
    g, t = gen(shape[1]), TYPES[kind]
    n, v = shape
    logits = randn(g, n, v, std=3.0, dtype=t).requires_grad_()
    tokens = torch.randint(0, v, (n,), generator=g, device="cuda")
    tokens[0] = -100 if n > 1 else 0
    w = logits.detach().double().requires_grad_()
    for top in sorted({0, 1, min(v, 5), min(v, 128)}):
        for temperature in (1.0, 0.6):
            outs = dcn.TokenScoresFunction.apply(logits, tokens, top, temperature)
            wants = ref.token_scores(w, tokens, top, temperature)
            close(outs[0], wants[0], "logprob", scale=1.0)    # (log p near 0 is a difference of logits of this size)
            close(outs[1], wants[1], "entropy", scale=1.0)
            if top == 0:
                assert outs[2] is None and outs[3] is None
            else:
                close(outs[2], wants[2], "top", scale=1.0)
                assert torch.equal(outs[3], wants[3]), "top tokens"
            gouts = randn(g, n), randn(g, n), randn(g, n, top) if top else None
            (got,) = grads(outs[:3], (logits,), gouts)
            (want,) = grads(wants[:3], (w,), [None if a is None else a.double() for a in gouts])
            close(got, want, "dlogits", scale=1e-3 if v == 1 else 0.0)
    with torch.no_grad():
        again = dcn.TokenScoresFunction.apply(logits, None, min(v, 5))
    assert again[0] is None and torch.equal(again[3], ref.token_scores(w, tokens, min(v, 5))[3])


def _rows_that_hide(kind, v):
    """Rows with masks, ties, order and special values, [rows, v]"""
    g, t = gen(v), TYPES[kind]
    lowest = torch.finfo(t).min
    rows = randn(g, 14, v, std=2.0, dtype=t)
    rows[0] = -math.inf                                       # nothing left
    rows[1] = lowest                                          # masked with the type's lowest value throughout
    rows[2, : v - 1] = -math.inf                              # one token left
    rows[3, 1:] = lowest
    rows[4] = 0.5                                             # all equal
    rows[5] = rows[5].sort().values                           # ascending, descending
    rows[6] = rows[6].sort(descending=True).values
    rows[7, ::2] = -math.inf
    rows[8] = rows[8].round()                                 # few values, many ties
    rows[9, v // 2] = math.nan
    rows[10, v // 3] = math.inf
    rows[11] = -0.0
    rows[11, v // 2] = 0.0
    rows[12, :] = -1.0
    per, threads = (4 if kind == "f32" else 8), 256           # large values in places that one thread reads
    at = torch.arange(v, device="cuda")
    big = (at // per) % threads == 3
    rows[12, big] = (torch.arange(int(big.sum()), device="cuda") % 977 + 1).to(t)
    rows[13] = lowest
    rows[13, min(v - 1, 11)] = -math.inf
    return rows


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [3, 300, 1500, 5000, 131072, 400003])
def test_scores_of_masked_tied_and_special_rows(kind, v):
    rows = _rows_that_hide(kind, v).requires_grad_()
    tokens = torch.full((rows.size(0),), v - 1, device="cuda")
    w = rows.detach().double()
    for top in (1, 3, min(v, 40), min(v, 128)):
        logprob, entropy, best, best_tokens = dcn.TokenScoresFunction.apply(rows, tokens, top)
        a, b, c, d = ref.token_scores(w, tokens, top)
        a[10], b[10], c[10] = math.nan, math.nan, math.nan    # inf - inf
        for got, want in ((logprob, a), (entropy, b), (best, c)):
            close(got, want, scale=1.0)
        assert torch.equal(best_tokens, d)
    (d,) = torch.autograd.grad((logprob.nan_to_num(0, 0, 0) * 0 + entropy).sum(), rows)
    p = torch.softmax(torch.where(w == -math.inf, -1e9, w), -1)
    assert not d[0].any()                                     # nothing left: no gradient
    good = [i for i in range(14) if i not in (9, 10)]
    assert bool(torch.isfinite(d[good]).all()) and bool(d[9].isnan().all())
    assert bool((d[2].abs() <= 2.0 ** -20).all())             # one token left: entropy 0 whatever it is
    logprob = dcn.TokenScoresFunction.apply(rows, tokens)[0]
    (d,) = torch.autograd.grad(logprob, rows, torch.ones_like(logprob))
    want = -p
    want[:, v - 1] += 1
    want[0] = 0.0
    close(d[[1, 4, 5, 6, 8, 11, 12]], want[[1, 4, 5, 6, 8, 11, 12]], scale=1e-3)
    assert not d[0].any()


def test_scores_layouts_and_tokens():
    g = gen(12)
    padded = randn(g, 6, 5, 1030, dtype=torch.bfloat16)
    for logits in (padded[..., :1000], padded[..., 1:1024], padded[..., 3:], padded.transpose(0, 1)[..., 5:], padded[:, :1].expand(6, 5, 1030)):
        logits = logits.detach().requires_grad_()
        tokens = torch.randint(0, logits.size(-1), logits.shape[:-1], generator=g, device="cuda", dtype=torch.int32)
        tokens[0, 0], tokens[1, 1], tokens[2, 2] = -7, logits.size(-1), -100
        w = logits.detach().double().requires_grad_()
        outs = dcn.TokenScoresFunction.apply(logits, tokens, 4, 1.0, -7)
        wants = ref.token_scores(w, tokens.long(), 4, 1.0, -7)
        assert float(outs[0][0, 0]) == 0.0 and bool(outs[0][1, 1].isnan()) and bool(outs[0][2, 2].isnan())
        for a, b in zip(outs[:3], wants):
            close(a, b, scale=1.0)
        assert torch.equal(outs[3], wants[3])
        go = randn(g, *tokens.shape)
        go2 = torch.where(torch.isnan(outs[0]), 0.0, go)
        (got,) = torch.autograd.grad(outs[0], logits, go2)
        (want,) = torch.autograd.grad(torch.where(torch.isnan(wants[0]), 0.0, wants[0]), w, go2.double())
        close(got, want)
    none = dcn.TokenScoresFunction.apply(torch.zeros(0, 9, device="cuda"), torch.zeros(0, dtype=torch.long, device="cuda"), 3)
    assert none[0].shape == (0,) and none[3].shape == (0, 3)


# ---- distillation ---------------------------------------------------------------------------------------------------------
def _teacher(g, n, v, k, std=2.0):
    logits = randn(g, n, v, std=std)
    best, tokens = logits.topk(k)
    return best - logits.logsumexp(-1, keepdim=True), tokens


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 2, 1), (4, 9, 9), (7, 31, 5), (32, 400, 10), (5, 2048, 128), (6, 2049, 64), (3, 10007, 100), (200, 600, 8), (2, 70001, 33), (1, 131072, 128)])
def test_distill(n, v, k, tail, kind):
    g, t = gen(v + k), TYPES[kind]
    logits = randn(g, n, v, std=2.0, dtype=t).requires_grad_()
    lq, tokens = _teacher(g, n, v, k)
    for temperature in (1.0, 2.0):
        loss = dcn.DistillTopkFunction.apply(logits, lq, tokens, temperature, tail)
        w = logits.detach().double().requires_grad_()
        want = ref.distill(w, lq.double(), tokens, temperature, tail)
        close(loss, want, "loss", scale=1.0)
        go = randn(g, n)
        (a,), (b,) = grads((loss,), (logits,), (go,)), grads((want,), (w,), (go.double(),))
        close(a, b, "dlogits", scale=1e-3 if k == v or (k == 1 and not tail) else 0.0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("v", [40, 3000, 40001])
def test_distill_of_unused_repeated_and_masked_places(kind, v):
    g, t, n, k = gen(v), TYPES[kind], 9, 12
    logits = randn(g, n, v, std=2.0, dtype=t)
    lq, tokens = _teacher(g, n, v, k)
    tokens[0] = -1                                            # no place used
    tokens[1, 3:] = -1
    tokens[2, 4], tokens[2, 7] = v, 10 ** 12                  # outside the vocabulary
    tokens[3, 5] = tokens[3, 6]                               # a token twice
    lq[4, 6:] = -math.inf                                     # without probability
    keep = logits[5, tokens[5]]
    logits[5] = -math.inf                                     # the student has nothing outside the teacher's places
    logits[5, tokens[5]] = keep
    logits[6] = -math.inf                                     # nothing at all
    logits[7, tokens[7, 0]] = -math.inf                       # nothing where the teacher is
    logits[8, v // 2] = math.nan
    logits.requires_grad_()
    for tail in (True, False):
        loss = dcn.DistillTopkFunction.apply(logits, lq.to(t), tokens, 1.0, tail)
        w = logits.detach().double().requires_grad_()
        want = ref.distill(w, lq.to(t).double(), tokens, 1.0, tail)
        assert float(loss[0]) == 0.0 and math.isinf(float(loss[6])) and math.isinf(float(loss[7])) and math.isnan(float(loss[8]))
        fine = [1, 2, 3, 4, 5]
        close(loss[fine], want[fine].detach(), scale=1.0)
        (a,) = torch.autograd.grad(loss, logits, torch.ones_like(loss))
        (b,) = torch.autograd.grad(want[fine].sum(), w)
        assert not a[0].any() and not a[6].any() and bool(torch.isfinite(a[7]).all()) and bool(a[8].isnan().all())
        close(a[fine], b[fine], scale=1e-3)


@pytest.mark.parametrize("v", [500, 50000])
def test_distill_with_nearly_all_mass_on_the_teachers_tokens(v):
    """The student's remaining probability is summed, not formed as one minus the others: it is right at 1e-12 too."""
    g, n, k = gen(v), 4, 6
    logits = randn(g, n, v, std=0.5)
    lq, tokens = _teacher(g, n, v, k)
    logits.scatter_(1, tokens, 40.0)
    logits.requires_grad_()
    loss = dcn.DistillTopkFunction.apply(logits, lq, tokens)
    w = logits.detach().double().requires_grad_()
    want = ref.distill(w, lq.double(), tokens)
    close(loss, want)
    (a,), (b,) = torch.autograd.grad(loss.sum(), logits), torch.autograd.grad(want.sum(), w)
    close(a, b)


def test_distill_takes_the_teachers_scores():
    g = gen(15)
    teacher, student = randn(g, 3, 8, 900, std=3.0), randn(g, 3, 8, 900, dtype=torch.bfloat16)
    loss = dcn.TopkDistillLoss(900 // 8, temperature=2.0)
    lq, tokens = loss.teacher(teacher)
    got = loss(student, lq, tokens)
    want = ref.distill(student.double().flatten(0, 1), lq.double().flatten(0, 1), tokens.flatten(0, 1), 2.0).mean()
    close(got, want)
    same = dcn.DistillTopkFunction.apply(teacher, lq, tokens, 2.0)
    assert float(same.abs().max()) <= 4 * ref.CHAIN * 10      # the teacher itself: terms of up to 10, difference 0


# ---- gradients against differences -----------------------------------------------------------------------------------------
def _slope(f, x, direction, h):
    with torch.no_grad():
        return (f(x + h * direction) - f(x - h * direction)) / (2 * h)


@pytest.mark.parametrize("op", ["scan_x", "scan_gate", "norm_x", "norm_block", "norm_gate", "norm_pre", "scores", "distill"])
def test_gradients_against_differences(op):
    """Central differences of the float32 forward pass along a direction: their error is h^2 = 1e-4 of a third derivative of the
    order of the sum, and roundings of 1e-6 of it over h = 1e-2: 1e-3 of the sum's scale is their sum, rounded up."""
    g, h = gen(21), 1e-2
    weight = randn(g, 3, 50, 36)
    if op.startswith("scan"):
        a, b = randn(g, 3, 50, 36), randn(g, 3, 50, 36, mean=1.0)
        fn = (lambda v: dcn.GatedScanFunction.apply(v, b)[0]) if op == "scan_x" else (lambda v: dcn.GatedScanFunction.apply(a, v)[0])
        at = a if op == "scan_x" else b
    elif op.startswith("norm"):
        parts = [randn(g, 3, 50, 36) for _ in range(3)] + [None, None, randn(g, 36, mean=1.0, std=0.1)]
        i = {"norm_x": 0, "norm_block": 1, "norm_gate": 2, "norm_pre": 5}[op]
        fn, at = (lambda v: sum(dcn.ResidualNormFunction.apply(*parts[:i], v, *parts[i + 1:]))), parts[i]
    else:
        at = randn(g, 3, 50, 36)
        if op == "scores":
            tokens = torch.randint(0, 36, (3, 50), generator=g, device="cuda")

            def fn(v):                                        # (not the alternatives: they change places along the way)
                return torch.stack(dcn.TokenScoresFunction.apply(v, tokens)[:2], -1)
        else:
            lq, tokens = _teacher(g, 150, 36, 5)
            fn = lambda v: dcn.DistillTopkFunction.apply(v, lq.view(3, 50, 5), tokens.view(3, 50, 5), 1.5)[..., None]  # noqa: E731

    def total(v):
        y = fn(v)
        return (y.double() * weight[..., :y.size(-1)].double()).sum()

    at = at.clone().requires_grad_()
    (grad,) = torch.autograd.grad(total(at), at)
    direction = torch.randn(at.shape, generator=g, device="cuda")
    got, want = float((grad.double() * direction).sum()), float(_slope(total, at.detach(), direction, h))
    with torch.no_grad():
        y = fn(at)
        scale = float((y.double() * weight[..., :y.size(-1)]).abs().sum().sqrt()) * 10
    assert abs(got - want) <= 1e-3 * max(abs(want), scale), (got, want, scale)


# ---- machinery ------------------------------------------------------------------------------------------------------------
def _calls():
    g = gen(30)
    x, gate = randn(g, 4, 200, 96), randn(g, 4, 200, 96)
    w = [randn(g, 96) for _ in range(3)]
    logits, tokens = randn(g, 40, 9001), torch.randint(0, 9001, (40,), generator=g, device="cuda")
    lq, tt = _teacher(g, 40, 9001, 20)
    return {
        "scan": (lambda a, b: dcn.GatedScanFunction.apply(a, b), [x, gate]),
        "norm": (lambda a, b, c, *v: dcn.ResidualNormFunction.apply(a, b, c, *v), [x, gate, x * 0.5] + w),
        "scores": (lambda a: dcn.TokenScoresFunction.apply(a, tokens, 10)[:3], [logits]),
        "distill": (lambda a: (dcn.DistillTopkFunction.apply(a, lq, tt),), [logits]),
    }


def _pass(fn, args):
    args = [a.detach().clone().requires_grad_() for a in args]
    outs = fn(*args)
    return [o.detach() for o in outs] + list(torch.autograd.grad([o.sum() for o in outs], args))


@pytest.mark.parametrize("name", ["scan", "norm", "scores", "distill"])
def test_results_repeat_on_any_stream_and_in_graphs(name):
    fn, args = _calls()[name]
    want = _pass(fn, args)
    for a, b in zip(_pass(fn, args), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _pass(fn, args)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    static = [a.detach().clone().requires_grad_() for a in args]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = fn(*static)
        got = [o.detach() for o in outs] + list(torch.autograd.grad([o.sum() for o in outs], static))
    graph.replay()
    graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["scan", "norm", "scores", "distill"])
def test_place_in_autograd(name):
    fn, args = _calls()[name]
    leaves = [a.detach().clone().requires_grad_() for a in args]
    outs = fn(*leaves)
    total = sum(o.sum() for o in outs)
    first = torch.autograd.grad(total, leaves, retain_graph=True)
    for i, leaf in enumerate(leaves):                         # some gradients only
        (one,) = torch.autograd.grad(total, leaf, retain_graph=True)
        assert torch.equal(one, first[i])
    again = torch.autograd.grad(total, leaves)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(total, leaves)
    outs = fn(*leaves)
    dys = [torch.ones_like(o, requires_grad=True) for o in outs]
    got = torch.autograd.grad(outs, leaves[0], dys, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got.sum().backward()
    outs = fn(*leaves)
    with torch.no_grad():
        leaves[0].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(sum(o.sum() for o in outs), leaves)
    traced = torch.jit.trace(lambda *a: tuple(fn(*a)), tuple(a.detach() for a in args), check_trace=False)
    other = [(a.detach() * 0.5).requires_grad_() for a in args]
    t, w = traced(*other), fn(*other)
    assert all(torch.equal(a, b) for a, b in zip(t, w))
    for a, b in zip(torch.autograd.grad(sum(o.sum() for o in t), other), torch.autograd.grad(sum(o.sum() for o in w), other)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: sum(o.sum() for o in fn(v, *[a.detach() for a in args[1:]])))(args[0].detach())


def test_refusals():
    E = dcn.DcnError
    x, g64 = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, 8, device="cuda", dtype=torch.float64)
    scan, norm, scores, distill = (f.apply for f in (dcn.GatedScanFunction, dcn.ResidualNormFunction, dcn.TokenScoresFunction, dcn.DistillTopkFunction))
    for call, words in [
            (lambda: scan(x.cpu(), x.cpu()), "CUDA"), (lambda: scan(g64, g64), "float32, bfloat16 or float16"),
            (lambda: scan(x, x.bfloat16()), "dtype"), (lambda: scan(x, x[:, :2]), "shape"), (lambda: scan(x[0], x[0]), "shape"),
            (lambda: scan(x, x, x[:, 0].bfloat16()), "dtype"), (lambda: scan(x, x, x[:, 0, :4]), "shape"),
            (lambda: scan(x, x, None, torch.zeros(2, device="cuda")), "int64"),
            (lambda: scan(x, x, None, torch.zeros(3, dtype=torch.long, device="cuda")), "shape"),
            (lambda: dcn.GatedScanFunction.step(x[0], x[0], x[0, :2].contiguous()), "fewer rows"),
            (lambda: dcn.GatedScanFunction.step(x[0], x[0], x[:, :, ::2].reshape(6, 4)), "state"),
            (lambda: dcn.GatedScanFunction.step(x[0].requires_grad_(), x[0], x[1].contiguous()), "no gradient"),
            (lambda: norm(x, x.half()), "dtype"), (lambda: norm(x, x[:1]), "shape"), (lambda: norm(x, None, x), "without a block"),
            (lambda: norm(x, x, x, torch.ones(7, device="cuda")), "shape"),
            (lambda: norm(x.half(), x.half(), None, torch.ones(8, device="cuda"), torch.ones(8, device="cuda").half()), "dtype"),
            (lambda: norm(torch.zeros(2, 8193, device="cuda")), "8192"), (lambda: norm(x, x, None, None, None, None, -1.0), "eps"),
            (lambda: scores(x, torch.zeros(2, 4, dtype=torch.long, device="cuda")), "shape"),
            (lambda: scores(x, None, 9), "top"), (lambda: scores(torch.zeros(2, 900, device="cuda"), None, 129), "top"),
            (lambda: scores(x, None, 1, 0.0), "temperature"), (lambda: scores(x, torch.zeros(2, 3, device="cuda")), "int64"),
            (lambda: distill(x, x[..., :2], torch.zeros(2, 3, 3, dtype=torch.long, device="cuda")), "shape"),
            (lambda: distill(x, x[..., :0], torch.zeros(2, 3, 0, dtype=torch.long, device="cuda")), "places"),
            (lambda: distill(x, x[..., :2].clone().requires_grad_(), torch.zeros(2, 3, 2, dtype=torch.long, device="cuda")), "detach"),
            (lambda: distill(x, x[..., :2].half(), torch.zeros(2, 3, 2, dtype=torch.long, device="cuda")), "dtype"),
            (lambda: distill(torch.zeros(1, 2 ** 20 + 1, device="cuda"), torch.zeros(1, 2, device="cuda"), torch.zeros(1, 2, dtype=torch.long, device="cuda")), "limited")]:
        with pytest.raises(E, match=words):
            call()
    with pytest.raises(TypeError):
        scan(x, None)
    for shape in ((2, 0), (0,)):
        with pytest.raises(E):
            scores(torch.zeros(shape, device="cuda"))


def test_sizes_of_several_host_threads():
    """Calls of one kernel with different amounts of shared memory at the same time"""
    import threading
    g = gen(91)
    norms = [randn(g, 8, c) for c in (300, 700, 1300, 2000)]
    wants = [dcn.ResidualNormFunction.apply(x, x) for x in norms]
    rows = [(randn(g, 300, v, dtype=torch.bfloat16), torch.randint(0, v, (300, 2), generator=g, device="cuda")) for v in (340000, 400000)]
    q = torch.full((300, 2), math.log(0.25), device="cuda")
    losses = [dcn.DistillTopkFunction.apply(x, q, t) for x, t in rows]
    torch.cuda.synchronize()
    start, bad = threading.Barrier(4), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(30)
                for _ in range(400):
                    got = dcn.ResidualNormFunction.apply(norms[i], norms[i])
                for _ in range(20):
                    loss = dcn.DistillTopkFunction.apply(rows[i % 2][0], q, rows[i % 2][1])
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, wants[i])) and torch.equal(loss, losses[i % 2])
        except Exception as e:                   # reported by the test's own thread
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("channels", [1, 2, 7, 63, 64, 65, 127, 130])
def test_scan_rows_that_start_anywhere(kind, channels):
    """The C calls on tensors that start in the middle of 16 bytes, between guards: the same bits, and nothing written beside"""
    import ctypes
    from deform_conv3d_pytorch_op_b200 import _lib
    L, t, b, n = _lib.lib(), TYPES[kind], 2, 150
    g = gen(92)
    x, gate, dy = (randn(g, b, n, channels, dtype=t) for _ in range(3))
    lengths = torch.tensor([n, 70], device="cuda")
    xr, gr = x.clone().requires_grad_(), gate.clone().requires_grad_()
    y, last = dcn.GatedScanFunction.apply(xr, gr, None, lengths)
    wants = (y.detach(),) + torch.autograd.grad(y, (xr, gr), dy)
    ptr = lambda a: ctypes.c_void_p(a.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for off in (0, 1, 2, 3, 4, 7):
        def shifted(a=None):
            big = torch.full((b * n * channels + 32,), 77.0, dtype=t, device="cuda")
            part = big[8 + off:8 + off + b * n * channels].view(b, n, channels)
            if a is not None:
                part.copy_(a)
            return big, part

        (_, sx), (_, sg), (_, sd) = shifted(x), shifted(gate), shifted(dy)
        outs = [shifted() for _ in range(3)]
        p = _lib.dcn_scan({"f32": 0, "bf16": 1, "f16": 2}[kind], b, n, channels, *(n * channels, channels) * 3)
        end, ckpt = torch.empty(b, channels, device="cuda"), torch.empty(b, 3, channels, device="cuda")
        assert L.dcn_scan_forward(ctypes.byref(p), ptr(sx), ptr(sg), None, ptr(lengths), ptr(outs[0][1]), ptr(end), ptr(ckpt), stream) == 0
        assert L.dcn_scan_backward(ctypes.byref(p), ptr(sx), ptr(sg), ptr(lengths), ptr(ckpt), ptr(sd), None, ptr(outs[1][1]),
                                   ptr(outs[2][1]), None, stream) == 0
        for (big, part), want in zip(outs, wants):
            assert torch.equal(part, want)
            assert bool((big[:8 + off] == 77).all()) and bool((big[8 + off + b * n * channels:] == 77).all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("channels", [1, 3, 33, 63, 65, 129, 511, 513, 1025, 2047, 4097, 8191])
def test_norm_rows_that_start_anywhere(kind, channels):
    """The C calls on odd rows that start in the middle of 16 bytes, between guards: the same bits, and nothing written beside"""
    import ctypes
    from deform_conv3d_pytorch_op_b200 import _lib
    L, t, n = _lib.lib(), TYPES[kind], 37
    g = gen(93)
    ins = [randn(g, n, channels, dtype=t) for _ in range(5)]           # x, block, gate and the gradients of the two results
    w = [randn(g, channels) for _ in range(3)]
    leaves = [a.clone().requires_grad_() for a in ins[:3]]
    outs = dcn.ResidualNormFunction.apply(*leaves, *w)
    wants = [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, ins[3:]))
    ptr = lambda a: ctypes.c_void_p(a.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for off in (0, 1, 2, 3, 4, 7):
        def shifted(a=None):
            big = torch.full((n * channels + 32,), 77.0, dtype=t, device="cuda")
            part = big[8 + off:8 + off + n * channels].view(n, channels)
            if a is not None:
                part.copy_(a)
            return big, part

        s = [shifted(a)[1] for a in ins]
        got = [shifted() for _ in wants]
        stats = torch.empty(n, 2, device="cuda")
        p = _lib.dcn_norm(dtype={"f32": 0, "bf16": 1, "f16": 2}[kind], weight_dtype=0, rows=n, channels=channels, x_row=channels,
                          block_row=channels, gate_row=channels, dstream_row=channels, dnormed_row=channels, eps=1e-6)
        assert L.dcn_norm_forward(ctypes.byref(p), *map(ptr, s[:3]), *map(ptr, w), ptr(got[0][1]), ptr(got[1][1]), ptr(stats), stream) == 0
        assert L.dcn_norm_backward(ctypes.byref(p), *map(ptr, s[:3]), *map(ptr, w), ptr(stats), ptr(s[3]), ptr(s[4]),
                                   *(ptr(a[1]) for a in got[2:]), None, None, None, None, 0, stream) == 0
        for (big, part), want in zip(got, wants):
            assert torch.equal(part, want)
            assert bool((big[:8 + off] == 77).all()) and bool((big[8 + off + n * channels:] == 77).all())

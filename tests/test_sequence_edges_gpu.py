"""The sequence operators at the edges of their values, and of how they are called."""
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


def wide(t):
    return t.detach().double().requires_grad_()


# ---- logits of any finite size ----------------------------------------------------------------------------------------------
def _masked_rows(g, v, value, t):
    """Rows of which a finite value masks everything, contiguous parts, the ends alone, all but a token, and rows near it"""
    rows = randn(g, 9, v, std=2.0, dtype=t)
    rows[0] = value
    rows[1, : v // 2] = value
    rows[2, v // 3:] = value
    rows[3, :3] = rows[3, -3:] = value
    rows[4, 3:-3] = value
    rows[5] = value
    rows[5, v // 2] = 1.0
    rows[6, ::2] = value
    rows[7] = value * (1 + randn(g, v).abs() / 16)            # nothing but values of this size, and all different
    rows[8] = value
    rows[8, 1] = -value                                       # both signs
    return rows


# Results are compared row by row at the bound of every other row: a difference to the largest logit is rounded once, relative
# to itself, whatever the size of the two.
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("value", [-1e6, -1e9, -1e10, -1e12, -1e20, -3e38, 1e10, 1e20])
def test_scores_of_rows_with_large_finite_values(kind, value):
    for v in (301, 1500, 5003, 70001):
        g, t = gen(v), TYPES[kind]
        logits = _masked_rows(g, v, value, t).requires_grad_()
        w = wide(logits)
        for temperature, top in ((1.0, 0), (0.1, 3), (1.0, min(v, 100))):
            if abs(value) > 1e38 and temperature < 1:
                continue                                      # (their log p is beyond float32)
            tokens = torch.tensor([0, v - 1, v // 2] * 3, device="cuda")
            outs = dcn.TokenScoresFunction.apply(logits, tokens, top, temperature)
            wants = ref.token_scores(w, tokens, top, temperature)
            gouts = [randn(g, *o.shape) for o in outs[:3] if o is not None]
            (got,) = torch.autograd.grad([o for o in outs[:3] if o is not None], logits, gouts)
            (want,) = torch.autograd.grad(wants[:3 if top else 2], w, [a.double() for a in gouts])
            for r in range(9):
                what = (v, temperature, top, r)
                for a, b in zip(outs[:3], wants):
                    if a is not None:
                        b = b[r].float().double() if abs(value) > 1e38 else b[r]
                        close(a[r], b, what, scale=1.0)
                if top:
                    assert torch.equal(outs[3][r], wants[3][r]), what
                close(got[r], want[r], what, scale=1e-3)


def _distill_by_formula(z, lq, tokens, dloss, temperature, tail):
    """Loss and gradient in 64 bits, from differences to the largest logit of each part: log p itself, of a size of 1e20, would
    not hold what the tokens of the rest are to one another."""
    z, lq, dloss = z.detach().double() / temperature, lq.double(), dloss.double()
    teachers = torch.zeros_like(z, dtype=torch.bool).scatter_(1, tokens, True)
    m, rest = z.amax(1, keepdim=True), z.masked_fill(teachers, -math.inf)
    top = rest.amax(1, keepdim=True)
    s = torch.exp(z - m).sum(1, keepdim=True)
    e = torch.exp(rest - top)
    if not tail:
        lq = torch.log_softmax(lq, 1)
    q = torch.exp(lq)
    left = (1 - q.sum(1, keepdim=True)).clamp(min=0) if tail else torch.zeros_like(m)
    loss = (q * (lq - (z.gather(1, tokens) - m - torch.log(s)))).sum(1, keepdim=True)
    loss = loss + torch.where(left > 0, left * (torch.log(left) - (top - m + torch.log(e.sum(1, keepdim=True)) - torch.log(s))), 0.0)
    dz = torch.exp(z - m) / s * (q.sum(1, keepdim=True) + left) - left * e / e.sum(1, keepdim=True)
    dz.scatter_add_(1, tokens, -q)
    return loss[:, 0] * temperature ** 2, dz * temperature * dloss[:, None]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("value", [-1e6, -1e9, -1e10, -1e12, -1e20, 1e10])
@pytest.mark.parametrize("tail", [True, False])
def test_distill_of_rows_with_large_finite_values(kind, value, tail):
    for v, k in ((301, 5), (2500, 20), (70001, 64)):
        g, t = gen(v + k), TYPES[kind]
        logits = _masked_rows(g, v, value, t)
        teacher = randn(g, 9, v, std=2.0)
        best, tokens = teacher.topk(k)
        lq = best - teacher.logsumexp(-1, keepdim=True)
        keep = logits[2].gather(0, tokens[2])
        logits[2] = value                                     # all that the teacher does not name
        logits[2].scatter_(0, tokens[2], torch.where(keep == value, torch.ones_like(keep), keep))
        logits.requires_grad_()
        for temperature in (1.0, 0.1):
            loss, go = dcn.DistillTopkFunction.apply(logits, lq, tokens, temperature, tail), randn(g, 9)
            (got,) = torch.autograd.grad(loss, logits, go)
            want, grad = _distill_by_formula(logits, lq, tokens, go, temperature, tail)
            for r in range(9):
                close(loss[r], want[r], (v, temperature, r), scale=1.0)
                close(got[r], grad[r], (v, temperature, r), scale=1e-3)


@pytest.mark.parametrize("temperature", [1.0, 1e-3])
def test_scores_of_float16_rows_at_the_ends_of_their_range(temperature):
    for v in (301, 1500, 70001):
        g = gen(v)
        logits = _masked_rows(g, v, -6e4, torch.float16).requires_grad_()
        w, tokens = wide(logits), torch.tensor([0, v - 1, v // 2] * 3, device="cuda")
        outs = dcn.TokenScoresFunction.apply(logits, tokens, 5, temperature)
        wants = ref.token_scores(w, tokens, 5, temperature)
        gouts = [randn(g, 9), randn(g, 9), randn(g, 9, 5)]
        (got,) = torch.autograd.grad(outs[:3], logits, [a * temperature for a in gouts])
        (want,) = torch.autograd.grad(wants[:3], w, [a.double() * temperature for a in gouts])
        for r in range(9):
            for a, b in zip(outs[:3], wants):
                close(a[r], b[r], (v, r), scale=1.0)
            assert torch.equal(outs[3][r], wants[3][r])
            close(got[r], want[r], (v, r), scale=1e-3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("value", [-1e29, -1e30, -1e36, -3e38])
@pytest.mark.parametrize("v", [301, 70001])
def test_distill_with_all_other_tokens_masked_by_the_lowest_values(kind, value, v):
    """The rest of the teacher's probability meets a log p of the mask's size: a loss that float32 holds, and the right one."""
    g, t, k = gen(v), TYPES[kind], 7
    teacher = randn(g, 4, v, std=2.0)
    best, tokens = teacher.topk(k)
    lq = best - teacher.logsumexp(-1, keepdim=True)
    logits = torch.full((4, v), value, device="cuda", dtype=t)
    logits.scatter_(1, tokens, randn(g, 4, k, dtype=t))
    logits.requires_grad_()
    loss = dcn.DistillTopkFunction.apply(logits, lq, tokens)
    (a,) = torch.autograd.grad(loss.sum(), logits)
    want, b = _distill_by_formula(logits, lq, tokens, torch.ones(4, device="cuda"), 1.0, True)
    close(loss, want)
    close(a, b, scale=1e-3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("temperature", [0.5, 0.05])
def test_distill_at_low_temperatures_beside_the_lowest_values(kind, tail, temperature):
    """temperature^2 KL is a number where log p itself, the lowest value over the temperature, is beyond float32."""
    for v, k in ((301, 7), (5003, 40)):
        g, t = gen(v), TYPES[kind]
        teacher = randn(g, 3, v, std=2.0)
        best, tokens = teacher.topk(k)
        lq = best - teacher.logsumexp(-1, keepdim=True)
        logits = randn(g, 3, v, dtype=t)
        logits[0, tokens[0, k // 2]] = torch.finfo(t).min     # one of the teacher's, all of the others, half of everything
        logits[1] = torch.full_like(logits[1], torch.finfo(t).min).scatter_(0, tokens[1], logits[1, tokens[1]])
        logits[2, v // 2:] = torch.finfo(t).min
        logits.requires_grad_()
        loss = dcn.DistillTopkFunction.apply(logits, lq, tokens, temperature, tail)
        go = randn(g, 3)
        (a,) = torch.autograd.grad(loss, logits, go)
        want, b = _distill_by_formula(logits, lq, tokens, go, temperature, tail)
        for r in range(3):
            close(loss[r], want[r], (v, r), scale=1.0)
            close(a[r], b[r], (v, r), scale=1e-3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dentropy,temperature", [(1.0, 1.0), (1e9, 1.0), (3e6, 1e-3), (-1e20, 2.0)])
def test_entropy_gradients_of_any_size_beside_masked_tokens(kind, dentropy, temperature):
    """p log p of a token that cannot come is 0 whatever it is multiplied with (loss scaling, low temperatures)."""
    g, t = gen(5), TYPES[kind]
    for v in (300, 5003):
        logits = randn(g, 5, v, std=0.01 if temperature < 1 else 1.0, dtype=torch.float32)
        logits[0, ::3], logits[1, v // 2:], logits[2, :5] = -math.inf, -math.inf, -1e4
        logits = logits.to(t).requires_grad_()
        w = wide(logits)
        entropy = dcn.TokenScoresFunction.apply(logits, None, 0, temperature)[1]
        want = ref.token_scores(w, torch.zeros(5, dtype=torch.long, device="cuda"), 0, temperature)[1]
        go = torch.full((5,), dentropy, device="cuda")
        (a,), (b,) = torch.autograd.grad(entropy, logits, go), torch.autograd.grad(want, w, go.double())
        for r in range(5):
            close(a[r], b[r], (v, r))


@pytest.mark.parametrize("start", [0, 3])
def test_scores_of_a_row_of_nearly_2_to_the_31_tokens(start):
    """Alternatives among equal values, whose last elements are counted behind the row's last vector"""
    v = 2 ** 31 - 1
    row = torch.zeros(v + start, device="cuda", dtype=torch.bfloat16)[start:][None]
    high = {v - 1: 3.0, v - 4: 2.0, 17: 2.5, 2 ** 30: 1.0}
    for at, value in high.items():
        row[0, at] = value
    logprob, entropy, best, best_tokens = dcn.TokenScoresFunction.apply(row, torch.tensor([v - 1], device="cuda"), 128)
    first = sorted(high, key=lambda at: -high[at])
    assert best_tokens[0].tolist() == first + [i for i in range(126) if i != 17][:124]
    total = v - len(high) + sum(math.exp(x) for x in high.values())
    wants = [x - math.log(total) for x in [high[at] for at in first] + [0.0] * 124]
    # a thread adds some 2^15 batches of its 2^20 elements to one float, each at half a unit of the sum's last place: 2^-10 of S, and
    # of U, at most
    log = 22 * ref.CHAIN + 2.0 ** -10
    assert float((best[0].double() - torch.tensor(wants, device="cuda", dtype=torch.float64)).abs().max()) <= log
    assert abs(float(logprob) - wants[0]) <= log
    mean = sum(x * math.exp(x) for x in high.values()) / total
    assert abs(float(entropy) - (math.log(total) - mean)) <= 2 * log + 4.4 * 2.0 ** -10      # (U / S is 3 / ln 2)


# ---- single steps -----------------------------------------------------------------------------------------------------------
def test_traced_steps_advance_the_pool():
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    torch.manual_seed(6)
    g = gen(6)
    slots = torch.tensor([3, 0, 5], device="cuda")
    step = lambda x, gate, state, slots: dcn.GatedScanFunction.step(x, gate, state, slots)  # noqa: E731
    example = [randn(g, 3, 20), randn(g, 3, 20), randn(g, 6, 20)]
    traced = torch.jit.trace(step, (*example, slots), check_trace=False)
    x, gate, pool = randn(g, 3, 20), randn(g, 3, 20), randn(g, 6, 20)
    for _ in range(3):
        want_pool = pool.clone()
        want = dcn.GatedScanFunction.step(x, gate, want_pool, slots)
        assert torch.equal(traced(x, gate, pool, slots), want) and torch.equal(pool, want_pool)
    head = SequenceHead(12, 24, 9, device="cuda")

    class Live(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.head = head

        def forward(self, f, a, b, s):
            return self.head.step(f, [a, b], s)

    live = torch.jit.trace(Live(), (randn(g, 3, 12), *head.new_pool(6), slots), check_trace=False)
    here, there = head.new_pool(6), head.new_pool(6)
    for _ in range(4):
        f = randn(g, 3, 12)
        assert torch.equal(live(f, *here, slots), head.step(f, there, slots))
        assert all(torch.equal(a, b) for a, b in zip(here, there))
    assert all(bool(a[slots].any()) for a in here)


def test_steps_refuse_derivatives_and_transforms():
    import torch.autograd.forward_ad as fwad
    g = gen(7)
    x, gate, pool = randn(g, 3, 20), randn(g, 3, 20), randn(g, 3, 20)
    before = pool.clone()
    with fwad.dual_level():
        for i in range(3):
            args = [x, gate, pool]
            args[i] = fwad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError), torch.no_grad():
                dcn.GatedScanFunction.step(*args)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a, b, c: dcn.GatedScanFunction.step(a[None], b[None], c[None]))(x, gate, pool)
    assert torch.equal(pool, before)


def test_steps_leave_an_inference_pool_alone_outside_inference_mode():
    g = gen(8)
    x, gate = randn(g, 3, 20), randn(g, 3, 20)
    with torch.inference_mode():
        pool = randn(g, 3, 20)
        before = pool.clone()
    with torch.no_grad(), pytest.raises(RuntimeError, match="nference"):
        dcn.GatedScanFunction.step(x, gate, pool)
    torch.cuda.synchronize()
    assert torch.equal(pool, before)
    with torch.inference_mode():
        y = dcn.GatedScanFunction.step(x, gate, pool)
        assert torch.equal(y, pool) and not torch.equal(pool, before)


# ---- infinite states --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("gates", ["mixed", "slow", "fast"])
@pytest.mark.parametrize("shape", [(1, 5, 3), (2, 40, 70), (1, 64, 5), (2, 130, 33), (1, 1500, 40), (160, 200, 64)])
def test_scan_keeps_infinite_states(shape, gates, kind):
    """They stay what they are while gates are above zero, wherever a thread's, a warp's or a CTA's steps end.  Gates of -8 give a
    product that float32 does not hold after a few of a thread's steps."""
    b, n, c = shape
    g, t = gen(n + c), TYPES[kind]
    mean, std = {"mixed": (1.0, 1.5), "slow": (12.0, 0.5), "fast": (-8.0, 0.5)}[gates]
    x, gate, state = randn(g, b, n, c, dtype=t), randn(g, b, n, c, mean=mean, std=std, dtype=t), randn(g, b, c)
    lengths = torch.randint(1, n + 1, (b,), generator=g, device="cuda")
    lengths[0] = n
    state[0, 0], state[-1, 1] = math.inf, -math.inf
    x[0, n // 2, 2] = math.inf                                # from a step on
    if b > 1:
        lengths[1], state[1, 0] = 0, -math.inf
    dy, dlast = randn(g, b, n, c, dtype=t), randn(g, b, c)
    ins = [v.requires_grad_() for v in (x, gate, state)]
    for le in (None, lengths):
        y, last = dcn.GatedScanFunction.apply(*ins, le)
        w = [wide(v) for v in ins]
        wy, wl = ref.scan(*w, le)
        close(y, wy, "y")
        close(last, wl, "last")
        got = torch.autograd.grad((y, last), ins, (dy, dlast))
        want = torch.autograd.grad((wy, wl), w, (dy.double(), dlast.double()))
        for name, a, v in zip(("dx", "dgate", "dstate"), got, want):
            if name != "dgate":
                close(a, v, name)
            else:                                             # (no number where the state, or x, is infinite)
                there = torch.isfinite(v) & torch.isfinite(a)
                assert bool((there | ~torch.isfinite(v)).all())
                close(torch.where(there, a, 0.0), torch.where(there, v, 0.0), name)


def test_scan_with_an_infinite_state_in_odd_channels_only():
    """Channels beside an infinite one, of its pair and its vectors, are not touched."""
    g = gen(11)
    x, gate, state = randn(g, 2, 300, 64), randn(g, 2, 300, 64, mean=2.0), randn(g, 2, 64)
    y, last = dcn.GatedScanFunction.apply(x, gate, state)
    state[:, 1::2] = math.inf
    z, end = dcn.GatedScanFunction.apply(x, gate, state)
    assert torch.equal(z[..., ::2], y[..., ::2]) and torch.equal(end[:, ::2], last[:, ::2])
    assert bool((z[..., 1::2] == math.inf).all()) and bool((end[:, 1::2] == math.inf).all())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [64, 7])
def test_steps_between_values_of_any_size(kind, channels):
    """An infinite state stays infinite, and finite ones of opposite signs meet in between, however far apart."""
    t = TYPES[kind]
    big = 3e38
    h = torch.tensor([math.inf, -math.inf, math.inf, 1.0, big, -big, big, math.inf, math.nan, 1e30, 2.0], device="cuda")
    x = torch.tensor([1.0, -2.0, math.inf, -math.inf, -big, big, big, -math.inf, 1.0, -1e30, math.nan], device="cuda").to(t)
    for gate in (-3.0, 0.0, 0.25, 9.0):
        pool = h[:, None].repeat(1, channels)
        xs, gs = x[:, None].repeat(1, channels), torch.full((len(x), channels), gate, device="cuda", dtype=t)
        want = ref.scan(xs[:, None].double(), gs[:, None].double(), pool.double())[1]
        y = dcn.GatedScanFunction.step(xs, gs, pool)
        for r in range(len(x)):                               # (a difference of two large values: their rounding)
            close(pool[r], want[r], r, scale=min(float(h[r].abs().nan_to_num(0, 0)), 3e38))
            close(y[r], torch.where(want[r].abs() > torch.finfo(t).max, want[r].sign() * math.inf, want[r]), r,
                  scale=min(float(h[r].abs().nan_to_num(0, 0)), 3e38))


# ---- the head ---------------------------------------------------------------------------------------------------------------
def test_padding_does_not_change_a_training_step():
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead, train_step
    g = gen(13)
    loss = dcn.TopkDistillLoss(4, temperature=1.5)
    x, judged = randn(g, 4, 9, 16), randn(g, 4, 9, 20, std=2.0)
    lengths = torch.tensor([9, 0, 3, 7], device="cuda")
    results = []
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        for clips in (9, 10, 40):
            torch.manual_seed(14)
            head = SequenceHead(16, 32, 20, device="cuda")
            opt = torch.optim.SGD(head.parameters(), lr=0.0)
            features, teacher = randn(g, 4, clips, 16), randn(g, 4, clips, 20)
            features[:, :9], teacher[:, :9] = x, judged
            value = train_step(head, loss, opt, features, loss.teacher(teacher), lengths)
            results.append([value] + [p.grad for p in head.parameters()])
        real = torch.arange(9, device="cuda")[None] < lengths[:, None]
        logits = head(x, lengths=lengths)[0]
        lq, classes = loss.teacher(judged)
        alone = dcn.DistillTopkFunction.apply(logits[real], lq[real], classes[real], 1.5)
        none = train_step(head, loss, opt, x, loss.teacher(judged), torch.zeros_like(lengths))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = tf32
    close(results[0][0], alone.mean().double(), chain=8 * ref.CHAIN)
    for other in results[1:]:                                 # products and sums of another number of rows: another order
        for a, b in zip(other, results[0]):
            close(a, b.double(), chain=8 * ref.CHAIN)
    assert float(none) == 0.0


def test_answers_of_few_classes():
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    head = SequenceHead(8, 16, 3, device="cuda")
    logits = randn(gen(15), 2, 4, 3)
    classes, p, entropy = head.answer(logits)
    assert classes.shape == p.shape == (2, 4, 3) and entropy.shape == (2, 4)
    assert torch.equal(classes, logits.sort(dim=-1, descending=True, stable=True).indices)
    assert head.answer(logits, top=2)[0].shape == (2, 4, 2)


# ---- views and callers --------------------------------------------------------------------------------------------------------
def _negated(t):
    """-t as a view whose memory holds t, as the imaginary part of a conjugate is"""
    v = torch._neg_view(t)
    assert v.is_neg() and v.stride(-1) == 1 and torch.equal(v, -t)
    return v


def test_negated_views():
    g = gen(16)
    x, gate, state = randn(g, 2, 30, 24), randn(g, 2, 30, 24), randn(g, 2, 24)
    logits, tokens = randn(g, 3, 700), torch.tensor([1, 2, 3], device="cuda")
    teacher = randn(g, 3, 700)
    best, places = teacher.topk(5)
    lq = best - teacher.logsumexp(-1, keepdim=True)
    weight = randn(g, 24)
    for fn, args in ((lambda a, b, c: dcn.GatedScanFunction.apply(a, b, c), (x, gate, state)),
                     (lambda a, b, c: dcn.ResidualNormFunction.apply(a, b, None, None, None, c), (x, gate, weight)),
                     (lambda a: dcn.TokenScoresFunction.apply(a, tokens, 3)[:3], (logits,)),
                     (lambda a: (dcn.DistillTopkFunction.apply(a, lq, places),), (logits,)),
                     (lambda a: (dcn.DistillTopkFunction.apply(logits, a, places),), (lq,))):
        wanted = [(-a).requires_grad_(a is not lq) for a in args]
        given = [_negated(a).detach().requires_grad_(a is not lq) for a in args]
        want, got = fn(*wanted), fn(*given)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        if args[0] is lq:
            continue
        gouts = [randn(g, *o.shape) for o in want]
        for a, b in zip(torch.autograd.grad(got, given, [_negated(v) for v in gouts]), torch.autograd.grad(want, wanted, [-v for v in gouts])):
            assert torch.equal(a, b)
    pool, same = state.clone(), state.clone()
    assert torch.equal(dcn.GatedScanFunction.step(_negated(x[:, 0]), _negated(gate[:, 0]), pool),
                       dcn.GatedScanFunction.step(-x[:, 0], -gate[:, 0], same)) and torch.equal(pool, same)
    with pytest.raises(dcn.DcnError, match="state"):
        dcn.GatedScanFunction.step(x[:, 0], gate[:, 0], _negated(state))


def test_compiled_callers_keep_the_operators():
    g = gen(17)
    x, gate, state = randn(g, 2, 30, 24), randn(g, 2, 30, 24), randn(g, 2, 24)
    logits, tokens = randn(g, 3, 700), torch.tensor([1, 2, 3], device="cuda")
    lq, places = torch.full((3, 4), -2.0, device="cuda"), torch.arange(4, device="cuda").expand(3, 4).contiguous()
    for fn, args in ((lambda a, b, c: dcn.GatedScanFunction.apply(a * 2, b, c)[0].relu(), (x, gate, state)),
                     (lambda a, b: dcn.ResidualNormFunction.apply(a * 2, b)[1].relu(), (x, gate)),
                     (lambda a: sum(o.sum() for o in dcn.TokenScoresFunction.apply(a * 2, tokens, 3)[:3]), (logits,)),
                     (lambda a: dcn.DistillTopkFunction.apply(a * 2, lq, places).relu(), (logits,))):
        args = [a.clone().requires_grad_() for a in args]
        y, want = torch.compile(fn, backend="aot_eager")(*args), fn(*args)
        assert torch.allclose(y, want, rtol=1e-6, atol=1e-6)
        for a, b in zip(torch.autograd.grad(y.sum(), args), torch.autograd.grad(want.sum(), args)):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    pool, same = state.clone(), state.clone()
    stepped = torch.compile(lambda a, b, p: dcn.GatedScanFunction.step(a * 2, b, p) + 1, backend="aot_eager")
    for i in range(3):
        want = dcn.GatedScanFunction.step(x[:, i] * 2, gate[:, i], same) + 1
        assert torch.equal(stepped(x[:, i], gate[:, i], pool), want) and torch.equal(pool, same)

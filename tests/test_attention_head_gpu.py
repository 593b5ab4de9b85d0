"""Decayed attention, its heads' norm and sampling as a head over clip features uses them, and the video network with group norms,
against the same in plain torch operations."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _plain(head, features, states=None, lengths=None):
    """SequenceHead.forward in float64, from the definitions"""
    from tests import more_sequence_reference as more
    from tests import sequence_reference as ref
    w = {n: p.detach().double().requires_grad_() for n, p in head.named_parameters()}

    def linear(name, x):
        y = x @ w[name + ".weight"].t()
        return y + w[name + ".bias"] if name + ".bias" in w else y

    stream = linear("embed", features.double())
    normed = ref.residual_norm(stream, pre=w["first.pre_weight"])[1]
    last = []
    for i, block in enumerate(head.blocks):
        b, m = "blocks.%d." % i, block.scan
        q, k, v = linear(b + "scan.proj", normed).split((m.heads * m.dk, m.kv_heads * m.dk, m.kv_heads * m.dv), -1)
        out, end = more.decay_attention(q.unflatten(-1, (m.heads, m.dk)), k.unflatten(-1, (m.kv_heads, m.dk)),
                                        v.unflatten(-1, (m.kv_heads, m.dv)), m.log_decay.double(),
                                        None if states is None else states[i].double(), lengths)
        y = more.group_norm_act(out.flatten(0, 1).flatten(1), m.heads, w[b + "scan.norm.weight"], w[b + "scan.norm.bias"], None, "silu")
        y = y.view(*out.shape[:2], -1)
        stream, normed = ref.residual_norm(stream, linear(b + "out", y), linear(b + "gate", normed), w[b + "norm.scale"],
                                           w[b + "norm.post_weight"], w[b + "norm.pre_weight"])
        last.append(end)
    return linear("fc", normed), last, w


def test_head_trains_like_its_definition():
    from deform_conv3d_pytorch_op_b200 import TopkDistillLoss
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    from tests import sequence_reference as ref
    torch.manual_seed(3)
    head = SequenceHead(24, 48, 30, device="cuda", mixer="attention", heads=4)
    x = torch.randn(5, 21, 24, device="cuda")
    lengths = torch.tensor([21, 0, 7, 20, 1], device="cuda")
    loss = TopkDistillLoss(6, temperature=1.5)
    lq, classes = loss.teacher(torch.randn(5, 21, 30, device="cuda") * 2)
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        logits, last = head(x, lengths=lengths)
        value = loss(logits, lq, classes)
        value.backward()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = tf32
    want, ends, w = _plain(head, x, None, lengths)
    total = ref.distill(want.flatten(0, 1), lq.double().flatten(0, 1), classes.flatten(0, 1), 1.5).mean()
    grads = dict(zip(w, torch.autograd.grad(total, list(w.values()))))
    # two blocks in a row, each with two norms in it, which divide by what may be a small deviation of a head's twelve outputs
    # (up to ten times less than theirs on the way there): eighty times one operator's bound
    close = lambda a, b, n: ref.close(a, b, n, chain=80 * ref.CHAIN)  # noqa: E731
    inside = torch.arange(21, device="cuda")[None, :] < lengths[:, None]
    close(logits[inside], want[inside], "logits")
    close(value, total, "loss")
    for a, b in zip(last, ends):
        close(a, b, "states")
    for n, p in head.named_parameters():
        close(p.grad, grads[n], n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_live_streams_give_the_stored_videos_answers(dtype):
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    torch.manual_seed(4)
    head = SequenceHead(32, 64, 50, device="cuda", dtype=dtype, mixer="attention", heads=2)
    x = torch.randn(4, 30, 32, device="cuda", dtype=dtype)
    with torch.no_grad():
        whole, last = head(x)
        first, states = head(x[:, :11])
        rest, ends = head(x[:, 11:], states)
    pool = head.new_pool(7)
    slots = torch.tensor([6, 0, 3, 2], device="cuda")
    live = torch.stack([head.step(x[:, t], pool, slots) for t in range(30)], 1)
    # as for the scan: the order of the linear layers' sums in float32; in bfloat16 the roundings between the layers, and behind each
    # block a norm that passes them on in full
    tol = 1e-4 if dtype == torch.float32 else 0.1
    size = float(whole.float().abs().max())
    assert float((torch.cat((first, rest), 1) - whole).float().abs().max()) <= tol * size
    assert float((live - whole).float().abs().max()) <= tol * size
    for a, b, c in zip(last, ends, pool):
        big = max(1.0, float(a.abs().max()))
        assert float((a - b).abs().max()) <= tol * big and float((a - c[slots]).abs().max()) <= tol * big
    untouched = [1, 4, 5]
    assert all(float(p[untouched].abs().max()) == 0 for p in pool)


def test_answers_are_drawn():
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    torch.manual_seed(6)
    head = SequenceHead(32, 64, 50, device="cuda", mixer="attention", heads=2)
    with torch.no_grad():
        logits, _ = head(torch.randn(4, 30, 32, device="cuda"))
    best, p, _ = head.answer(logits, top=5)
    drawn, logprob = head.sample(logits, top_k=5)
    assert drawn.shape == (4, 30) and bool((drawn[..., None] == best).any(-1).all())
    q = torch.where(drawn[..., None] == best, p, 0.0).sum(-1) / p.sum(-1)
    assert float((logprob - q.log()).abs().max()) <= 1e-5
    assert torch.equal(head.sample(logits, temperature=0)[0], best[..., 0])
    u = torch.rand(4, 30, device="cuda")
    assert torch.equal(head.sample(logits, u)[0], head.sample(logits, u)[0])


def test_command_runs(capsys):
    from deform_conv3d_pytorch_op_b200 import video_sequence
    video_sequence.main("attention")
    out = capsys.readouterr().out
    assert "drawn answers" in out and "nan" not in out


@pytest.mark.parametrize("storage", [torch.contiguous_format, torch.channels_last_3d])
def test_video_network_with_group_norms(storage):
    """Against the same network with torch's group norm, both in float32, and its step captured"""
    import torch.nn as nn

    from deform_conv3d_pytorch_op_b200 import GroupNormAct
    from deform_conv3d_pytorch_op_b200.r3d import BasicBlock, GraphedTrainStep, R3D18Deform

    class Plain(nn.Module):
        def __init__(self, like):
            super().__init__()
            self.like = like

        def forward(self, x, residual=None):
            n = self.like
            y = nn.functional.group_norm(x, n.groups, n.weight, n.bias, n.eps)
            y = y if residual is None else y + residual
            return y if n.activation is None else torch.relu(y)

    torch.manual_seed(7)
    net = R3D18Deform(num_classes=7, width=16, deform=False, norm="group").cuda().to(memory_format=storage)
    clips = torch.randn(2, 3, 8, 32, 32, device="cuda").to(memory_format=storage)
    labels = torch.tensor([1, 5], device="cuda")
    tf32 = torch.backends.cudnn.allow_tf32
    torch.backends.cudnn.allow_tf32 = False
    try:
        loss = nn.functional.cross_entropy(net(clips), labels)
        loss.backward()
        got = [p.grad.clone() for p in net.parameters()]
        net.zero_grad(set_to_none=True)
        for m in list(net.modules()):
            if isinstance(m, BasicBlock):
                m.bn1, m.bn2 = Plain(m.bn1), Plain(m.bn2)
                if m.down is not None:
                    m.down[1] = Plain(m.down[1])
        net.stem[1] = Plain(net.stem[1])
        want = nn.functional.cross_entropy(net(clips), labels)
        want.backward()
        expected = [p.grad for p in net.parameters()]
    finally:
        torch.backends.cudnn.allow_tf32 = tf32
    # seventeen convolutions of up to 3456 terms a product in a row, in other orders of summation: some tens of roundings each
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-4
    for a, b in zip(got, expected):
        assert float((a - b).norm()) <= 1e-2 * float(b.norm()) + 1e-6

    torch.manual_seed(8)
    net = R3D18Deform(num_classes=7, width=16, norm="group").cuda().to(memory_format=storage)
    assert any(isinstance(m, GroupNormAct) for m in net.modules()) and not any(isinstance(m, nn.BatchNorm3d) for m in net.modules())
    opt = torch.optim.SGD(net.parameters(), lr=0.05)
    step = GraphedTrainStep(net, opt, clips, labels)
    losses = [float(step(clips, labels)) for _ in range(6)]
    assert all(l == l for l in losses)
    assert net.features(clips).shape == (2, 128)


def test_refusals():
    from deform_conv3d_pytorch_op_b200 import DcnError, GroupNormAct
    from deform_conv3d_pytorch_op_b200.r3d import R3D18Deform
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    with pytest.raises(DcnError, match="mixer"):
        SequenceHead(8, 16, 4, mixer="attention", heads=3)
    with pytest.raises(DcnError, match="mixer"):
        SequenceHead(8, 16, 4, mixer="mean")
    with pytest.raises(DcnError, match="do not divide"):
        GroupNormAct(5, 12)
    with pytest.raises(ValueError, match="norm"):
        R3D18Deform(norm="layer")

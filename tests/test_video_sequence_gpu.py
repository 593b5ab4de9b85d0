"""The sequence operators used together: a head over clip features, against the same head in plain torch operations."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _plain(head, features, states=None, lengths=None):
    """SequenceHead.forward in float64, from the definitions"""
    from tests import sequence_reference as ref
    w = {n: p.detach().double().requires_grad_() for n, p in head.named_parameters()}

    def linear(name, x):
        y = x @ w[name + ".weight"].t()
        return y + w[name + ".bias"] if name + ".bias" in w else y

    stream = linear("embed", features.double())
    normed = ref.residual_norm(stream, pre=w["first.pre_weight"])[1]
    last = []
    for i in range(len(head.blocks)):
        b = "blocks.%d." % i
        x, gate = linear(b + "scan.proj", normed).chunk(2, -1)
        y, end = ref.scan(x, gate, None if states is None else states[i].double(), lengths)
        stream, normed = ref.residual_norm(stream, linear(b + "out", y), linear(b + "gate", normed), w[b + "norm.scale"],
                                           w[b + "norm.post_weight"], w[b + "norm.pre_weight"])
        last.append(end)
    return linear("fc", normed), last, w


def test_head_trains_like_its_definition():
    from deform_conv3d_pytorch_op_b200 import TopkDistillLoss
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    from tests import sequence_reference as ref
    torch.manual_seed(3)
    head = SequenceHead(24, 48, 30, device="cuda")
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
    # two blocks in a row, each a few operators and products of up to 48 terms: eight times one operator's bound
    close = lambda a, b, n: ref.close(a, b, n, chain=8 * ref.CHAIN)  # noqa: E731
    close(logits, want, "logits")
    close(value, total, "loss")
    for a, b in zip(last, ends):
        close(a, b, "states")
    for n, p in head.named_parameters():
        close(p.grad, grads[n], n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_live_streams_give_the_stored_videos_answers(dtype):
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    torch.manual_seed(4)
    head = SequenceHead(32, 64, 50, device="cuda", dtype=dtype)
    x = torch.randn(4, 30, 32, device="cuda", dtype=dtype)
    with torch.no_grad():
        whole, last = head(x)
        first, states = head(x[:, :11])
        rest, ends = head(x[:, 11:], states)
    pool = head.new_pool(7)
    slots = torch.tensor([6, 0, 3, 2], device="cuda")
    live = torch.stack([head.step(x[:, t], pool, slots) for t in range(30)], 1)
    # products of the linear layers are summed in an order of the shape's choosing: float32 up to a few 1e-6 of a row's size,
    # bfloat16 a rounding or two of what passes between the layers
    tol = 1e-4 if dtype == torch.float32 else 6e-2
    size = float(whole.float().abs().max())
    assert float((torch.cat((first, rest), 1) - whole).float().abs().max()) <= tol * size
    assert float((live - whole).float().abs().max()) <= tol * size
    for a, b, c in zip(last, ends, pool):
        assert float((a - b).abs().max()) <= tol and float((a - c[slots]).abs().max()) <= tol
    classes, p, entropy = head.answer(whole, top=50)
    assert torch.equal(classes.sort(-1).values, torch.arange(50, device="cuda").expand_as(classes))
    assert float((p.sum(-1) - 1).abs().max()) <= 1e-5 and bool((entropy >= 0).all())


def test_command_learns(capsys):
    from deform_conv3d_pytorch_op_b200 import video_sequence
    video_sequence.main()
    out = capsys.readouterr().out
    losses = [float(line.split()[-1]) for line in out.splitlines() if line.startswith("step")]
    assert losses[-1] < 0.7 * losses[0], out


def test_features_of_the_video_network_feed_the_head():
    from deform_conv3d_pytorch_op_b200.r3d import R3D18Deform
    from deform_conv3d_pytorch_op_b200.video_sequence import SequenceHead
    torch.manual_seed(5)
    net = R3D18Deform(num_classes=10, width=16).cuda().eval()
    head = SequenceHead(8 * 16, 64, 10, device="cuda")
    clips = torch.randn(2 * 3, 3, 8, 32, 32, device="cuda")
    with torch.no_grad():
        f = net.features(clips)
        assert torch.equal(net.fc(f), net(clips))
        logits, _ = head(f.view(2, 3, -1))
    assert logits.shape == (2, 3, 10) and bool(torch.isfinite(logits).all())

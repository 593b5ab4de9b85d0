"""Group norm with an activation against its definition in 64 bits."""
import pytest
import torch

from tests import more_sequence_reference as more
from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu


def check(t, shape, groups, act=None, residual=False, weights="f32", bias=True, mean=0.5, chain=ref.CHAIN, seed=0, eps=1e-5):
    import deform_conv3d_pytorch_op_b200 as dcn
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, w = shape[-1], ref.TYPES[weights] if weights else None

    def normal(*s, dtype=t, std=1.0, mean=0.0):
        return torch.randn(*s, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    x = normal(*shape, std=1.5, mean=mean)
    args = [x, normal(c, dtype=w, std=0.2, mean=1.0) if w else None, normal(c, dtype=w, std=0.2) if w and bias else None,
            normal(*shape) if residual else None]
    leaves = [v.requires_grad_() if v is not None else None for v in args]
    y = dcn.GroupNormActFunction.apply(leaves[0], groups, leaves[1], leaves[2], leaves[3], act, eps)
    assert y.dtype == t and y.shape == x.shape
    wide = [v.detach().double().requires_grad_() if v is not None else None for v in args]
    want = more.group_norm_act(wide[0], groups, wide[1], wide[2], wide[3], act, eps)
    ref.close(y, want, "y", chain=chain)
    dy = normal(*shape)
    got = torch.autograd.grad(y, [v for v in leaves if v is not None], dy)
    expected = torch.autograd.grad(want, [v for v in wide if v is not None], dy.double())
    names = [n for n, v in zip(("dx", "dweight", "dbias", "dresidual"), leaves) if v is not None]
    # (a relu's derivative jumps where z is within a rounding of 0: such elements, and only those, may differ)
    near = None
    if act == "relu":
        near = more.group_norm_act(wide[0], groups, wide[1], wide[2], wide[3], None, eps).abs() < 1e-5
        assert float(near.double().mean()) < 1e-3
    rows = x.numel() // c
    for name, a, b in zip(names, got, expected):
        if name in ("dx", "dresidual") and near is not None and bool(near.any()):
            a, b = torch.where(near, 0, a), torch.where(near, 0, b)
        # sums over all rows of terms of about unit size and any sign; one jump of the relu is one term
        ref.close(a, b, name, chain=chain, scale=rows ** 0.5 if name in ("dweight", "dbias") else 1.0)


@pytest.mark.parametrize("shape,groups", [
    ((1, 1, 1), 1), ((3, 1, 8), 8), ((5, 512), 8), ((2, 7, 30), 5), ((4, 33, 64), 32), ((2, 5, 6, 7, 16), 4), ((3, 1000, 24), 3),
    ((2, 4097, 64), 32), ((1, 20000, 8), 1), ((2, 700, 520), 4), ((1, 3, 8192), 64), ((2, 2, 8191), 1), ((3, 1, 4100), 41),
    ((1, 300, 1026), 2), ((700, 96), 3), ((2, 0, 16), 2), ((0, 4, 16), 2), ((1, 2500, 333), 333)])
@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_shapes(t, shape, groups):
    if 0 in shape:
        import deform_conv3d_pytorch_op_b200 as dcn
        x, w = torch.zeros(shape, device="cuda", dtype=t, requires_grad=True), torch.ones(16, device="cuda", requires_grad=True)
        y = dcn.GroupNormActFunction.apply(x, groups, w, None, None, "relu")
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert dx.shape == x.shape and float(dw.abs().max()) == 0
        return
    if shape[-1] // groups * max(1, int(torch.tensor(shape[1:-1]).prod())) < 2:
        return check(t, shape, groups, weights="f32", eps=1.0)       # (one element a group: x - mean is 0)
    check(t, shape, groups, act="silu", residual=len(shape) == 3)


@pytest.mark.parametrize("act", [None, "none", "relu", "silu"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("t,weights", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", None), ("f32", None)])
def test_forms(t, weights, residual, act):
    for shape in ((3, 100, 48), (2, 5000, 40)):
        check(ref.TYPES[t], shape, 8, act, residual, weights, bias=residual or act is None)


@pytest.mark.parametrize("shape,groups", [
    ((1, 128), 32), ((3000, 128), 32), ((7, 12), 4), ((1500, 60), 20), ((300, 96), 8), ((40, 2048), 16), ((9, 8192), 512),
    ((5, 8190), 2730), ((2001, 256), 1), ((6, 640), 2), ((3, 1050), 30), ((5000, 30), 6), ((1, 7), 1), ((2, 1040), 4)])
@pytest.mark.parametrize("t,weights,act,residual", [("f32", "f32", "silu", True), ("bf16", "bf16", "silu", False), ("bf16", "f32", None, True),
                                                    ("f16", "f16", "relu", False), ("f32", None, None, False)])
def test_single_positions(t, shape, groups, weights, act, residual):
    check(ref.TYPES[t], shape, groups, act, residual, weights, seed=shape[0])


@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_single_positions_each_by_itself(t):
    """A sample's result owes nothing to the others: NaN, infinities and an outlier stay in their groups; odd places in memory"""
    import deform_conv3d_pytorch_op_b200 as dcn
    g = torch.Generator(device="cuda").manual_seed(3)
    flat = torch.randn(601 * 48 + 1, generator=g, device="cuda").to(t)
    x, w = flat[1:].view(601, 48), torch.randn(48, generator=g, device="cuda")
    want = dcn.GroupNormActFunction.apply(x, 4, w, None, None, "silu")
    # (the order of a group's sums is that of the vectors, which the place in memory decides: bits are compared at one place)
    for y in (want, dcn.GroupNormActFunction.apply(x.clone(), 4, w, None, None, "silu")):
        ref.close(y, more.group_norm_act(x.double(), 4, w.double(), None, None, "silu"))
    bad = flat.clone()[1:].view(601, 48)
    bad[5, 3], bad[600, 47], bad[77, 12] = float("nan"), float("inf"), 6e4
    got = dcn.GroupNormActFunction.apply(bad, 4, w, None, None, "silu").view(601, 4, 12)
    ref.close(got[77], more.group_norm_act(bad[77:78].double(), 4, w.double(), None, None, "silu").view(4, 12), "outlier")
    assert bool(torch.isnan(got[5, 0]).all()) and bool(torch.isnan(got[600, 3]).all())
    same = torch.ones(601, 4, dtype=torch.bool, device="cuda")
    same[5, 0] = same[600, 3] = same[77, 1] = False
    assert torch.equal(got[same], want.view(601, 4, 12)[same])


@pytest.mark.parametrize("mean", [100.0, -3000.0])
@pytest.mark.parametrize("shape", [(2, 50, 32), (2, 9000, 32)])
def test_means_far_from_zero(shape, mean):
    # the mean is float32: half a step of it, over a deviation of 1.5, is off in every element
    check(torch.float32, shape, 4, "silu", chain=ref.CHAIN + abs(mean) * 2.0 ** -24, mean=mean)


def test_an_outlier_first():
    """The first position is what variances are summed about"""
    import deform_conv3d_pytorch_op_b200 as dcn
    x = torch.randn(2, 30000, 16, device="cuda")
    x[:, 0] = 1e4
    want = more.group_norm_act(x.double(), 4)
    ref.close(dcn.GroupNormActFunction.apply(x, 4), want, "y")
    x = torch.full((1, 5000, 8), 7.25, device="cuda")               # no variance at all
    assert float(dcn.GroupNormActFunction.apply(x, 2).abs().max()) == 0


def test_video_layout_and_views():
    """[samples, channels, frames, height, width] stored channels last is read as it is; others are copied"""
    import deform_conv3d_pytorch_op_b200 as dcn
    x = torch.randn(2, 32, 3, 9, 7, device="cuda").contiguous(memory_format=torch.channels_last_3d)
    w, b = torch.randn(32, device="cuda"), torch.randn(32, device="cuda")
    y = dcn.GroupNormActFunction.apply(x.movedim(1, -1), 4, w, b, None, "relu").movedim(-1, 1)
    assert y.is_contiguous(memory_format=torch.channels_last_3d)
    ref.close(y, torch.relu(torch.nn.functional.group_norm(x.double(), 4, w.double(), b.double())), "y")
    z = dcn.GroupNormActFunction.apply(x.contiguous().movedim(1, -1), 4, w, b, None, "relu").movedim(-1, 1)
    assert torch.equal(y, z)
    part = torch.randn(4, 50, 80, device="cuda")[:, :, 3:67]
    ref.close(dcn.GroupNormActFunction.apply(part, 8), more.group_norm_act(part.double(), 8), "part")
    odd = torch.randn(4 * 50 * 64 + 1, device="cuda").half()[1:].view(4, 50, 64)
    ref.close(dcn.GroupNormActFunction.apply(odd, 8), more.group_norm_act(odd.double(), 8), "odd")


def test_sums_repeat_and_graphs():
    import deform_conv3d_pytorch_op_b200 as dcn
    x = torch.randn(4, 6000, 64, device="cuda").bfloat16()
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    dy = torch.randn_like(x)

    def run(x):
        leaf = x.detach().requires_grad_()
        y = dcn.GroupNormActFunction.apply(leaf, 8, w, b, None, "silu")
        return (y.detach(),) + torch.autograd.grad(y, (leaf, w, b), dy)

    first = run(x)
    assert all(torch.equal(p, q) for p, q in zip(first, run(x)))
    held = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(p, q) for p, q in zip(first, run(held)))
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(held)
    held.mul_(2.0)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(run(held), out))


def test_refusals():
    import deform_conv3d_pytorch_op_b200 as dcn
    apply = dcn.GroupNormActFunction.apply
    x, w = torch.zeros(2, 5, 12, device="cuda"), torch.ones(12, device="cuda")
    for args, text in [((x.cpu(), 2), "CUDA"), ((x, 5), "do not divide"), ((x, 0), "do not divide"), ((x[0, 0], 2), "expected \\(samples"),
                       ((x, 2, w[:6]), "weight has shape"), ((x, 2, w, w.half()), "bias has dtype"), ((x, 2, w.half()), "weight has dtype"),
                       ((x, 2, w, w, x[:1]), "residual has shape"), ((x, 2, w, w, x.half()), "residual has dtype"),
                       ((x, 2, w, w, x, "tanh"), "activation"), ((x, 2, w, w, x, "relu", -1.0), "eps"), ((x.double(), 2), "float32"),
                       ((torch.zeros(1, 8193, device="cuda"), 1), "8192")]:
        with pytest.raises(dcn.DcnError, match=text):
            apply(*args)
    leaf = x.clone().requires_grad_()
    y = apply(leaf, 2)
    got = torch.autograd.grad(y, leaf, torch.ones_like(y).requires_grad_(), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got.sum().backward()


@pytest.mark.parametrize("shape,groups", [((40, 24), 24), ((40, 24), 12), ((9, 2, 10), 10), ((5, 1, 6, 4), 4)])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_groups_of_one_and_two_elements(t, shape, groups):
    """One element has no gradient; of two, what is left is eps / (var + eps) of terms that cancel: as exact as the same steps in float32"""
    import deform_conv3d_pytorch_op_b200 as dcn
    g = torch.Generator(device="cuda").manual_seed(9)
    c = shape[-1]
    x, dy = (torch.randn(*shape, generator=g, device="cuda").to(t) for _ in range(2))
    w, b = (torch.randn(c, generator=g, device="cuda") for _ in range(2))
    if len(shape) == 4:                              # [5, 1, 6, 4] as one position of 24 channels
        x, dy, w, b, groups, c = x.reshape(5, 24), dy.reshape(5, 24), torch.ones(24, device="cuda"), torch.zeros(24, device="cuda"), 24, 24
    leaf = x.clone().requires_grad_()
    y = dcn.GroupNormActFunction.apply(leaf, groups, w, b)
    dx = torch.autograd.grad(y, leaf, dy)[0]
    split = (x.numel() // c // x.size(0), groups, c // groups)
    v = x.float().reshape(x.size(0), *split)
    d = v - v.mean((1, 3), keepdim=True)
    r = torch.rsqrt(d.square().mean((1, 3), keepdim=True) + 1e-5)
    h = d * r
    dh = (dy.float() * w).reshape(v.shape)
    want = (r * (dh - dh.mean((1, 3), keepdim=True) - h * (dh * h).mean((1, 3), keepdim=True))).reshape(x.shape)
    if split[0] * split[2] == 1:
        assert float(dx.abs().max()) == 0 and torch.equal(y.float(), b.to(t).float().expand_as(y))
    else:
        ref.close(dx, want.double(), "dx")

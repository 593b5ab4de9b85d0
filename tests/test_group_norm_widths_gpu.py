"""Group norm with as many groups as channels, up to the largest numbers of either."""
import pytest
import torch

from tests import more_sequence_reference as more
from tests import sequence_reference as ref
from tests.test_group_norm_gpu import check

pytestmark = pytest.mark.gpu
dcn = pytest.importorskip("deform_conv3d_pytorch_op_b200")


@pytest.mark.parametrize("shape,groups", [((2, 6912), 6912), ((3, 8192), 8192), ((2, 60, 6912), 6912), ((2, 60, 8192), 8192), ((1, 9, 8191), 8191),
                                          ((2, 40, 8190), 4095), ((1, 700, 7168), 7168)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("t", list(ref.TYPES.values()), ids=list(ref.TYPES))
def test_many_groups(t, residual, shape, groups):
    # (of one element a group x - mean is 0: nothing but roundings of 0 is compared, at eps 1)
    check(t, shape, groups, act="silu", residual=residual, eps=1.0 if len(shape) == 2 else 1e-5)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_many_groups_off_16_bytes(t):
    """Vectors of one element: more threads to a row of channels than a CTA has"""
    flat = torch.randn(2 * 30 * 8192 + 1, device="cuda").to(t)
    x, w = flat[1:].view(2, 30, 8192), torch.randn(8192, device="cuda")
    ref.close(dcn.GroupNormActFunction.apply(x, 8192, w, None, None, "relu"), more.group_norm_act(x.double(), 8192, w.double(), None, None, "relu"))


@pytest.mark.parametrize("shape,groups,eps", [((5, 8192), 4096, 1e-5), ((3, 8192), 8192, 1e-5), ((4, 2, 6000), 6000, 1e-5), ((3, 2, 8191), 8191, 1e-5),
                                              ((2, 2, 4400), 4400, 1e-3), ((3, 7000), 3500, 1e-5)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("apart", [False, True])
def test_many_groups_of_one_and_two_elements(t, shape, groups, eps, residual, apart):
    """What is left of two elements' gradient is eps / (var + eps) of terms that cancel, and nothing of one's: as exact as the definition's
    steps in float32, in samples that no CTA holds too"""
    g = torch.Generator(device="cuda").manual_seed(9)
    n, c = shape[0], shape[-1]
    x, dy, res = (torch.randn(*shape, generator=g, device="cuda").to(t) for _ in range(3))
    w, b = (torch.randn(c, generator=g, device="cuda") for _ in range(2))
    if apart:                                        # two elements some 2 apart each: a gradient of 1e-5 of its terms everywhere
        one = torch.where(torch.arange(2, device="cuda") == 0, 1.0, -1.0)
        x = (0.1 * x.float() + (one[:, None] if len(shape) == 3 else one.repeat(c // 2))).to(t)
    leaf = x.clone().requires_grad_()
    y = dcn.GroupNormActFunction.apply(leaf, groups, w, b, res if residual else None, None, eps)
    dx = torch.autograd.grad(y, leaf, dy)[0]
    split = (x.numel() // c // n, groups, c // groups)
    v = x.float().reshape(n, *split)
    d = v - v.mean((1, 3), keepdim=True)
    r = torch.rsqrt(d.square().mean((1, 3), keepdim=True) + eps)
    h = d * r
    dh = (dy.float() * w).reshape(v.shape)
    want = (r * (dh - dh.mean((1, 3), keepdim=True) - h * (dh * h).mean((1, 3), keepdim=True))).reshape(x.shape)
    z = (h.reshape(x.shape).double() * w + b) + (res.double() if residual else 0)
    ref.close(y, z, "y")
    if split[0] * split[2] == 1:
        assert float(dx.abs().max()) == 0
    else:
        ref.close(dx, want.double(), "dx")

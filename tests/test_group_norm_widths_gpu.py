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

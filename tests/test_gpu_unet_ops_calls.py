"""Calls of the UNet operators that their documentation allows and that go wrong
easily: other defaults, saved-tensor hooks, masks and tensors at their limits.
Bounds are unet_ops_plain's."""

import pytest
import torch

import unet_ops_plain as P
from nova_winograd import nova_cross_attention, nova_group_norm
from test_gpu_unet_ops import cross_case, cross_check, near, norm_case, norm_check, rand

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = float("inf")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,C,G,H,W", [(2, 64, 32, 8, 8), (2, 960, 32, 40, 24)])
def test_norm_under_another_default_type(dtype, B, C, G, H, W):
    case = norm_case(B, C, G, H, W, F16, shift=F16)
    want = norm_check(*case, G, "silu")
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        got = norm_check(*case, G, "silu")
    finally:
        torch.set_default_dtype(before)
    assert all(torch.equal(got[n], want[n]) for n in want)

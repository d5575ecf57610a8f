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


class FromCpuInThisLayout:
    """Saved-tensor hooks that keep what is saved on the CPU, with other strides."""

    def __init__(self):
        self.hooks = torch.autograd.graph.saved_tensors_hooks(self.pack, lambda t: t.cuda())

    @staticmethod
    def pack(t):
        last = t.dim() - 1
        return t.cpu().transpose(0, last).contiguous().transpose(0, last)


@pytest.mark.parametrize("hooks", [
    lambda: torch.autograd.graph.save_on_cpu(),
    lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    lambda: FromCpuInThisLayout().hooks,
], ids=["cpu", "pinned", "transposed"])
@pytest.mark.parametrize("sliced", [False, True])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_norm_with_saved_tensors_kept_elsewhere(hooks, sliced, dtype):
    x, w, b, s, dy = norm_case(2, 64, 4, 7, 9, dtype, shift=dtype)
    if sliced:
        wide = torch.zeros(2, 7, 9, 100, device="cuda", dtype=dtype).permute(0, 3, 1, 2)
        wide[:, 8:72] = x
        x = wide[:, 8:72]
    want = norm_check(x, w, b, s, dy, 4, "silu")
    with hooks():
        got = norm_check(x, w, b, s, dy, 4, "silu")
    # A slice's copy may be read in wider vectors: other sums, the same bounds.
    assert sliced or all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("hooks", [
    lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    lambda: FromCpuInThisLayout().hooks,
], ids=["pinned", "transposed"])
@pytest.mark.parametrize("Nk", [77, 300])
@pytest.mark.parametrize("mask", [None, "bool", "f16"])
def test_cross_with_saved_tensors_kept_elsewhere(hooks, Nk, mask):
    q, k, v, m, do = cross_case(3, 150, Nk, 2, 40, F16, mask)
    kv = torch.stack([k, v], 2)  # k and v as parts of one projection
    want = cross_check(q, kv[:, :, 0], kv[:, :, 1], m, do)
    with hooks():
        got = cross_check(q, kv[:, :, 0], kv[:, :, 1], m, do)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,Nk,tile", [(64, 300, 112), (160, 200, 80)])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -12, 2.0 ** -6])
def test_cross_values_small_in_one_tile_of_keys(dtype, D, Nk, tile, which, size):
    """Padded encoder states through a projection without bias: v is zero, or far
    smaller, for some keys.  What dP - delta comes to there is delta, from the others.
    The bound's step of the smallest dS holds: |delta| is at most the largest |dp|."""
    q, k, v, _, do = cross_case(2, 150, Nk, 2, D, dtype)
    v[:, which * tile:(which + 1) * tile] *= size
    cross_check(q, k, v, None, do)

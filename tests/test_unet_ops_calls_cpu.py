"""What the UNet operators hand to the library, on a CPU-only machine: the library
call is recorded in place of being made."""

import pytest
import torch

from nova_winograd import unet_ops


@pytest.fixture
def calls(monkeypatch):
    """The library's calls, (name, arguments), and no kernel; every size query gives 0."""
    made = []
    monkeypatch.setattr(unet_ops, "_call", lambda name, device, *args: made.append((name, args)))
    monkeypatch.setattr(unet_ops, "_workspace", lambda name, device, *sizes: (None, None, 0))
    return made


@pytest.fixture
def default_dtype():
    before = torch.get_default_dtype()
    yield torch.set_default_dtype
    torch.set_default_dtype(before)


def cl(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).to(memory_format=torch.channels_last)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float64])
def test_statistics_are_32_bits_whatever_the_default_type(calls, default_dtype, dtype):
    """The kernels write float[2][B][groups] and float[B][H][Nq]."""
    default_dtype(dtype)
    x = cl(2, 8, 4, 4)
    stats = unet_ops._norm_forward(x, (128, 8), 4, None, None, 1e-5, 0, None, True)[1]
    assert stats.dtype == torch.float32 and stats.shape == (2, 2, 4)
    q = torch.zeros(2, 3, 2, 16, dtype=torch.float16)
    lse = unet_ops._cross_forward(q, q, q, None, 0.25, True)[2]
    assert lse.dtype == torch.float32 and lse.shape == (2, 2, 3)
    assert [c[0] for c in calls] == ["nova_group_norm_v2", "nova_cross_attention_v2"]

"""What the UNet operators hand to the library, on a CPU-only machine: the library
call is recorded in place of being made."""

import pytest
import torch
from torch.autograd import forward_ad

from nova_winograd import ops, unet_ops


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


class Hooks:
    """Saved-tensor hooks that hand back ``again(tensor)``, and remember what."""

    def __init__(self, again):
        self.again, self.given = again, []

    def __enter__(self):
        def unpack(t):
            self.given.append(self.again(t))
            return self.given[-1]
        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack)
        return self.hooks.__enter__()

    def __exit__(self, *args):
        return self.hooks.__exit__(*args)


@pytest.mark.parametrize("sliced", [False, True])
def test_norm_gradient_goes_by_the_strides_of_what_hooks_hand_back(calls, sliced):
    # Channels 8 .. 15 of 32: pixel pitch 32 as it is, 8 in a compact copy.
    x = cl(2, 32, 4, 5)[:, 8:16] if sliced else cl(2, 8, 4, 5)
    compact = dict(memory_format=torch.channels_last if sliced else torch.contiguous_format)
    with Hooks(lambda t: t.clone(**compact) if t.dim() == 4 else t.clone()):
        y = unet_ops._GroupNorm.apply(x.requires_grad_(), None, None, None,
                                      unet_ops._pixel_strides(x), 2, 1e-5, 0)
        y.backward(torch.zeros_like(y))
    name, args = calls[-1]
    assert name == "nova_group_norm_grad_v2"
    assert args[16:18] == (4 * 5 * 8, 8)  # batch and pixel stride of x


def test_norm_gradient_copies_what_no_strides_fit(calls):
    x = cl(2, 8, 4, 5)
    hooks = Hooks(lambda t: t.clone(memory_format=torch.contiguous_format))
    with hooks:
        y = unet_ops._GroupNorm.apply(x.requires_grad_(), None, None, None, (160, 8), 2, 1e-5, 0)
        y.backward(torch.zeros_like(y))
    assert calls[-1][1][0] not in [t.data_ptr() for t in hooks.given]  # NCHW memory


def test_cross_gradient_takes_rows_as_hooks_hand_them_back(calls):
    def heads_first(t):  # every 4-D tensor with its heads before its tokens, off 16 bytes
        if t.dim() != 4:
            return torch.stack([t, t], -1)[..., 0]
        B, N, H, D = t.shape
        return torch.zeros(B, H, N, D + 1, dtype=t.dtype)[..., 1:].transpose(1, 2)
    q = torch.zeros(2, 3, 2, 16, dtype=torch.float16, requires_grad=True)
    k = torch.zeros(2, 200, 2, 16, dtype=torch.float16)
    hooks = Hooks(heads_first)
    with hooks:
        o = unet_ops._CrossAttention.apply(q, k, k, None, 0.25)
        o.backward(torch.zeros_like(o))
    name, args = calls[-1]
    assert name == "nova_cross_attention_grad_v2"
    given = [t.data_ptr() for t in hooks.given]
    assert len(given) == 6  # q, k, v, o, low, lse
    assert all(args[i] not in given for i in (0, 1, 2, 4, 5, 7))
    dense = [200 * 32, 32, 16]
    assert list(args[18]) == [3 * 32, 32, 16] + dense + dense + [0, 0] + [3 * 32, 32, 16]


@pytest.mark.parametrize("again", [lambda t: t.double(), lambda t: t[:1], lambda t: t.to("meta")])
def test_other_tensors_from_hooks_are_refused(calls, again):
    x = cl(2, 8, 4, 5)
    with Hooks(again):
        y = unet_ops._GroupNorm.apply(x.requires_grad_(), None, None, None, (160, 8), 2, 1e-5, 0)
        with pytest.raises(RuntimeError, match="hook"):
            y.backward(torch.zeros_like(y))
    q = torch.zeros(2, 3, 2, 16, dtype=torch.float16, requires_grad=True)
    with Hooks(again):
        o = unet_ops._CrossAttention.apply(q, q, q, None, 0.25)
        with pytest.raises(RuntimeError, match="hook"):
            o.backward(torch.zeros_like(o))
    assert not any("grad" in c[0] for c in calls)


def test_workspace_sizes_are_asked_for_each_device(monkeypatch):
    """Two devices may have another number of SMs, hence other splits: the size is
    asked with the operands' device current, and kept for that device alone."""
    current, asked = [0], []

    class On:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *args):
            current[0] = self.before

    def size(*sizes):
        asked.append((current[0], sizes))
        return 0

    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(unet_ops, "_fn", lambda name: size)
    monkeypatch.setattr(unet_ops, "_workspace_sizes", {})
    for index in (1, 0, 1, 2):
        assert unet_ops._workspace("x_workspace_bytes", torch.device("cuda", index), 3, 4)[2] == 0
    assert asked == [(1, (3, 4)), (0, (3, 4)), (2, (3, 4))]
    assert current == [0]


@pytest.mark.parametrize("sizes", [(6, 5727, 2640, 8), (1, 9606, 1088, 16), (29, 7956, 1016, 4),
                                   (8, 4096, 320, 32), (1, 64, 1280, 32)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("grad", [0, 1])
def test_workspace_for_unknown_alignment_does_for_both(sizes, dtype, grad):
    lib = ops.load_library(ops._find_lib())
    unknown, aligned = (lib.nova_group_norm_workspace_bytes(*sizes, dtype, a, grad) for a in (0, 1))
    assert unknown >= aligned >= 0


def test_rows_off_16_bytes_are_copied_although_contiguous():
    flat = torch.arange(1 + 2 * 5 * 2 * 16, dtype=torch.float16)
    t = flat[1:].view(2, 5, 2, 16)
    assert t.is_contiguous() and t.data_ptr() % 16
    one = torch.zeros(3 * 164, dtype=torch.float16).as_strided((3, 5, 2, 16), (164, 32, 16, 1))[:1]
    assert one.is_contiguous() and one.stride(0) % 8  # the stride of a single sample
    token = torch.zeros(2, 1, 2, 16, dtype=torch.float16).as_strided((2, 1, 2, 16), (32, 3, 16, 1))
    for x in (t, one, token):
        y = unet_ops._rows(x)
        assert torch.equal(x, y) and y.data_ptr() % 16 == 0
        assert all(s % 8 == 0 for s in y.stride()[:3]) and y.stride(1) > 0
    dense = torch.zeros(2, 5, 2, 16, dtype=torch.float16)
    assert unet_ops._rows(dense) is dense


@pytest.mark.parametrize("B,HW,C,G", [(1, 2 ** 31 - 4096, 1, 1), (1, 2 ** 31 - 4096, 24, 3),
                                      (1, 2 ** 31 - 4096, 4, 2), (3, 715826517, 2, 2),
                                      (2 ** 31 - 4096, 1, 1, 1), (2 ** 20, 2047, 8, 2)])
def test_workspace_of_the_most_pixels(B, HW, C, G):
    """Up to 2^31 - 4096 pixels and groups; a part of 12 bytes at most for a channel of
    a block, of which a sample has at most 8 for each of 148 SMs, and the samples' sums."""
    size = ops.load_library(ops._find_lib()).nova_group_norm_workspace_bytes
    assert B * HW <= 2 ** 31 - 4096
    for dtype in (0, 1, 2):
        for aligned in (0, 1):
            for grad in (0, 1):
                n = size(B, HW, C, G, dtype, aligned, grad)
                assert 0 <= n <= 12 * C * (B + max(B, 8 * 148)) + 512
    assert size(1, 2 ** 31 - 4095, 1, 1, 0, 0, 0) == -1
    assert size(2 ** 16, 2 ** 16, 1, 1, 0, 0, 0) == -1
    assert size(2 ** 27, 1, 64, 32, 0, 0, 0) == -1


def test_tangents_reach_the_functions_that_refuse_them(calls):
    x, q = cl(2, 8, 4, 5), torch.zeros(2, 3, 2, 16, dtype=torch.float16)
    assert not unet_ops._differentiated(x, None)
    for grad in (False, True):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            assert unet_ops._differentiated(dual, None)
            with pytest.raises(NotImplementedError):
                unet_ops._GroupNorm.apply(dual, None, None, None, (160, 8), 2, 1e-5, 0)
            dual = forward_ad.make_dual(q, torch.ones_like(q))
            for at in range(3):
                qkv = [q, q, q]
                qkv[at] = dual
                with pytest.raises(NotImplementedError):
                    unet_ops._CrossAttention.apply(*qkv, None, 0.25)
            # Without a tangent the level changes nothing.
            assert unet_ops._GroupNorm.apply(x, None, None, None, (160, 8), 2, 1e-5, 0).shape == x.shape
    x.requires_grad_()
    assert unet_ops._differentiated(None, x)
    with torch.no_grad():
        assert not unet_ops._differentiated(None, x)


def test_norm_refuses_what_the_library_would():
    x = torch.empty(1, 2 * 8193, 1, 1, dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="8192 channels"):
        unet_ops.nova_group_norm(x, 2)
    many = torch.empty(2 ** 26, 64, 1, 1, dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="groups"):
        unet_ops.nova_group_norm(many, 64)
    with pytest.raises(ValueError, match="CUDA"):
        unet_ops.nova_group_norm(torch.empty(1, 2 * 8192, 1, 1, dtype=torch.float16, device="meta"), 2)

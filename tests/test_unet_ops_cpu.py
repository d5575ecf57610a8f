"""Group norm and cross attention on a CPU-only machine: what the public entry
points and the C entry points refuse (nothing is launched here), and the plain
forms that the GPU tests compare with, against torch's."""

import ctypes
import os

import pytest
import torch
import torch.nn.functional as F

import nova_winograd
from nova_winograd import NovaGroupNorm, nova_cross_attention, nova_group_norm, ops
from nova_winograd.unet_ops import _pixel_strides

import unet_ops_plain as P


@pytest.fixture(scope="module")
def lib():
    return ops.load_library(ops._find_lib())


def cl(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).to(memory_format=torch.channels_last)


@pytest.mark.parametrize("args,kw,error", [
    ((torch.zeros(2, 8, 4, dtype=torch.float16), 2), {}, ValueError),
    ((cl(2, 8, 4, 4, dtype=torch.float64), 2), {}, TypeError),
    ((cl(2, 8, 4, 4, dtype=torch.int32), 2), {}, TypeError),
    ((cl(2, 8, 4, 4), 3), {}, ValueError),
    ((cl(2, 8, 4, 4), 0), {}, ValueError),
    ((cl(2, 8, 4, 4), 2), {"activation": "gelu"}, ValueError),
    ((cl(2, 8, 4, 4), 2), {"eps": -1e-5}, ValueError),
    ((cl(2, 8, 4, 4), 2), {"eps": float("nan")}, ValueError),
    ((torch.zeros(2, 8, 4, 4, dtype=torch.float16), 2), {}, ValueError),           # NCHW
    ((cl(2, 8, 4, 4)[:, :, :, ::2], 2), {"weight": torch.ones(7)}, ValueError),
    ((cl(2, 8, 4, 6)[:, :, :, :4], 2), {}, ValueError),                             # cropped rows
    ((cl(2, 8, 1, 1).expand(2, 8, 4, 4), 2), {}, ValueError),                       # one pixel, spread
    ((cl(2, 8, 4, 4), 2), {"weight": torch.ones(4)}, ValueError),
    ((cl(2, 8, 4, 4), 2), {"weight": torch.ones(8, dtype=torch.float64)}, TypeError),
    ((cl(2, 8, 4, 4), 2), {"weight": torch.ones(8), "bias": torch.ones(8).half()}, TypeError),
    ((cl(2, 8, 4, 4), 2), {"shift": torch.ones(8)}, ValueError),
    ((cl(2, 8, 4, 4), 2), {"shift": torch.ones(1, 8)}, ValueError),
    ((cl(2, 8, 4, 4), 2), {}, ValueError),                                          # on the CPU
])
def test_group_norm_refuses(args, kw, error):
    with pytest.raises(error):
        nova_group_norm(*args, **kw)


def qkv(B=2, Nq=3, Nk=5, H=2, D=16, dtype=torch.float16):
    return [torch.zeros(B, n, H, D, dtype=dtype) for n in (Nq, Nk, Nk)]


@pytest.mark.parametrize("args,kw,error", [
    (qkv(dtype=torch.float32), {}, TypeError),
    (qkv(D=12), {}, ValueError),
    (qkv(D=168), {}, ValueError),
    ((qkv()[0][0], *qkv()[1:]), {}, ValueError),
    ((qkv()[0], qkv()[1].bfloat16(), qkv()[2]), {}, TypeError),
    ((qkv()[0], qkv()[1], qkv(Nk=4)[2]), {}, ValueError),
    ((qkv()[0], *qkv(H=1)[1:]), {}, ValueError),                                    # shared heads
    ((qkv()[0], *qkv(B=1)[1:]), {}, ValueError),
    (qkv(), {"key_mask": torch.ones(2, 4, dtype=torch.bool)}, ValueError),
    (qkv(), {"key_mask": torch.ones(5, dtype=torch.bool)}, ValueError),
    (qkv(), {"key_mask": torch.ones(2, 5, dtype=torch.int64)}, TypeError),
    (qkv(), {"key_mask": torch.ones(2, 5, dtype=torch.float64)}, TypeError),
    (qkv(), {"key_mask": torch.ones(2, 5).requires_grad_()}, ValueError),
    (qkv(), {}, ValueError),                                                        # on the CPU
])
def test_cross_attention_refuses(args, kw, error):
    with pytest.raises(error):
        nova_cross_attention(*args, **kw)


def test_sizes_past_32_bits_are_refused():
    # The library counts pixels and rows in 32 bits: 2^32 + 65536 must not become 65536.
    x = torch.empty(1, 1, 65536, 65537, dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="pixels"):
        nova_group_norm(x, 1)
    q = torch.empty(1, 1, 1, 8, dtype=torch.float16, device="meta")
    k = torch.empty(1, 2 ** 32 + 5, 1, 8, dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="rows"):
        nova_cross_attention(q, k, k)
    with pytest.raises(ValueError, match="rows"):
        nova_cross_attention(k, q, q)


def test_module_refuses_and_shares_parameters():
    with pytest.raises(ValueError):
        NovaGroupNorm(4, 8, activation="relu")
    norm = torch.nn.GroupNorm(4, 8, eps=1e-6)
    new = NovaGroupNorm.from_group_norm(norm, "silu")
    assert new.weight is norm.weight and new.bias is norm.bias
    assert (new.eps, new.num_groups, new.num_channels, new.activation) == (1e-6, 4, 8, "silu")
    plain = NovaGroupNorm.from_group_norm(torch.nn.GroupNorm(4, 8, affine=False))
    assert plain.weight is None and plain.bias is None and plain.activation is None


def test_names_are_reachable_from_the_package():
    for name in ("nova_group_norm", "nova_cross_attention", "NovaGroupNorm"):
        assert hasattr(nova_winograd, name)


@pytest.mark.parametrize("shape,layout,want", [
    ((2, 8, 4, 5), "cl", (160, 8)),
    ((1, 8, 4, 5), "cl", (0, 8)),
    ((2, 8, 1, 5), "cl", (40, 8)),
    ((2, 8, 4, 1), "cl", (32, 8)),
    ((2, 8, 1, 1), "nchw", (8, 8)),
    ((2, 1, 4, 5), "nchw", (20, 1)),
    ((2, 8, 4, 5), "nchw", None),
    ((2, 8, 4, 1), "nchw", None),
])
def test_pixel_strides(shape, layout, want):
    x = torch.zeros(shape)
    if layout == "cl":
        x = x.contiguous(memory_format=torch.channels_last)
    assert _pixel_strides(x) == want
    if want:
        # The same tensor as channels 8..8+C of a wider one.
        wide = cl(shape[0], shape[1] + 24, *shape[2:])[:, 8:8 + shape[1]]
        pixels = shape[2] * shape[3]
        assert _pixel_strides(wide) == (
            (shape[1] + 24) * pixels if shape[0] > 1 else 0,
            shape[1] + 24 if pixels > 1 else shape[1])


def norm_args(**kw):
    a = dict(x=16, w=16, b=16, s=16, y=16, stats=16, ws=256, n=1 << 20, B=1, HW=4, C=8, G=2, sb=32,
             sp=8, t=0, wt=2, st=2, act=0, eps=1e-5)
    a.update(kw)
    return [*a.values(), None]


# More than the resident form holds: a workspace is needed.
BIG = {"B": 8, "HW": 1 << 16, "C": 64, "G": 2, "sb": 1 << 22, "sp": 64}


@pytest.mark.parametrize("kw,status", [
    ({"x": None}, 1), ({"y": None}, 1), ({"ws": None, **BIG}, 1), ({"ws": 128, **BIG}, 1), ({"B": 0}, 1),
    ({"HW": 0}, 1), ({"C": 0}, 1), ({"G": 0}, 1), ({"G": 3}, 1), ({"sp": 7}, 1), ({"sb": -1}, 1),
    ({"t": 3}, 1), ({"wt": -1}, 1), ({"act": 2}, 1), ({"eps": -1.0}, 1),
    ({"B": 1 << 20, "HW": 1 << 20}, 1), ({"n": 8, **BIG}, 3),
])
def test_group_norm_entry_validates(lib, kw, status):
    assert lib.nova_group_norm_v2(*norm_args(**kw)) == status
    assert b"group_norm" in lib.nova_last_error_string()


def test_group_norm_grad_entry_validates(lib):
    def call(**kw):
        a = dict(x=16, dy=16, w=16, b=16, s=16, stats=16, dx=16, dw=16, db=16, ds=16, ws=256,
                 n=1 << 20, B=1, HW=4, C=8, G=2, sb=32, sp=8, gb=32, gp=8, t=0, wt=2, st=2, act=0)
        a.update(kw)
        return lib.nova_group_norm_grad_v2(*a.values(), None)
    for kw in ({"x": None}, {"dy": None}, {"stats": None}, {"dx": None}, {"gp": 4}, {"act": -1},
               {"gb": -8}):
        assert call(**kw) == 1, kw
    assert call(n=0) == 3
    assert lib.nova_group_norm_workspace_bytes(1, 4, 8, 3, 0, 1, 0) == -1
    assert lib.nova_group_norm_workspace_bytes(0, 4, 8, 2, 0, 1, 1) == -1
    assert lib.nova_group_norm_workspace_bytes(1, 4, 8, 2, 3, 1, 1) == -1
    assert lib.nova_group_norm_workspace_bytes(1, 4, 8, 2, 0, 1, 0) == 0


def cross_strides(B, Nq, Nk, H, D, **kw):
    v = [Nq * H * D, H * D, D, Nk * H * D, H * D, D, Nk * H * D, H * D, D, Nk, 1, Nq * H * D, H * D, D]
    for i, x in kw.items():
        v[int(i[1:])] = x
    return (ctypes.c_longlong * 14)(*v)


@pytest.mark.parametrize("kw,status", [
    ({"q": None}, 1), ({"k": None}, 1), ({"v": None}, 1), ({"o": None}, 1), ({"q": 8}, 1),
    ({"o": 8}, 1), ({"B": 0}, 1), ({"Nq": 0}, 1), ({"Nk": 0}, 1), ({"H": 0}, 1), ({"D": 12}, 1),
    ({"D": 168}, 1), ({"D": 0}, 1), ({"t": 2}, 1), ({"mt": 4}, 1), ({"mt": -2}, 1),
    ({"mt": 3, "m": None}, 1), ({"st": None}, 1),
    ({"st": cross_strides(1, 4, 4, 2, 16, i1=33)}, 1),
    ({"st": cross_strides(1, 4, 4, 2, 16, i4=-32)}, 1),
    ({"st": cross_strides(1, 4, 4, 2, 16, i9=-1)}, 1),
    ({"st": cross_strides(1, 4, 4, 2, 16, i4=0)}, 1), ({"low": 8}, 1),
    ({"B": 1 << 20, "Nq": 1 << 10, "H": 2}, 1), ({"Nk": (1 << 30) + 1}, 1),
])
def test_cross_attention_entry_validates(lib, kw, status):
    a = dict(q=16, k=16, v=16, m=16, o=16, low=None, lse=16, ws=256, n=1 << 40, B=1, Nq=4, Nk=4, H=2, D=16,
             st=cross_strides(1, 4, 4, 2, 16), t=0, mt=-1, scale=1.0)
    a.update(kw)
    assert lib.nova_cross_attention_v2(*a.values(), None) == status
    assert b"cross_attention" in lib.nova_last_error_string()


def test_cross_attention_grad_entry_validates(lib):
    def call(**kw):
        a = dict(q=16, k=16, v=16, m=16, o=16, low=16, do=16, lse=16, dq=16, dk=16, dv=16, ws=256,
                 n=1 << 40, B=1, Nq=4, Nk=4, H=2, D=16, st=cross_strides(1, 4, 4, 2, 16), t=0,
                 mt=-1, scale=1.0)
        a.update(kw)
        return lib.nova_cross_attention_grad_v2(*a.values(), None)
    long = {"Nk": 300, "st": cross_strides(1, 4, 300, 2, 16)}
    for kw in ({"o": None, **long}, {"low": None, **long}, {"low": 8, **long}, {"do": None}, {"lse": None}, {"dq": None}, {"dk": None}, {"dv": None},
               {"do": 8}, {"dk": 8}, {"st": cross_strides(1, 4, 4, 2, 16, i12=20)}):
        assert call(**kw) == 1, kw
    # More keys than one tile: a workspace is needed.
    assert lib.nova_cross_attention_workspace_bytes(1, 4, 300, 2, 16, 1) > 0
    assert call(n=0, **long) == 3
    assert call(ws=None, **long) == 1
    assert call(ws=128, **long) == 1
    assert lib.nova_cross_attention_workspace_bytes(1, 4, 4, 2, 12, 0) == -1


# ---- the plain forms themselves ---------------------------------------------

@pytest.mark.parametrize("act", [None, "silu"])
def test_plain_group_norm_is_torchs(act):
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 12, 5, 3), (12,), (12,)))
    s, dy = (torch.randn(*t, generator=g, dtype=torch.float64) for t in ((2, 12), (2, 12, 5, 3)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b, s)]
    y = F.group_norm(leaves[0] + leaves[3][:, :, None, None], 4, leaves[1], leaves[2], 1e-5)
    y = F.silu(y) if act else y
    want = (y, *torch.autograd.grad(y, leaves, dy))
    got = P.group_norm(x, 4, w, b, 1e-5, act, s, dy)
    for name, t in zip(("y", "dx", "dw", "db", "ds"), want):
        assert torch.allclose(got[name], t, rtol=1e-10, atol=1e-12), name


@pytest.mark.parametrize("mask", [None, "bool", "bias"])
def test_plain_cross_attention_is_torchs(mask):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(3, n, 2, 8, generator=g, dtype=torch.float64) for n in (4, 6, 6))
    do = torch.randn(3, 4, 2, 8, generator=g, dtype=torch.float64)
    m = None
    if mask:
        m = torch.rand(3, 6, generator=g) < 0.6
        m[:, 0] = True
        if mask == "bias":
            m = torch.where(m, torch.randn(3, 6, generator=g, dtype=torch.float64), float("-inf"))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = F.scaled_dot_product_attention(*(t.transpose(1, 2) for t in leaves),
                                       attn_mask=None if m is None else m[:, None, None, :])
    o = o.transpose(1, 2)
    want = (o, *torch.autograd.grad(o, leaves, do))
    got = P.cross_attention(q, k, v, m, 8 ** -0.5, do)
    for name, t in zip(("o", "dq", "dk", "dv"), want):
        assert torch.allclose(got[name], t, rtol=1e-9, atol=1e-12), name

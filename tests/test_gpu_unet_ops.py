"""Group norm and cross attention against their plain forms in 64 bits, with the
bounds that unet_ops_plain derives, and what their users do with them: other
layouts, streams, graphs, masks that leave nothing, a UNet's block."""

import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import unet_ops_plain as P
from nova_winograd import NovaGroupNorm, nova_cross_attention, nova_group_norm

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = float("inf")


def rand(*shape, seed, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def near(got, want, tol, what):
    got = got.double()
    assert torch.isfinite(got).all(), what
    off = (got - want).abs() / tol
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 1, f"{what}: {worst:.3g} times the bound"


# ---------------------------------------------------------------------------
# Group norm
# ---------------------------------------------------------------------------

def norm_case(B, C, G, H, W, dtype, act=None, shift=None, wtype=F32, spread=1.0, mean=0.5, seed=0):
    x = (spread * rand(B, H, W, C, seed=seed) + mean * rand(C, seed=seed + 1)).to(dtype)
    x = x.permute(0, 3, 1, 2)
    w = (1 + 0.2 * rand(C, seed=seed + 2)).to(wtype) if wtype else None
    b = (0.2 * rand(C, seed=seed + 3)).to(wtype) if wtype else None
    s = (0.5 * rand(B, C, seed=seed + 4)).to(shift) if shift else None
    dy = rand(B, H, W, C, seed=seed + 5, dtype=dtype).permute(0, 3, 1, 2)
    return x, w, b, s, dy


def norm_check(x, w, b, s, dy, G, act, eps=1e-5):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b, s)]
    y = nova_group_norm(leaves[0], G, leaves[1], leaves[2], eps, act, leaves[3])
    assert y.dtype == x.dtype and y.shape == x.shape
    assert y.is_contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        assert torch.equal(nova_group_norm(x, G, w, b, eps, act, s), y)
    have = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, have, dy))
    got = {"y": y.detach()}
    for name, t in zip(("dx", "dw", "db", "ds"), leaves):
        if t is not None:
            got[name] = next(grads)
            assert got[name].dtype == t.dtype and got[name].shape == t.shape
    d = [None if t is None else t.detach().double() for t in (x, w, b, s, dy)]
    types = (x.dtype, F32 if w is None else w.dtype, F32 if s is None else s.dtype)
    want = P.group_norm(d[0], G, d[1], d[2], eps, act, d[3], d[4], types)
    for name, t in got.items():
        near(t, want[name], want[name + "_tol"], name)
    return got


@pytest.mark.parametrize("B,C,G,H,W", [
    (1, 1280, 32, 8, 8), (2, 320, 32, 16, 16), (3, 190, 10, 37, 29), (2, 8, 1, 1, 1),
    (1, 8, 8, 3, 1), (2, 3, 1, 5, 7), (1, 1, 1, 9, 9), (5, 64, 4, 1, 33), (2, 2560, 32, 4, 4),
    (1, 2048, 1, 2, 3), (1, 4104, 8, 3, 3), (1, 320, 32, 129, 65), (3, 96, 3, 2, 2),
    (2, 960, 32, 40, 24), (17, 40, 4, 3, 3),
])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_norm_shapes(B, C, G, H, W, dtype):
    norm_check(*norm_case(B, C, G, H, W, dtype, shift=dtype), G, "silu")


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("shift", [None, F16, F32])
@pytest.mark.parametrize("wtype", [None, F16, F32])
def test_norm_options(act, shift, wtype):
    norm_check(*norm_case(2, 80, 8, 11, 13, F16, shift=shift, wtype=wtype), 8, act)


def test_norm_weight_or_bias_alone():
    x, w, b, s, dy = norm_case(2, 32, 4, 6, 6, BF16)
    norm_check(x, w, None, None, dy, 4, "silu")
    norm_check(x, None, b, None, dy, 4, "silu")


@pytest.mark.parametrize("dtype,mean", [(F16, 100.0), (F32, 3000.0)])
def test_norm_mean_far_from_zero(dtype, mean):
    # One mean for all channels: the spread is what the norm has to find.
    x = (mean + rand(2, 24, 24, 64, seed=1)).to(dtype).permute(0, 3, 1, 2)
    norm_check(x, *norm_case(2, 64, 4, 24, 24, dtype)[1:], 4, None)


# Slabs of 32-bit values that the forward pass keeps in part and reads the rest of
# again; beside them 16-bit ones of the same size, which it does not.
@pytest.mark.parametrize("B,C,G,H,W,dtype", [(4, 320, 32, 61, 67, F32), (2, 640, 32, 59, 71, F32),
                                             (7, 128, 4, 53, 97, F32), (4, 320, 32, 61, 67, BF16)])
@pytest.mark.parametrize("how", ["plain", "far mean", "slice", "one sample for all"])
def test_norm_slabs_read_again(B, C, G, H, W, dtype, how):
    x, w, b, s, dy = norm_case(B, C, G, H, W, dtype, shift=dtype)
    if how == "far mean":
        x = (x.float() + 64).to(dtype)
    if how == "slice":
        wide = torch.zeros(B, H, W, C + 20, device="cuda", dtype=dtype).permute(0, 3, 1, 2)
        wide[:, 8:8 + C] = x
        x = wide[:, 8:8 + C]
    if how == "one sample for all":
        x = x[:1].expand(B, C, H, W)
    norm_check(x, w, b, s, dy, G, "silu")


def test_norm_first_pixel_far_out():
    x, w, b, s, dy = norm_case(1, 64, 4, 32, 32, F32)
    x[:, :, 0, 0] = 4000.0
    norm_check(x, w, b, s, dy, 4, "silu")


def test_norm_constant_group():
    # No spread at all: n is zero, eps carries the division.
    x = torch.full((2, 5, 5, 16), 3.0, device="cuda", dtype=F16).permute(0, 3, 1, 2)
    _, w, b, s, dy = norm_case(2, 16, 2, 5, 5, F16)
    norm_check(x, w, b, None, dy, 2, "silu")


def test_norm_channel_slice_and_broadcast_batch():
    wide, w, b, s, dy = norm_case(3, 64, 4, 7, 9, F16)
    _, w, b, s, _ = norm_case(3, 32, 4, 7, 9, F16, shift=F16)
    norm_check(wide[:, 16:48], w, b, s, dy[:, :32], 4, "silu")
    norm_check(wide[:, 3:35], w, b, s, dy[:, 5:37], 4, "silu")   # not on 16 bytes
    norm_check(wide[:1, :32].expand(3, 32, 7, 9), w, b, s, dy[:, :32], 4, None)
    # A gradient that is one number everywhere, and one in NCHW memory.
    norm_check(wide[:, :32], w, b, s, torch.ones(1, device="cuda", dtype=F16).expand(3, 32, 7, 9), 4, "silu")
    norm_check(wide[:, :32], w, b, s, dy[:, :32].contiguous(), 4, "silu")


def test_norm_rows_around_a_slice_stay():
    big = torch.full((2, 9, 9, 64), 7.0, device="cuda", dtype=F16)
    x = big.permute(0, 3, 1, 2)[:, 8:40]
    x.copy_(rand(2, 32, 9, 9, seed=3))
    nova_group_norm(x, 4, activation="silu")
    assert (big[..., :8] == 7).all() and (big[..., 40:] == 7).all()


def test_norm_nonfinite_stays_in_its_group():
    x, w, b, s, dy = norm_case(2, 32, 4, 6, 6, F16)
    x[0, 9, 2, 2] = float("nan")
    x[1, 31, 0, 0] = INF
    y = nova_group_norm(x, 4, w, b)
    bad = torch.zeros(2, 4, dtype=torch.bool)
    bad[0, 1] = bad[1, 3] = True
    assert torch.equal(torch.isnan(y).reshape(2, 4, -1).all(-1).cpu(), bad)
    assert torch.equal(torch.isnan(y).reshape(2, 4, -1).any(-1).cpu(), bad)


def test_norm_empty():
    w = torch.ones(8, device="cuda", requires_grad=True)
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4)):
        x = torch.zeros(shape, device="cuda", dtype=F16).contiguous(memory_format=torch.channels_last)
        y = nova_group_norm(x, 2, w)
        assert y.shape == shape
        assert (torch.autograd.grad(y.sum(), w)[0] == 0).all()


def test_norm_gradient_by_differences():
    # float32, a direction in every input: (f(+h) - f(-h)) / 2h has an error of about
    # h^2 f''' / 6 + 2^-23 |f| / h, here below 2e-3 of the slope.
    x, w, b, s, dy = norm_case(2, 12, 3, 5, 4, F32, shift=F32, seed=9)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, s)]
    y = nova_group_norm(leaves[0], 3, leaves[1], leaves[2], 1e-5, "silu", leaves[3])
    grads = torch.autograd.grad(y, leaves, dy)
    for i in range(4):
        t = (x, w, b, s)[i]
        d = torch.randn_like(t)
        h = 1e-2
        vals = []
        for sign in (1, -1):
            a = [x, w, b, s]
            a[i] = t + sign * h * d
            vals.append((nova_group_norm(a[0], 3, a[1], a[2], 1e-5, "silu", a[3]).double() * dy).sum())
        slope = ((vals[0] - vals[1]) / (2 * h)).item()
        want = (grads[i].double() * d).sum().item()
        size = (grads[i].double().norm() * d.double().norm()).item()
        assert abs(slope - want) <= 5e-3 * size, i


def test_norm_repeats_and_refuses_second_derivative():
    x, w, b, s, dy = norm_case(4, 320, 32, 33, 31, F16, shift=F16)
    a = norm_check(x, w, b, s, dy, 32, "silu")
    for _ in range(3):
        c = norm_check(x, w, b, s, dy, 32, "silu")
        assert all(torch.equal(a[n], c[n]) for n in a)
    leaf = x.detach().requires_grad_()
    g = torch.autograd.grad(nova_group_norm(leaf, 32, w, b).float().sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_norm_module_layouts():
    norm = torch.nn.GroupNorm(4, 32).cuda()
    m = NovaGroupNorm.from_group_norm(norm, "silu")
    x = rand(2, 32, 9, 5, seed=2)
    want = P.group_norm(x.double(), 4, act="silu", types=(F32, F32, F32))
    for t in (x, x.contiguous(memory_format=torch.channels_last)):
        y = m(t)
        assert y.stride() == t.stride()
        near(y, want["y"], want["y_tol"], "y")


# ---------------------------------------------------------------------------
# Cross attention
# ---------------------------------------------------------------------------

def cross_case(B, Nq, Nk, H, D, dtype, mask=None, seed=0, wide=1.5):
    q = (wide * rand(B, Nq, H, D, seed=seed)).to(dtype)
    k, v = rand(B, Nk, H, D, seed=seed + 1, dtype=dtype), rand(B, Nk, H, D, seed=seed + 2, dtype=dtype)
    do = rand(B, Nq, H, D, seed=seed + 3, dtype=dtype)
    m = None
    if mask:
        g = torch.Generator(device="cuda").manual_seed(seed + 4)
        m = torch.rand(B, Nk, generator=g, device="cuda") < 0.7
        if B > 2:
            m[1] = False
        if mask != "bool":
            bias = 0.5 * rand(B, Nk, seed=seed + 5)
            m = torch.where(m, bias, -INF).to({"f16": F16, "bf16": BF16, "f32": F32}[mask])
    return q, k, v, m, do


def cross_check(q, k, v, m, do, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = nova_cross_attention(*leaves, key_mask=m, scale=scale)
    assert o.dtype == q.dtype and o.shape == q.shape and o.is_contiguous()
    with torch.no_grad():
        assert torch.equal(nova_cross_attention(q, k, v, key_mask=m, scale=scale), o)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)), o=o.detach())
    d = [t.detach().double() for t in (q, k, v, do)]
    md = m if m is None or m.dtype == torch.bool else m.double()
    c = q.shape[-1] ** -0.5 if scale is None else scale
    want = P.cross_attention(*d[:3], md, c, d[3], q.dtype)
    for name, t in got.items():
        near(t, want[name], want[name + "_tol"], name)
    return got


@pytest.mark.parametrize("B,Nq,Nk,H,D", [
    (2, 64, 77, 8, 40), (1, 300, 77, 3, 64), (2, 64, 77, 8, 160), (1, 257, 77, 5, 80),
    (1, 1, 1, 1, 8), (2, 1, 77, 4, 64), (1, 1, 2041, 3, 64), (3, 5, 129, 2, 32), (1, 129, 1, 2, 16),
    (1, 127, 128, 1, 128), (1, 128, 129, 1, 96), (2, 200, 333, 2, 64), (1, 77, 1000, 1, 160),
    (1, 40, 16, 2, 152), (1, 33, 17, 2, 24), (1, 513, 64, 2, 48), (70, 3, 3, 2, 8),
    (1, 1000, 256, 1, 72), (1, 600, 300, 2, 136), (4, 16, 700, 1, 120), (2, 3, 1111, 3, 160), (3, 2, 131, 2, 40), (1, 4, 5000, 2, 128),
    (2, 1, 300, 2, 72), (1, 1, 40000, 1, 64), (1, 2, 9000, 2, 8), (1, 40, 12800, 1, 64), (1, 8, 40000, 1, 48), (2, 8, 517, 3, 56), (1, 7, 300, 2, 104), (2, 9, 300, 2, 64),
    (14, 10, 200, 10, 160), (3, 640, 77, 3, 40), (40, 130, 20, 8, 64),
])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_cross_shapes(B, Nq, Nk, H, D, dtype):
    cross_check(*cross_case(B, Nq, Nk, H, D, dtype))


@pytest.mark.parametrize("mask", ["bool", "f16", "bf16", "f32"])
@pytest.mark.parametrize("Nq,Nk", [(70, 77), (1, 300), (130, 400), (3, 9000)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_cross_masks(mask, Nq, Nk, dtype):
    case = cross_case(3, Nq, Nk, 2, 64, dtype, mask)
    got = cross_check(*case)
    assert (got["o"][1] == 0).all() and all((got[n][1] == 0).all() for n in ("dq", "dk", "dv"))
    gone = ~case[3] if mask == "bool" else case[3] == -INF
    assert (got["dk"][gone] == 0).all() and (got["dv"][gone] == 0).all()


@pytest.mark.parametrize("Nk", [40, 77, 300])
@pytest.mark.parametrize("poison", [float("nan"), INF, -INF])
def test_cross_masked_keys_are_never_multiplied(Nk, poison):
    q, k, v, m, do = cross_case(3, 150, Nk, 2, 64, F16, "bool", seed=5)
    want = cross_check(q, k, v, m, do)
    bias = torch.where(m, 0.0, -INF)
    k[~m], v[~m] = poison, poison
    for mask in (m, bias):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = nova_cross_attention(*leaves, key_mask=mask)
        got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)), o=o.detach())
        for n in got:
            assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_cross_lowest_value_everywhere_is_uniform(dtype):
    q, k, v, _, do = cross_case(2, 20, 50, 2, 32, F16, wide=0.5)
    low = torch.full((2, 50), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    o = nova_cross_attention(q, k, v, key_mask=low)
    if dtype == F16:  # 65504 leaves the scores some digits in 32 bits (steps of 2^-8)
        want = P.cross_attention(q.double(), k.double(), v.double(), low.double(), 32 ** -0.5)["o"]
        assert (o.double() - want).abs().max() <= 2 ** -7 * v.abs().max() + 2 ** -10
    else:
        want = v.double().mean(1, keepdim=True).expand(q.shape)
        assert (o.double() - want).abs().max() <= 2 ** -10 * v.abs().max()
    # Beside keys that take part, the lowest value takes nothing.
    low[:, :30] = 0
    o = nova_cross_attention(q, k, v, key_mask=low)
    assert torch.equal(o, nova_cross_attention(q, k, v, key_mask=low == 0))


def test_cross_one_key_left():
    # One key: p is one, whatever the score, and its gradient nothing.
    for Nk in (1, 77, 300):
        q, k, v, _, do = cross_case(2, 130, Nk, 2, 64, F16)
        m = torch.zeros(2, Nk, dtype=torch.bool, device="cuda")
        m[:, Nk // 2] = True
        got = cross_check(q, k, v, m, do)
        assert torch.equal(got["o"], v[:, Nk // 2: Nk // 2 + 1].expand_as(q))


def test_cross_nonfinite_stays_in_its_head():
    q, k, v, _, do = cross_case(2, 140, 90, 3, 40, F16)
    v[0, 3, 1, 2] = INF
    q[1, 7, 2, 0] = float("nan")
    o = nova_cross_attention(q, k, v)
    ok = torch.ones_like(o, dtype=torch.bool)
    ok[0, :, 1, 2] = False
    ok[1, 7, 2] = False
    assert torch.isfinite(o[ok]).all() and not torch.isfinite(o[~ok]).any()


@pytest.mark.parametrize("Nq,Nk", [(1, 77), (150, 77), (140, 290)])
def test_cross_layouts(Nq, Nk):
    B, H, D = 2, 3, 40
    # Heads before tokens; k and v as halves of one projection; a slice off 16 bytes.
    q = rand(B, H, Nq, D, seed=1, dtype=F16).transpose(1, 2)
    kv = rand(B, Nk, H, 2, D, seed=2, dtype=F16)
    do = rand(B, H, Nq, D, seed=3, dtype=F16).transpose(1, 2)
    m = (rand(Nk, B, seed=4) > -1).transpose(0, 1)
    a = cross_check(q, kv[:, :, :, 0], kv[:, :, :, 1], m, do)
    b = cross_check(q.contiguous(), kv[:, :, :, 0].contiguous(), kv[:, :, :, 1].contiguous(),
                    m.contiguous(), do.contiguous())
    assert all(torch.equal(a[n], b[n]) for n in a)
    odd = rand(B, Nk, H, D + 1, seed=5, dtype=F16)[..., 1:]
    cross_check(q, odd, kv[:, :, :, 1], m, do)
    # Encoder states, a mask and a gradient that all samples share.
    one = rand(1, Nk, H, D, seed=6, dtype=F16).expand(B, Nk, H, D)
    cross_check(q, one, one, m[:1].expand(B, Nk), do[:1].expand(B, Nq, H, D))
    head = rand(B, Nk, 1, D, seed=7, dtype=F16).expand(B, Nk, H, D)
    cross_check(q, head, head, None, torch.ones((), device="cuda", dtype=F16).expand(q.shape))


def test_cross_shared_states_collect_their_gradient():
    q, k, v, _, do = cross_case(3, 40, 50, 2, 32, F16)
    leaf = k[:1].detach().requires_grad_()
    o = nova_cross_attention(q, leaf.expand_as(k), v)
    got = torch.autograd.grad(o, leaf, do)[0]
    parts = cross_check(q, k[:1].expand_as(k).contiguous(), v, None, do)["dk"]
    assert torch.equal(got, parts.sum(0, keepdim=True))


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_cross_scale(scale):
    cross_check(*cross_case(2, 60, 77, 2, 16, F16, wide=0.5), scale=scale)


@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** 6])
def test_cross_small_and_large_gradients(size):
    # Below fp16's normal range: what is off grows by its last step, 2^-25, at most.
    q, k, v, m, do = cross_case(2, 300, 77, 2, 64, F16, "bool")
    do = (do * size).half()
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    got = dict(zip(("dq", "dk", "dv"),
                   torch.autograd.grad(nova_cross_attention(*leaves, key_mask=m), leaves, do)))
    d = [t.double() for t in (q, k, v, do)]
    want = P.cross_attention(*d[:3], m, 0.125, d[3], F16)
    for n in got:
        near(got[n], want[n], want[n + "_tol"] + 2.0 ** -25, n)


def test_cross_gradient_by_differences():
    q, k, v, m, do = cross_case(2, 9, 20, 2, 16, F16, "bool", wide=0.5)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(nova_cross_attention(*leaves, key_mask=m), leaves, do)
    d = [t.double() for t in (q, k, v)]
    for i in range(3):
        step = torch.randn_like(d[i])
        h = 1e-5
        vals = []
        for sign in (1, -1):
            a = list(d)
            a[i] = d[i] + sign * h * step
            vals.append((P.cross_attention(*a, m, 0.25)["o"] * do.double()).sum())
        slope = ((vals[0] - vals[1]) / (2 * h)).item()
        size = (grads[i].double().norm() * step.norm()).item()
        assert abs(slope - (grads[i].double() * step).sum().item()) <= 2 ** -9 * size


def test_cross_empty():
    for B, Nq, Nk in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        q, k, v, _, do = cross_case(B, Nq, Nk, 2, 16, F16)
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = nova_cross_attention(*leaves)
        assert o.shape == q.shape and (o == 0).all()
        for g, t in zip(torch.autograd.grad(o, leaves, do), leaves):
            assert g.shape == t.shape and (g == 0).all()


def test_cross_repeats():
    case = cross_case(3, 700, 333, 4, 64, BF16, "f32")
    a = cross_check(*case)
    for _ in range(3):
        b = cross_check(*case)
        assert all(torch.equal(a[n], b[n]) for n in a)


# ---------------------------------------------------------------------------
# Streams, graphs, the block
# ---------------------------------------------------------------------------

def both_ops(x, s, w, b, k, v, m):
    """Norm with activation, then attention of its pixels to the states."""
    y = nova_group_norm(x, 4, w, b, activation="silu", shift=s)
    q = y.permute(0, 2, 3, 1).flatten(1, 2).unflatten(-1, (2, 32))
    return nova_cross_attention(q, k, v, key_mask=m)


def block_inputs(seed=0, B=2, side=17, Nk=77):
    x, w, b, s, _ = norm_case(B, 64, 4, side, side, F16, shift=F16, seed=seed)
    _, k, v, m, do = cross_case(B, side * side, Nk, 2, 32, F16, "bool", seed=seed + 20)
    return x, s, w, b, k, v, m, do


def test_on_another_stream():
    x, s, w, b, k, v, m, do = block_inputs()
    want = both_ops(x, s, w, b, k, v, m)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [both_ops(x, s, w, b, k, v, m) for _ in range(4)]
    # Meanwhile the same operators on the stream before.
    again = [both_ops(x, s, w, b, k, v, m) for _ in range(4)]
    torch.cuda.synchronize()
    for t in got + again:
        assert torch.equal(t, want)


def test_calls_from_two_threads():
    """Two host threads, a stream each, every result as from one."""
    import threading
    sets = [block_inputs(i, B=2 + i, Nk=(77, 300)[i]) for i in range(2)]
    want = [both_ops(*s[:7]) for s in sets]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(both_ops(*sets[i][:7]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(t, want[i]) for t in got[i])


def test_long_cache_offsets_past_32_bits():
    """Keys whose bytes lie past 2^32 of the cache's start: the last ones decide."""
    B, Nk, H, D = 1, 2 ** 21 + 3, 16, 64
    k = torch.zeros(B, Nk, H, D, device="cuda", dtype=F16)
    v = torch.zeros(B, Nk, H, D, device="cuda", dtype=F16)
    k[:, -1] = 8.0
    v[:, -1] = rand(H, D, seed=1, dtype=F16)
    for Nq in (1, 20):
        q = torch.full((B, Nq, H, D), 8.0, device="cuda", dtype=F16)
        # The last key's score is 8 * 8 * 64 / 8 = 512; e^-512 of the others is nothing.
        o = nova_cross_attention(q, k, v)
        assert torch.equal(o, v[:, -1:].expand_as(o))


@pytest.mark.parametrize("Nk", [77, 300])
def test_captured_step_replays_on_new_values(Nk):
    a, c = block_inputs(0, Nk=Nk), block_inputs(100, Nk=Nk)
    held = [t.clone() for t in a]

    def step(x, s, w, b, k, v, m, do):
        leaves = [t.requires_grad_() for t in (x.detach(), s.detach(), w.detach(), b.detach(), k.detach(), v.detach())]
        o = both_ops(*leaves, m)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    want = [step(*a), step(*c)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of the same step: each its own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*held)
        graphs.append((g, out))
    for inputs, w in ((c, want[1]), (a, want[0])):
        for t, n in zip(held, inputs):
            t.copy_(n)
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for x, y in zip(out, w):
                assert torch.equal(x, y)


def test_run_of_both_against_the_plain_forms():
    x, s, w, b, k, v, m, do = block_inputs(3)
    y = nova_group_norm(x, 4, w, b, activation="silu", shift=s)
    q = y.permute(0, 2, 3, 1).flatten(1, 2).unflatten(-1, (2, 32))
    want = P.group_norm(x.double(), 4, w.double(), b.double(), 1e-5, "silu", s.double(), types=(F16, F32, F16))
    near(y, want["y"], want["y_tol"], "norm")
    # The attention is held to what the norm gave it.
    o = P.cross_attention(q.double(), k.double(), v.double(), m, 32 ** -0.5, dtype=F16)
    near(both_ops(x, s, w, b, k, v, m), o["o"], o["o_tol"], "attention")


@pytest.mark.parametrize("xl", [False, True])
def test_unet_caller_on_the_operators(xl):
    """The UNet callers with their norms and cross attentions on the operators: every
    one of them is called, and the step stays with the 32-bit model as near as the
    16-bit model does (twice its distance: both round the same intermediate results)."""
    import unet_callers as U
    import nova_winograd
    if xl:
        spec = U.UNetSpec(channels=(32, 64, 64), attn_depth=(0, 1, 2), mid_depth=2,
                          context_dim=24, head_dim=16, linear_proj=True, add_embed=True, groups=8,
                          pooled_dim=20, add_time_dim=8)
    else:
        spec = U.UNetSpec(channels=(32, 64), attn_depth=(1, 1), mid_depth=1, context_dim=16,
                          heads=4, groups=8)
    torch.manual_seed(0)
    exact = U.UNet(spec).cuda().eval()
    model = U.UNet(spec).cuda().eval()
    model.load_state_dict(exact.state_dict())
    model = model.half().to(memory_format=torch.channels_last)
    x, t, ctx, extra = U.make_inputs(spec, 2, 16, "cuda", F32, seed=3)
    calls = {"nova_group_norm": 0, "nova_cross_attention": 0}
    saved = {n: getattr(nova_winograd, n) for n in calls}

    def counted(n):
        def f(*a, **k):
            calls[n] += 1
            return saved[n](*a, **k)
        return f

    with torch.no_grad():
        want = exact(x, t, ctx, **extra)
        args = (x.half().contiguous(memory_format=torch.channels_last), t, ctx.half())
        before = model(*args, **extra)
        U.use_nova_ops(model)
        try:
            for n in calls:
                setattr(nova_winograd, n, counted(n))
            got = model(*args, **extra)
        finally:
            for n in calls:
                setattr(nova_winograd, n, saved[n])
        U.use_nova_ops(model, False)
        assert torch.equal(model(*args, **extra), before)
    norms = sum(isinstance(m, torch.nn.GroupNorm) for m in model.modules())
    layers = sum(isinstance(m, U.TransformerLayer) for m in model.modules())
    assert calls == {"nova_group_norm": norms, "nova_cross_attention": layers}
    assert torch.isfinite(got).all()
    assert (got.float() - want).norm() <= 2 * (before.float() - want).norm()


def test_unet_caller_gradients_on_the_operators():
    """A training step's gradients through the operators against the 32-bit model's."""
    import unet_callers as U
    spec = U.UNetSpec(channels=(32, 64), attn_depth=(1, 1), mid_depth=1, context_dim=16, heads=4,
                      groups=8)
    torch.manual_seed(1)
    exact = U.UNet(spec).cuda()
    model = U.UNet(spec).cuda()
    model.load_state_dict(exact.state_dict())
    model = model.half().to(memory_format=torch.channels_last)
    x, t, ctx, _ = U.make_inputs(spec, 2, 16, "cuda", F32, seed=4)
    args = (x.half().contiguous(memory_format=torch.channels_last), t, ctx.half())

    def grads(m, *a):
        m.zero_grad()
        m(*a).float().square().mean().backward()
        return torch.cat([p.grad.float().flatten() for p in m.parameters()])

    want = grads(exact, x, t, ctx)
    before = grads(model, *args)
    U.use_nova_ops(model)
    got = grads(model, *args)
    assert torch.isfinite(got).all()
    assert (got - want).norm() <= 2 * (before - want).norm()


def test_cross_status_is_clear():
    from nova_winograd import ops
    assert ops.get_lib().nova_cross_attention_status() == 0

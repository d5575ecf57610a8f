"""Calls of the UNet operators that their documentation allows and that go wrong
easily: other defaults, saved-tensor hooks, masks and tensors at their limits.
Bounds are unet_ops_plain's."""

import pytest
import torch
from torch.autograd import forward_ad

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


# Biases that every key of a sample has, and beside which a score is less than half a
# step of 32 bits: the softmax in 32 bits is uniform.
SHARED = [(BF16, torch.finfo(BF16).min), (F32, torch.finfo(F32).min), (F32, -1e9), (F32, 3e38)]


@pytest.mark.parametrize("mtype,low", SHARED)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Nq,Nk,H,D", [
    (2, 20, 50, 2, 32), (3, 300, 77, 8, 40),    # one tile of keys; many heads for a block
    (1, 150, 300, 2, 64), (2, 70, 200, 2, 160),  # keys split, the last part shorter
    (9, 260, 333, 20, 64),                       # several tiles, not split
    (2, 1, 300, 3, 64), (1, 3, 9000, 2, 64),     # few queries: a cluster, blocks joined after
])
def test_cross_one_bias_for_all_keys(mtype, low, dtype, B, Nq, Nk, H, D):
    q, k, v, _, do = cross_case(B, Nq, Nk, H, D, dtype, wide=0.5)
    mask = torch.full((B, Nk), low, device="cuda", dtype=mtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = nova_cross_attention(*leaves, key_mask=mask)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)), o=o.detach())
    # The uniform row in 64 bits: scores of zero.  dq knows q by them alone, dk knows k.
    d = [t.double() for t in (q, k, v, do)]
    flat = P.cross_attention(torch.zeros_like(d[0]), *d[1:3], None, D ** -0.5, d[3], dtype)
    keys = P.cross_attention(d[0], torch.zeros_like(d[1]), d[2], None, D ** -0.5, d[3], dtype)
    for name, want in (("o", flat), ("dq", flat), ("dv", flat), ("dk", keys)):
        near(got[name], want[name], want[name + "_tol"], name)


@pytest.mark.parametrize("low", [-1e4, -65504.0, -1e6])
@pytest.mark.parametrize("Nq,Nk", [(64, 77), (64, 300), (4, 300)])
def test_cross_probabilities_sum_to_one_beside_a_large_bias(low, Nq, Nk):
    """do of ones: what dv comes to over the keys is the sum of all probabilities, Nq.
    Each is rounded once, and dv once: 2 half steps of FP16, and 2^-16 for the sums."""
    q, k, v, _, _ = cross_case(2, Nq, Nk, 2, 64, F16)
    mask = torch.full((2, Nk), low, device="cuda", dtype=F32)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = nova_cross_attention(*leaves, key_mask=mask)
    dv = torch.autograd.grad(o, leaves[2], torch.ones_like(o))[0]
    # Probabilities of less than FP16's normal 2^-14 / 2^10 keep a step of 2^-34.
    bound = Nq * (2 * P.half_step(F16) + 2.0 ** -16) + Nq * Nk * 2.0 ** -35
    # dv below 2^-14 has steps of 2^-24.
    bound += Nk * 2.0 ** -25
    assert ((dv.double().sum(1) - Nq).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Nq,Nk", [(70, 77), (150, 300), (1, 300), (3, 9000)])
def test_cross_far_biases_keep_their_order(dtype, Nq, Nk):
    """Finite biases of any size count as the sums with them do in 32 bits: the larger
    one takes all, the smaller nothing."""
    q, k, v, _, do = cross_case(2, Nq, Nk, 2, 64, dtype, wide=0.5)
    g = torch.Generator(device="cuda").manual_seed(7)
    take = torch.rand(2, Nk, generator=g, device="cuda") < 0.5
    for high, low in ((-3.3e38, torch.finfo(F32).min), (-1e38, -2.5e38), (3.4e38, 2.4e38),
                      (-8e37, -9e37)):
        mask = torch.where(take, high, low).float()
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = nova_cross_attention(*leaves, key_mask=mask)
        got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)), o=o.detach())
        d = [t.double() for t in (q, k, v, do)]
        flat = P.cross_attention(torch.zeros_like(d[0]), *d[1:3], take, 0.125, d[3], dtype)
        keys = P.cross_attention(d[0], torch.zeros_like(d[1]), d[2], take, 0.125, d[3], dtype)
        for name, want in (("o", flat), ("dq", flat), ("dv", flat), ("dk", keys)):
            near(got[name], want[name], want[name + "_tol"], name)


@pytest.mark.parametrize("Nq,Nk", [(1, 300), (70, 77), (130, 300)])
@pytest.mark.parametrize("offset", [1, 4])
def test_cross_contiguous_tensors_off_16_bytes(Nq, Nk, offset):
    q, k, v, m, do = cross_case(2, Nq, Nk, 2, 40, F16, "bool")
    want = cross_check(q, k, v, m, do)

    def moved(t):
        flat = torch.cat([t.new_zeros(offset), t.flatten()])
        return flat[offset:].view(t.shape)
    got = cross_check(*map(moved, (q, k, v)), m, moved(do))
    assert all(torch.equal(got[n], want[n]) for n in want)
    # A gradient that comes back through a concatenation, at an odd element.
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = nova_cross_attention(*leaves, key_mask=m)
    joined = torch.cat([torch.zeros(offset, device="cuda", dtype=F16), o.flatten()])
    grads = torch.autograd.grad(joined, leaves, torch.cat([joined.new_zeros(offset), do.flatten()]))
    assert all(torch.equal(g, want[n]) for g, n in zip(grads, ("dq", "dk", "dv")))
    # One sample, one token, whose strides belong to the tensor that they are a part of.
    wide = torch.zeros(3 * (Nk * 80 + 4), device="cuda", dtype=F16)
    one = wide.as_strided((3, Nk, 2, 40), (Nk * 80 + 4, 80, 40, 1))[:1]
    one.copy_(k[:1])
    a = cross_check(q[:1], one, v[:1], m[:1], do[:1])
    b = cross_check(q[:1].contiguous(), k[:1].contiguous(), v[:1], m[:1], do[:1])
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_norm_of_the_most_pixels():
    """2^31 - 4096 pixels of one channel, the last of them too; piece by piece in 64 bits."""
    H, W = 524287, 4096
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(1, 1, H, W, device="cuda", dtype=F16)
    dy = torch.empty(1, 1, H, W, device="cuda", dtype=F16)
    pieces = [slice(i, min(i + 16384, H)) for i in range(0, H, 16384)]
    for p in pieces:
        for t, at in ((x, 0.5), (dy, 0.25)):
            t[:, :, p] = torch.randn(1, 1, p.stop - p.start, W, generator=g, device="cuda") + at
    w = torch.tensor([1.25], device="cuda", requires_grad=True)
    b = torch.tensor([-0.5], device="cuda", requires_grad=True)
    x.requires_grad_()
    y = nova_group_norm(x, 1, w, b, 1e-5, "silu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x, y = x.detach(), y.detach()
    n = H * W
    mean = sum(x[:, :, p].double().sum() for p in pieces) / n
    r = (sum((x[:, :, p].double() - mean).square().sum() for p in pieces) / n + 1e-5) ** -0.5

    def step(p):
        m = (x[:, :, p].double() - mean) * r
        z = m * 1.25 - 0.5
        s = torch.sigmoid(z)
        dz = dy[:, :, p].double() * s * (1 + z * (1 - s))
        return m, z, s, dz
    A = D = size = sized = 0.0
    for p in pieces:
        m, z, s, dz = step(p)
        A, D = A + dz.sum(), D + (dz * m).sum()
        size, sized = size + dz.abs().sum(), sized + (dz * m).abs().sum()
    near(db[0], A, P.half_step(F32) * A.abs() + 2 * P.SUM * P.F32 * size, "db")
    near(dw[0], D, P.half_step(F32) * D.abs() + 2 * P.SUM * P.F32 * sized, "dw")
    for p in pieces:
        m, z, s, dz = step(p)
        m_off = P.OPS * P.F32 * (m.abs() + mean.abs() * r)
        z_off = 1.25 * m_off + P.OPS * P.F32 * (z.abs() + 0.5)
        near(y[:, :, p], z * s, P.rounded(F16, z * s) + 1.1 * z_off + P.OPS * P.F32 * (z * s).abs(), "y")
        want = r * (1.25 * dz - 1.25 * A / n - m * 1.25 * D / n)
        off = r * (1.25 * dy[:, :, p].double().abs() * (0.5 * z_off + P.OPS * P.F32)
                   + 2 * P.SUM * P.F32 * 1.25 * (size + m.abs() * sized) / n
                   + m_off * (1.25 * D / n).abs()
                   + P.OPS * P.F32 * 1.25 * (dz.abs() + (A / n).abs() + (m * D / n).abs()))
        near(dx[:, :, p], want, P.rounded(F16, want) + off + 1e-12, "dx")


def test_tangents_are_refused():
    x, w, b, s, _ = norm_case(2, 32, 4, 6, 6, F16, shift=F16)
    q, k, v, m, _ = cross_case(2, 9, 20, 2, 16, F16, "f32")
    want = nova_group_norm(x, 4, w, b, shift=s), nova_cross_attention(q, k, v, key_mask=m)
    with forward_ad.dual_level(), torch.no_grad():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for i in range(4):
            a = [x, w, b, s]
            a[i] = dual(a[i])
            with pytest.raises(NotImplementedError):
                nova_group_norm(a[0], 4, a[1], a[2], shift=a[3])
        for i in range(4):
            a = [q, k, v, m]
            a[i] = dual(a[i])
            with pytest.raises(NotImplementedError):
                nova_cross_attention(*a[:3], key_mask=a[3])
        got = nova_group_norm(x, 4, w, b, shift=s), nova_cross_attention(q, k, v, key_mask=m)
    assert all(torch.equal(g, t) for g, t in zip(got, want))


def test_norm_of_the_most_channels_in_a_group():
    norm_check(*norm_case(2, 2 * 8192, 2, 3, 3, F16, shift=F16), 2, "silu")
    norm_check(*norm_case(1, 8192, 1, 5, 1, F32), 1, None)


@pytest.mark.parametrize("B,C,G,H,W", [(2, 12000, 2, 3, 3), (2, 16384, 2, 30, 30), (1, 5000, 1, 4, 4),
                                       (4, 1024, 1, 40, 41), (2, 2048, 1, 64, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_norm_of_many_channels_in_a_group(B, C, G, H, W, dtype):
    norm_check(*norm_case(B, C, G, H, W, dtype, shift=dtype), G, "silu")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("mask", ["bool", "f32"])
@pytest.mark.parametrize("Nk", [77, 300])
@pytest.mark.parametrize("poison", [float("nan"), INF])
def test_cross_sample_without_keys_passes_nothing_on(dtype, mask, Nk, poison):
    """A padded sample: its queries and what comes back for them may hold anything."""
    q, k, v, m, do = cross_case(3, 150, Nk, 2, 64, dtype, mask)
    want = cross_check(q, k, v, m, do)
    for bad in ((q,), (do,), (q, k, v, do)):
        held = [t[1].clone() for t in bad]
        for t in bad:
            t[1] = poison
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = nova_cross_attention(*leaves, key_mask=m)
        got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)), o=o.detach())
        assert all(torch.equal(got[n], want[n]) and (got[n][1] == 0).all() for n in want)
        for t, h in zip(bad, held):
            t[1] = h


@pytest.mark.parametrize("B,Nq,Nk,H,D", [(300, 20, 50, 2, 32), (49, 20, 288, 3, 160), (200, 3, 300, 2, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_cross_one_bias_for_all_keys_of_each_sample(dtype, B, Nq, Nk, H, D):
    """Blocks that go from one sample to the next, whose biases differ."""
    q, k, v, _, do = cross_case(B, Nq, Nk, H, D, dtype, wide=0.5)
    mask = (-1e9 * (1 + torch.arange(B, device="cuda") % 5)).float()[:, None].expand(B, Nk)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = nova_cross_attention(*leaves, key_mask=mask)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)), o=o.detach())
    d = [t.double() for t in (q, k, v, do)]
    flat = P.cross_attention(torch.zeros_like(d[0]), *d[1:3], None, D ** -0.5, d[3], dtype)
    keys = P.cross_attention(d[0], torch.zeros_like(d[1]), d[2], None, D ** -0.5, d[3], dtype)
    for name, want in (("o", flat), ("dq", flat), ("dv", flat), ("dk", keys)):
        near(got[name], want[name], want[name + "_tol"], name)


def test_unet_caller_in_64_bits_keeps_torchs_layers():
    """What the operators do not take stays with torch's layers, switched on or not."""
    import unet_callers as U
    spec = U.UNetSpec(channels=(32, 64), attn_depth=(1, 1), mid_depth=1, context_dim=16, heads=4,
                      groups=8)
    torch.manual_seed(0)
    model = U.UNet(spec).cuda().double().to(memory_format=torch.channels_last).eval()
    norm, x = model.norm_out, rand(2, 32, 9, 9, seed=1).double()
    x = x.contiguous(memory_format=torch.channels_last)
    U.use_nova_ops(model)
    assert torch.equal(U.norm_act(norm, x, True, "silu"), U.norm_act(norm, x, False, "silu"))
    layer = model.mid_attn
    ctx = rand(2, 5, 16, seed=2).double()
    h = rand(2, 64, 6, 6, seed=3).double().contiguous(memory_format=torch.channels_last)
    on = layer(h, ctx)
    U.use_nova_ops(model, False)
    assert torch.equal(layer(h, ctx), on)

"""What the UNet operators' kernels write lies in the buffers that the C entry points
were given: every output and the workspace between guards, results as from the public
functions."""

import ctypes

import pytest
import torch

import unet_ops_plain as P
from nova_winograd import nova_cross_attention, nova_group_norm, ops, unet_ops
from test_gpu_unet_ops import cross_case, near, norm_case

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
GUARD, FILL = 8192, 0xA5


class Guarded:
    """Buffers between guards, in one allocation each."""

    def __init__(self):
        self.all = []

    def bytes(self, n):
        whole = torch.full((n + 2 * GUARD,), FILL, dtype=torch.uint8, device="cuda")
        self.all.append((whole, n))
        return whole[GUARD:GUARD + n]

    def tensor(self, shape, dtype):
        n = torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()
        return self.bytes(n).view(dtype).view(shape)

    def intact(self):
        for whole, n in self.all:
            assert (whole[:GUARD] == FILL).all() and (whole[GUARD + n:] == FILL).all()


def run(name, *args):
    ops.check(getattr(ops.get_lib(), name)(*args, torch.cuda.current_stream().cuda_stream), name)


@pytest.mark.parametrize("B,C,G,H,W", [
    (1, 1280, 32, 8, 8), (3, 190, 10, 37, 29), (2, 8, 1, 1, 1), (2, 3, 1, 5, 7), (5, 64, 4, 1, 33),
    (1, 4104, 8, 3, 3), (1, 2056, 8, 61, 67), (8, 320, 32, 64, 65), (2, 333, 3, 101, 97),
    (4, 320, 32, 61, 67), (17, 40, 4, 3, 3), (1, 1, 1, 1000, 1001),
])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_norm_writes_within_its_buffers(B, C, G, H, W, dtype):
    x, w, b, s, dy = norm_case(B, C, G, H, W, dtype, shift=dtype, wtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, s)]
    want_y = nova_group_norm(leaves[0], G, leaves[1], leaves[2], 1e-5, "silu", leaves[3])
    want = torch.autograd.grad(want_y, leaves, dy)
    lib, code, V = ops.get_lib(), unet_ops.DTYPES[dtype], 4 if dtype == F32 else 8
    strides = unet_ops._pixel_strides(x)
    size = [B, H * W, C, G]
    aligned = int(C % V == 0)
    for stats_wanted in (True, False):
        g = Guarded()
        y = g.tensor((B, H, W, C), dtype)
        stats = g.tensor((2, B, G), F32)
        n = lib.nova_group_norm_workspace_bytes(*size, code, aligned, 0)
        ws = g.bytes(n)
        run("nova_group_norm_v2", x.data_ptr(), w.data_ptr(), b.data_ptr(), s.data_ptr(),
            y.data_ptr(), stats.data_ptr() if stats_wanted else None, ws.data_ptr() if n else None, n,
            *size, *strides, code, code, code, 1, 1e-5)
        g.intact()
        assert torch.equal(y.permute(0, 3, 1, 2), want_y.detach())
        if stats_wanted:
            kept = stats.clone()
    g = Guarded()
    dx = g.tensor((B, H, W, C), dtype)
    dw, db, ds = g.tensor((C,), dtype), g.tensor((C,), dtype), g.tensor((B, C), dtype)
    n = lib.nova_group_norm_workspace_bytes(*size, code, aligned, 1)
    ws = g.bytes(n)
    run("nova_group_norm_grad_v2", x.data_ptr(), dy.data_ptr(), w.data_ptr(), b.data_ptr(),
        s.data_ptr(), kept.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ds.data_ptr(),
        ws.data_ptr(), n, *size, *strides, *unet_ops._pixel_strides(dy), code, code, code, 1)
    g.intact()
    for got, t in zip((dx.permute(0, 3, 1, 2), dw, db, ds), want):
        assert torch.equal(got, t)


@pytest.mark.parametrize("B,Nq,Nk,H,D", [
    (2, 64, 77, 8, 40), (1, 1, 1, 1, 8), (1, 129, 1, 2, 16), (2, 200, 333, 2, 64),
    (1, 77, 1000, 1, 160), (3, 5, 129, 2, 32), (2, 3, 1111, 3, 160), (1, 2, 9000, 2, 8),
    (1, 1000, 256, 1, 72), (40, 130, 20, 8, 64), (14, 10, 200, 10, 152), (1, 513, 64, 2, 48),
])
@pytest.mark.parametrize("mask", [None, "bool", "f16"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_cross_writes_within_its_buffers(B, Nq, Nk, H, D, mask, dtype):
    q, k, v, m, do = cross_case(B, Nq, Nk, H, D, dtype, mask)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    want_o = nova_cross_attention(*leaves, key_mask=m)
    want = torch.autograd.grad(want_o, leaves, do)
    lib, code, size = ops.get_lib(), unet_ops.DTYPES[dtype], [B, Nq, Nk, H, D]
    at = m.data_ptr() if mask else None
    kind = unet_ops._mask_type(m)
    n = lib.nova_cross_attention_workspace_bytes(*size, 0)
    for train in (True, False):
        g = Guarded()
        o, low, lse = g.tensor(q.shape, dtype), g.tensor(q.shape, dtype), g.tensor((B, H, Nq), F32)
        ws = g.bytes(n)
        run("nova_cross_attention_v2", q.data_ptr(), k.data_ptr(), v.data_ptr(), at, o.data_ptr(),
            *((low.data_ptr(), lse.data_ptr()) if train else (None, None)),
            ws.data_ptr() if n else None, n, *size, unet_ops._strides(q, k, v, m), code, kind,
            ctypes.c_float(D ** -0.5))
        g.intact()
        assert torch.equal(o, want_o.detach())
        if train:
            kept = o.clone(), low.clone(), lse.clone()
    g = Guarded()
    dq, dk, dv = g.tensor(q.shape, dtype), g.tensor(k.shape, dtype), g.tensor(k.shape, dtype)
    n = lib.nova_cross_attention_workspace_bytes(*size, 1)
    ws = g.bytes(n)
    run("nova_cross_attention_grad_v2", q.data_ptr(), k.data_ptr(), v.data_ptr(), at,
        kept[0].data_ptr(), kept[1].data_ptr(), do.data_ptr(), kept[2].data_ptr(), dq.data_ptr(),
        dk.data_ptr(), dv.data_ptr(), ws.data_ptr() if n else None, n, *size,
        unet_ops._strides(q, k, v, m, do), code, kind, ctypes.c_float(D ** -0.5))
    g.intact()
    for got, t in zip((dq, dk, dv), want):
        assert torch.equal(got, t)


def test_norm_offsets_past_32_bits():
    """4.4 billion elements: the first and the last group, each against its plain form."""
    C, G, H, W, c = 520, 130, 2048, 4096, 4
    g = torch.Generator(device="cuda").manual_seed(5)
    x, dy = (torch.empty(1, H, W, C, device="cuda", dtype=F16).normal_(generator=g).permute(0, 3, 1, 2)
             for _ in range(2))
    w, b = (torch.randn(C, generator=g, device="cuda") for _ in range(2))
    s = torch.randn(1, C, generator=g, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, b, s)]
    y = nova_group_norm(*leaves[:1], G, w, b, 1e-5, "silu", s)
    dx, dw, db, ds = torch.autograd.grad(y, leaves, dy)
    for part in (slice(0, c), slice(C - c, C)):
        d = [t.detach().double() for t in (x[:, part], w[part], b[part], s[:, part], dy[:, part])]
        want = P.group_norm(d[0], 1, d[1], d[2], 1e-5, "silu", d[3], d[4], (F16, F32, F32))
        for name, t in (("y", y.detach()[:, part]), ("dx", dx[:, part]), ("dw", dw[part]),
                        ("db", db[part]), ("ds", ds[:, part])):
            near(t, want[name], want[name + "_tol"], name)


def test_cross_offsets_past_32_bits():
    """4.8 billion elements of q; the last queries are those that have a gradient."""
    Nq, Nk, H, D, n = 2 ** 22 + 128, 9, 16, 72, 256
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.empty(1, Nq, H, D, device="cuda", dtype=BF16).normal_(generator=g)
    k, v = (torch.empty(1, Nk, H, D, device="cuda", dtype=BF16).normal_(generator=g) for _ in range(2))
    do = torch.zeros_like(q)
    do[:, -n:] = torch.randn(1, n, H, D, generator=g, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = nova_cross_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    last = [t.detach()[:, -n:] for t in (q, do)]
    part = [t.detach().clone().requires_grad_() for t in (last[0], k, v)]
    alone = nova_cross_attention(*part)
    assert torch.equal(o.detach()[:, -n:], alone.detach())
    assert torch.equal(dq[:, -n:], torch.autograd.grad(alone, part[0], last[1])[0])
    assert not dq[:, :-n].any()
    want = P.cross_attention(*(t.detach().double() for t in part), None, D ** -0.5, last[1].double(), BF16)
    near(dk, want["dk"], want["dk_tol"], "dk")
    near(dv, want["dv"], want["dv_tol"], "dv")

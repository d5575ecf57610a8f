"""Measured cases of the UNet operators around the 3x3 convolutions: group
normalisation with its activation on channels-last activations, and cross
attention to an encoder's states.

``run`` is the plain form (elementary torch operations in 32 bits) where ``own``
is false, and the framework's operators where it is true.  ``exact`` is the
definition in 64 bits, with the gradients written out by hand.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _norm(name, B, C, G, H, W, dtype, act, shift, train):
    return {"name": name, "op": "norm", "B": B, "C": C, "G": G, "H": H, "W": W, "dtype": dtype,
            "act": act, "shift": shift, "train": train}


def _cross(name, B, Nq, Nk, H, D, dtype, mask, train):
    return {"name": name, "op": "cross", "B": B, "Nq": Nq, "Nk": Nk, "H": H, "D": D,
            "dtype": dtype, "mask": mask, "train": train}


def listed():
    return [
        # Second norm of a residual block in the SD 1.5 middle, one image: launch latency.
        _norm("norm-mid-1", 1, 1280, 32, 8, 8, "fp16", "silu", True, False),
        # The same norm at the SD 1.5 top level, eight images.
        _norm("norm-top-8", 8, 320, 32, 64, 64, "fp16", "silu", True, False),
        # First norm of the SDXL up path's top level (640 + 320 channels): larger than L2.
        _norm("norm-xl-up-8", 8, 960, 32, 128, 128, "fp16", "silu", False, False),
        # A norm without activation at sizes no vector width divides.
        _norm("norm-odd", 3, 190, 10, 37, 29, "bf16", "none", False, False),
        # Training: second norm of an SD 1.5 residual block at 32 x 32, with the
        # gradient of the time embedding added before it.
        _norm("norm-train-32", 8, 640, 32, 32, 32, "fp16", "silu", True, True),
        # Training in 32 bits on an odd image.
        _norm("norm-train-fp32", 4, 320, 32, 61, 67, "fp32", "silu", False, True),
        # Cross attention to 77 text tokens at the top level of SD 1.5, eight images.
        _cross("cross-top-8", 8, 4096, 77, 8, 40, "fp16", "none", False),
        # The same in SDXL's 640-channel level.
        _cross("cross-xl-8", 8, 4096, 77, 10, 64, "fp16", "none", False),
        # One image in the SD 1.5 middle: launch latency, 160-wide heads.
        _cross("cross-mid-1", 1, 64, 77, 8, 160, "fp16", "none", False),
        # One new token per sequence against long padded encoder states.
        _cross("cross-token", 4, 1, 2041, 20, 64, "bf16", "bool", False),
        # Training at the 640-channel level of SD 1.5, prompts of different lengths.
        _cross("cross-train-32", 8, 1024, 77, 8, 80, "fp16", "bool", True),
        # Training against longer states, ragged on both sides, an additive mask
        # that leaves one sample without keys.
        _cross("cross-train-long", 3, 1021, 333, 10, 64, "bf16", "bias", True),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        while True:
            G = rng.choice([1, 4, 10, 16, 32, 32])
            C = G * _logint(rng, 1, 80)
            B, H, W = _logint(rng, 1, 16), _logint(rng, 1, 128), _logint(rng, 1, 128)
            shift, train = rng.random() < 0.5, rng.random() < 0.5
            # With one channel per group a shift cancels: its gradient is zero and
            # whatever comes back is rounding.
            if (B * C * H * W <= 40_000_000 and (C // G) * H * W >= 8
                    and not (C == G and shift and train)):
                break
        return _norm("", B, C, G, H, W, rng.choice(["fp16", "fp16", "bf16", "fp32"]),
                     rng.choice(["silu", "silu", "none"]), shift, train)
    while True:
        B, H, D = _logint(rng, 1, 16), rng.randint(1, 20), 8 * rng.randint(1, 20)
        Nq, Nk = _logint(rng, 1, 4096), _logint(rng, 1, 2048)
        if B * H * Nq * Nk * D <= 800_000_000 and B * H * (Nq + Nk) * D <= 20_000_000:
            break
    return _cross("", B, Nq, Nk, H, D, rng.choice(["fp16", "fp16", "bf16"]),
                  rng.choice(["none", "bool", "bias"]), rng.random() < 0.5)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["B"] * case["C"] * case["H"] * case["W"]
        bc = case["B"] * case["C"]
        nbytes = 2 * n * e + 8 * case["C"] + (bc * e if case["shift"] else 0)
        flops = 10 * n
        if case["train"]:
            nbytes += 2 * n * e + 8 * case["C"] + (bc * e if case["shift"] else 0)
            flops += 20 * n
        return {"bytes": nbytes, "flops": flops}
    q = case["B"] * case["Nq"] * case["H"] * case["D"]
    k = case["B"] * case["Nk"] * case["H"] * case["D"]
    mm = 2 * case["B"] * case["H"] * case["Nq"] * case["Nk"] * case["D"]
    mask = {"none": 0, "bool": 1, "bias": 4}[case["mask"]] * case["B"] * case["Nk"]
    if case["train"]:
        return {"bytes": e * (4 * q + 4 * k) + mask, "flops": 7 * mm}
    return {"bytes": e * (2 * q + 2 * k) + mask, "flops": 2 * mm}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = dict(case)
    leaf = case["train"]
    if case["op"] == "norm":
        B, C, H, W = case["B"], case["C"], case["H"], case["W"]
        # Conv outputs: unit spread, another mean per channel.  Channels-last memory.
        x = (_rand(g, B, H, W, C) + 0.5 * _rand(g, C)).to(dt).permute(0, 3, 1, 2)
        w, b = 1 + 0.2 * _rand(g, C), 0.2 * _rand(g, C)
        st["x"], st["w"], st["b"] = x, w, b
        st["s"] = (0.5 * _rand(g, B, C)).to(dt) if case["shift"] else None
        if leaf:
            st["dy"] = _rand(g, B, H, W, C).to(dt).permute(0, 3, 1, 2)
        names = ["x", "w", "b"] + (["s"] if case["shift"] else [])
    else:
        B, Nq, Nk, H, D = case["B"], case["Nq"], case["Nk"], case["H"], case["D"]
        # Projections of normalised states: [B, N, H, D], the linear layer's output viewed.
        st["q"] = (1.5 * _rand(g, B, Nq, H, D)).to(dt)
        st["k"] = _rand(g, B, Nk, H, D).to(dt)
        st["v"] = _rand(g, B, Nk, H, D).to(dt)
        st["mask"] = None
        if case["mask"] != "none":
            lens = torch.randint(1, Nk + 1, (B,), generator=g, device="cuda")
            if case["mask"] == "bias" and B > 1:
                lens[B // 2] = 0
            keep = torch.arange(Nk, device="cuda")[None, :] < lens[:, None]
            if case["mask"] == "bool":
                st["mask"] = keep
            else:
                st["mask"] = torch.where(keep, 0.5 * _rand(g, B, Nk), float("-inf"))
        if leaf:
            st["dy"] = _rand(g, B, Nq, H, D).to(dt)
        names = ["q", "k", "v"]
    st["leaves"] = []
    if leaf:
        st["leaves"] = [st[n].requires_grad_() for n in names]
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _plain_norm(st):
    B, C, H, W, G = st["B"], st["C"], st["H"], st["W"], st["G"]
    u = st["x"].float()
    if st["s"] is not None:
        u = u + st["s"].float()[:, :, None, None]
    u = u.reshape(B, G, C // G, H, W)
    d = u - u.mean(dim=(2, 3, 4), keepdim=True)
    var = (d * d).mean(dim=(2, 3, 4), keepdim=True)
    n = (d / torch.sqrt(var + 1e-5)).reshape(B, C, H, W)
    z = n * st["w"][:, None, None] + st["b"][:, None, None]
    if st["act"] == "silu":
        z = z / (1 + torch.exp(-z))
    return z.to(st["x"].dtype)


def _plain_cross(st):
    q, k, v = (st[n].float().transpose(1, 2) for n in ("q", "k", "v"))
    s = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(st["D"]))
    m = st["mask"]
    if m is not None:
        if m.dtype == torch.bool:
            m = torch.where(m, 0.0, float("-inf"))
        s = s + m[:, None, None, :]
    top = s.amax(dim=-1, keepdim=True).detach()
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return (p @ v).transpose(1, 2).contiguous().to(st["q"].dtype)


def _entry_points():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "nova-wino-amd_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from nova_winograd import nova_cross_attention, nova_group_norm
    return nova_group_norm, nova_cross_attention


def _forward(st):
    if not own:
        return _plain_norm(st) if st["op"] == "norm" else _plain_cross(st)
    group_norm, cross_attention = _entry_points()
    if st["op"] == "norm":
        act = "silu" if st["act"] == "silu" else None
        return group_norm(st["x"], st["G"], st["w"], st["b"], eps=1e-5, activation=act,
                          shift=st["s"])
    return cross_attention(st["q"], st["k"], st["v"], key_mask=st["mask"])


def run(state):
    if not state["train"]:
        with torch.no_grad():
            return _forward(state)
    y = _forward(state)
    return (y.detach(),) + torch.autograd.grad(y, state["leaves"], state["dy"])


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_norm(st):
    """One sample at a time; a pixel-major [pixels, groups, channels] view."""
    B, C, H, W, G = st["B"], st["C"], st["H"], st["W"], st["G"]
    w, b = st["w"].detach().double().view(G, -1), st["b"].detach().double().view(G, -1)
    ys, dxs, dss = [], [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for i in range(B):
        u = st["x"].detach()[i].permute(1, 2, 0).reshape(H * W, G, C // G).double()
        if st["s"] is not None:
            u = u + st["s"].detach()[i].double().view(G, C // G)
        var, mean = torch.var_mean(u, dim=(0, 2), unbiased=False, keepdim=True)
        r = torch.rsqrt(var + 1e-5)
        n = (u - mean) * r
        z = torch.addcmul(b, n, w)
        sg = torch.sigmoid(z) if st["act"] == "silu" else torch.ones_like(z)
        ys.append((z * sg if st["act"] == "silu" else z).view(H, W, C).permute(2, 0, 1))
        if not st["train"]:
            continue
        dz = st["dy"][i].permute(1, 2, 0).reshape(H * W, G, C // G).double()
        if st["act"] == "silu":
            dz = dz * sg * (1 + z * (1 - sg))
        dw += (dz * n).sum(0)
        db += dz.sum(0)
        e = dz * w
        dx = r * (e - e.mean(dim=(0, 2), keepdim=True)
                  - n * (e * n).mean(dim=(0, 2), keepdim=True))
        dxs.append(dx.view(H, W, C).permute(2, 0, 1))
        dss.append(dx.sum(0).view(C))
    y = torch.stack(ys)
    if not st["train"]:
        return y
    out = (y, torch.stack(dxs), dw.view(C), db.view(C))
    return out + ((torch.stack(dss),) if st["s"] is not None else ())


def _exact_cross(st):
    """One sample at a time, over the keys that its mask leaves."""
    B, Nq, H, D = st["B"], st["Nq"], st["H"], st["D"]
    c = 1.0 / math.sqrt(D)
    full = [torch.zeros(st[n].shape, dtype=torch.float64, device="cuda")
            for n in ("q", "q", "k", "v")]
    o, dq, dk, dv = full
    for i in range(B):
        keep = torch.ones(st["Nk"], dtype=torch.bool, device="cuda")
        add = torch.zeros(st["Nk"], dtype=torch.float64, device="cuda")
        if st["mask"] is not None:
            m = st["mask"][i]
            keep = m if m.dtype == torch.bool else m > float("-inf")
            add = add if m.dtype == torch.bool else m.double()
        idx = keep.nonzero()[:, 0]
        if idx.numel() == 0:
            continue
        q = st["q"].detach()[i].double()
        k, v = st["k"].detach()[i, idx].double(), st["v"].detach()[i, idx].double()
        p = torch.softmax(torch.einsum("qhd,khd->hqk", q, k) * c + add[idx], dim=-1)
        o[i] = torch.einsum("hqk,khd->qhd", p, v)
        if not st["train"]:
            continue
        do = st["dy"][i].double()
        dv[i, idx] = torch.einsum("hqk,qhd->khd", p, do)
        ds = torch.einsum("qhd,khd->hqk", do, v)
        ds = p * (ds - (p * ds).sum(-1, keepdim=True)) * c
        dq[i] = torch.einsum("hqk,khd->qhd", ds, k)
        dk[i, idx] = torch.einsum("hqk,qhd->khd", ds, q)
    return (o, dq, dk, dv) if st["train"] else o


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(st) if case["op"] == "norm" else _exact_cross(st)

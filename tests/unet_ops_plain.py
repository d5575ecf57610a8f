"""Group norm and cross attention with their gradients in 64 bits, from the
formulas, with an error bound for every value that comes out.

The bounds count roundings.  u = eps / 2 of the element type is one rounding of a
result; f = 2^-24 one operation in 32 bits.  Sums of n terms in 32 bits are taken
to lose at most ``SUM`` * f of the sum of magnitudes, and the exponential and the
quotient of the activation, the reciprocal root and the joining of the statistics
a few f each: ``OPS`` covers them together.
"""

import torch

F32 = 2.0 ** -24
OPS = 64      # element-wise steps of one value: about twenty operations, __expf included
SUM = 256     # partial sums of at most 64 terms a thread, joined over threads and blocks


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(dtype, value):
    """One rounding of a result to its type: half a step, eps / 2 of the value down to
    the smallest normal number and a fixed eps / 2 of that number below it (fp16:
    2^-11 * 2^-14 = 2^-25, half of the subnormals' spacing)."""
    return half_step(dtype) * value.abs().clamp(min=torch.finfo(dtype).tiny)


def group_norm(x, groups, w=None, b=None, eps=1e-5, act=None, shift=None, dy=None, types=None):
    """y, and with dy the gradients, of float64 inputs.  ``types`` = (x's, the
    parameters', the shift's dtype) adds the bounds under "<name>_tol"."""
    B, C, H, W = x.shape
    w = torch.ones(C, dtype=x.dtype, device=x.device) if w is None else w
    b = torch.zeros(C, dtype=x.dtype, device=x.device) if b is None else b
    u = x if shift is None else x + shift[:, :, None, None]

    def spread(t):  # [B, groups] -> [B, C, 1, 1]
        return t.repeat_interleave(C // groups, dim=1)[:, :, None, None]

    g = u.reshape(B, groups, -1)
    mean, var = spread(g.mean(-1)), spread(g.var(-1, unbiased=False))
    r = (var + eps) ** -0.5
    n = (u - mean) * r
    wc, bc = w[None, :, None, None], b[None, :, None, None]
    z = n * wc + bc
    s = torch.sigmoid(z) if act else torch.ones_like(z)
    y = z * s if act else z
    out = {"y": y}
    # n carries the rounding of the mean (and of the shift) beside its own.
    n_off = OPS * F32 * (n.abs() + (mean.abs() + (u - x).abs()) * r)
    z_off = n_off * wc.abs() + OPS * F32 * (z.abs() + bc.abs())
    if types:
        # |act'| <= 1.1
        out["y_tol"] = rounded(types[0], y) + 1.1 * z_off + OPS * F32 * y.abs() + 1e-12
    if dy is None:
        return out
    da = s * (1 + z * (1 - s)) if act else s
    dz = dy * da

    def mean_g(t):
        return spread(t.reshape(B, groups, -1).mean(-1))

    A, D = mean_g(wc * dz), mean_g(wc * dz * n)
    out["dx"] = r * (wc * dz - A - n * D)
    out["dw"], out["db"] = (dz * n).sum((0, 2, 3)), dz.sum((0, 2, 3))
    out["ds"] = out["dx"].sum((2, 3))
    if types:
        # |act''| <= 0.5
        dz_off = dy.abs() * ((0.5 * z_off if act else 0) + OPS * F32)
        A_off = mean_g(wc.abs() * dz_off) + SUM * F32 * mean_g((wc * dz).abs())
        D_off = (mean_g(wc.abs() * (dz_off * n.abs() + dz.abs() * n_off))
                 + SUM * F32 * mean_g((wc * dz * n).abs()))
        dx_off = r * (wc.abs() * dz_off + A_off + n.abs() * D_off + n_off * D.abs()
                      + OPS * F32 * ((wc * dz).abs() + A.abs() + (n * D).abs()))
        out["dx_tol"] = rounded(types[0], out["dx"]) + dx_off + 1e-12
        out["dw_tol"] = (rounded(types[1], out["dw"]) + 1e-12 + (dz_off * n.abs() + dz.abs() * n_off
                         + SUM * F32 * (dz * n).abs()).sum((0, 2, 3)))
        out["db_tol"] = (rounded(types[1], out["db"]) + 1e-12
                         + (dz_off + SUM * F32 * dz.abs()).sum((0, 2, 3)))
        whole = r * ((wc * dz).abs() + A.abs() + (n * D).abs())
        out["ds_tol"] = (rounded(types[2], out["ds"]) + 1e-12
                         + (dx_off + SUM * F32 * whole).sum((2, 3)))
    return out


def cross_attention(q, k, v, mask=None, scale=1.0, do=None, dtype=None):
    """o, and with do the gradients, of float64 inputs; ``dtype`` (the element type)
    adds the bounds.  Masked keys are left out altogether."""
    B, Nq, H, D = q.shape
    keep = torch.ones(B, k.shape[1], dtype=torch.bool, device=q.device)
    bias = torch.zeros(B, k.shape[1], dtype=q.dtype, device=q.device)
    if mask is not None:
        if mask.dtype == torch.bool:
            keep = mask
        else:
            keep = mask != float("-inf")
            bias = torch.where(keep, mask, torch.zeros_like(mask)).to(q.dtype)
    kk = torch.where(keep[:, :, None, None], k, torch.zeros_like(k))
    vv = torch.where(keep[:, :, None, None], v, torch.zeros_like(v))
    kept = keep[:, None, None, :]
    s = torch.einsum("bqhd,bkhd->bhqk", q, kk) * scale + bias[:, None, None, :]
    top = s.masked_fill(~kept, float("-inf")).amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    e = torch.where(kept, torch.exp(s - top), torch.zeros_like(s))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    out = {"o": torch.einsum("bhqk,bkhd->bqhd", p, vv)}
    if dtype:
        h = half_step(dtype)
        # What a probability is off by, relative: the score's 32-bit sum (D terms and
        # the change of base) enters the exponent, of its own row and of the maximum.
        mag = torch.einsum("bqhd,bkhd->bhqk", q.abs(), kk.abs()) * abs(scale)
        mag = (mag + torch.where(kept, bias[:, None, None, :].abs().clamp(max=1e4), 0.0)).amax(-1, keepdim=True)
        p_rel = 4 * F32 * (D + 8) * (mag + 1) + SUM * F32
        # One rounding of p to the element type for the product.  Below fp16's normal
        # range that is half a subnormal step, 2^-25, of what the kernels hold: e^(s -
        # max), at least p, in the forward pass; 2^10 p in the gradient.
        p_off = p * (h + p_rel)
        tail = (2.0 ** -25 if dtype == torch.float16 else 0.0) * kept
        out["o_tol"] = (rounded(dtype, out["o"]) + 1e-12 + torch.einsum(
            "bhqk,bkhd->bqhd", p_off + tail + SUM * F32 * p, vv.abs()))
    if do is None:
        return out
    out["dv"] = torch.einsum("bhqk,bqhd->bkhd", p, do)
    dp = torch.einsum("bqhd,bkhd->bhqk", do, vv)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    out["dq"] = torch.einsum("bhqk,bkhd->bqhd", ds, kk)
    out["dk"] = torch.einsum("bhqk,bqhd->bkhd", ds, q)
    if dtype:
        out["dv_tol"] = (rounded(dtype, out["dv"]) + 1e-12
                         + torch.einsum("bhqk,bqhd->bkhd", p_off + tail / 1024 + SUM * F32 * p,
                                        do.abs()))
        dp_mag = torch.einsum("bqhd,bkhd->bhqk", do.abs(), vv.abs())
        dp_off = F32 * (D + 8) * dp_mag
        # sum(p dp) from the probabilities, or from the rounded o: one rounding of each
        # element of o against do.
        o_mag = torch.einsum("bqhd,bqhd->bhq", do.abs(), out["o_tol"])[..., None]
        delta_off = ((p * dp_off).sum(-1, keepdim=True) + o_mag
                     + ((p * p_rel + SUM * F32 * p) * dp.abs()).sum(-1, keepdim=True))
        # One rounding of ds to the element type for the products.  fp16 holds ds scaled
        # so that twice the largest |dp| of some earlier tile of the head, or of this
        # one, came to 2^10 or more: half a subnormal step, 2^-25, is then at most
        # 2^-25 * 2 / 2^10 = 2^-34 of the head's largest |dp|.
        ds_off = abs(scale) * p * ((h + p_rel) * (dp - delta).abs() + dp_off + delta_off)
        if dtype == torch.float16:
            biggest = (dp * kept).abs().amax((-1, -2), keepdim=True)
            ds_off = ds_off + abs(scale) * 2.0 ** -34 * biggest * kept
        out["dq_tol"] = (rounded(dtype, out["dq"]) + 1e-12 + torch.einsum(
            "bhqk,bkhd->bqhd", ds_off + SUM * F32 * ds.abs(), kk.abs()))
        out["dk_tol"] = (rounded(dtype, out["dk"]) + 1e-12 + torch.einsum(
            "bhqk,bqhd->bkhd", ds_off + SUM * F32 * ds.abs(), q.abs()))
    return out

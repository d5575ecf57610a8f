"""The UNet operators around the 3x3 convolutions, on the GPU kernels of
``libnova_winograd.so``:

    nova_group_norm        group normalisation with its activation on channels-last
                           activations, a per-sample channel shift added first
    nova_cross_attention   attention of one set of tokens to an encoder's states
    NovaGroupNorm          module form of the norm, drop-in for ``nn.GroupNorm`` of
                           [B, C, H, W]

No reference counterpart: the reference's UNet callers leave both to the host
framework (Jayluci4/nova-wino-amd ``benchmarks/bench_sd_unet.py:38-109``).  Both
are differentiable once (backwards: a tangent is refused), run on the caller's current CUDA stream, allocate through
torch's caching allocator only and never synchronize, so both can be captured
into a CUDA graph.  Like the rest of the package they have no CPU fallback.
"""

import ctypes

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from nova_winograd.conv2d import _raw_stream
from nova_winograd.ops import check, get_lib

DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MASK_NONE, MASK_BOOL = -1, 3
ACTIVATIONS = {None: 0, "silu": 1}
MAX_HEAD_DIM = 160
MAX_GROUP_CHANNELS = 8192
_MOST = 2 ** 31 - 4096  # pixels, groups or rows that the library counts in 32 bits

_fns, _workspace_sizes = {}, {}


def _fn(name):
    """A library function, looked up once."""
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(get_lib(), name)
    return f


def _workspace(name, device, *sizes):
    """Workspace of a call: the library says how much, by the SMs of the device, the
    caching allocator gives it."""
    key = (name, device.index, sizes)
    n = _workspace_sizes.get(key)
    if n is None:
        with torch.cuda.device(device):
            n = _fn(name)(*sizes)
        if n < 0:
            raise ValueError(f"bad sizes for {name[:-len('_workspace_bytes')]}: {sizes}")
        if len(_workspace_sizes) > 4096:
            _workspace_sizes.clear()
        _workspace_sizes[key] = n
    if n == 0:
        return None, None, 0
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), n


def _call(name, device, *args):
    """One library call on ``device`` (the library goes by the operands' device) and
    its current stream."""
    status = (_fns.get(name) or _fn(name))(*args, _raw_stream(device.index))
    if status:
        check(status, name)


def _p(t):
    return None if t is None else t.data_ptr()


def _expect(t, dtype, shape, device):
    """Refuses a saved tensor that a hook (one that keeps it elsewhere meanwhile, say)
    handed back as another.  Its strides may differ, and are asked anew."""
    if t is not None and not (t.dtype is dtype and t.shape == shape and t.device == device):
        raise RuntimeError(f"a saved-tensor hook handed back {t.dtype} {list(t.shape)} on "
                           f"{t.device} for {dtype} {list(shape)} on {device}")


def _differentiated(*tensors):
    """Whether a call goes through its autograd function: a gradient is wanted, or a
    dual level is open, in which the function refuses an input that has a tangent
    (torch counts the open levels from -1)."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


# ---------------------------------------------------------------------------
# Group norm
# ---------------------------------------------------------------------------

def _pixel_strides(x):
    """(batch stride, pixel stride) of x [B, C, H, W] whose channels lie next to
    each other and whose pixels are evenly spaced (channels-last, or channels of a
    wider channels-last tensor); None for any other layout."""
    B, C, H, W = x.shape
    sb, sc, sh, sw = x.stride()
    if C > 1 and sc != 1:
        return None
    pitch = sw if W > 1 else sh if H > 1 else C
    if pitch < C or (H > 1 and W > 1 and sh != W * pitch):
        return None
    return (sb if B > 1 else 0), pitch


def _even_pixels(x):
    """x, or a channels-last copy where its pixels are not evenly spaced, and its strides."""
    strides = _pixel_strides(x)
    if strides is None:
        x = x.contiguous(memory_format=torch.channels_last)
        strides = _pixel_strides(x)
    return x, strides


def _vectors(dtype, t, strides):
    """Whether the pixels of t start on 16 bytes."""
    v = 3 if dtype == 2 else 7
    return 0 if t.data_ptr() & 15 or (strides[0] | strides[1]) & v else 1


def _empty_channels_last(x):
    B, C, H, W = x.shape
    return torch.empty_strided((B, C, H, W), (H * W * C, 1, W * C, C), dtype=x.dtype,
                               device=x.device)


def _norm_forward(x, strides, num_groups, weight, bias, eps, act, shift, want_stats):
    B, C, H, W = x.shape
    device = x.device
    y = _empty_channels_last(x)
    stats = None
    if want_stats:
        stats = torch.empty((2, B, num_groups), dtype=torch.float32, device=device)
    if B and H and W:
        dtype = DTYPES[x.dtype]
        ws, at, n = _workspace("nova_group_norm_workspace_bytes", device, B, H * W, C, num_groups,
                               dtype, _vectors(dtype, x, strides), 0)
        param = weight if weight is not None else bias
        _call("nova_group_norm_v2", device, x.data_ptr(), _p(weight), _p(bias), _p(shift),
              y.data_ptr(), _p(stats), at, n, B, H * W, C, num_groups, *strides, dtype,
              2 if param is None else DTYPES[param.dtype],
              2 if shift is None else DTYPES[shift.dtype], act, eps)
    return y, stats


class _GroupNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, shift, strides, num_groups, eps, act):
        y, stats = _norm_forward(x, strides, num_groups, weight, bias, eps, act, shift, True)
        param_type = weight.dtype if weight is not None else bias.dtype if bias is not None else None
        ctx.save_for_backward(x, weight, bias, shift, stats)
        ctx.num_groups, ctx.act = num_groups, act
        ctx.types = param_type, None if shift is None else shift.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_norm_backward_once if torch.is_grad_enabled() else _norm_backward)(ctx, dy)


def _norm_backward(ctx, dy):
    x, *rest = ctx.saved_tensors
    weight, bias, shift, stats = map(_dense, rest)
    B, C, H, W = dy.shape
    device, (param_type, shift_type) = dy.device, ctx.types
    _expect(x, dy.dtype, dy.shape, device)
    _expect(weight, param_type, (C,), device)
    _expect(bias, param_type, (C,), device)
    _expect(shift, shift_type, (B, C), device)
    _expect(stats, torch.float32, (2, B, ctx.num_groups), device)
    need = ctx.needs_input_grad
    dx = _empty_channels_last(x)
    dw = torch.empty_like(weight) if need[1] else None
    db = torch.empty_like(bias) if need[2] else None
    ds = torch.empty_like(shift) if need[3] else None
    if not dx.numel():
        for t in (dw, db, ds):
            if t is not None:
                t.zero_()
        return dx, dw, db, ds, None, None, None, None
    x, xs = _even_pixels(x)
    dy, ys = _even_pixels(dy)
    dtype = DTYPES[x.dtype]
    ws, at, n = _workspace("nova_group_norm_workspace_bytes", x.device, B, H * W, C,
                           ctx.num_groups, dtype,
                           _vectors(dtype, x, xs) and _vectors(dtype, dy, ys), 1)
    param = weight if weight is not None else bias
    _call("nova_group_norm_grad_v2", x.device, x.data_ptr(), dy.data_ptr(), _p(weight), _p(bias),
          _p(shift), stats.data_ptr(), dx.data_ptr(), _p(dw), _p(db), _p(ds), at, n, B, H * W, C,
          ctx.num_groups, *xs, *ys, dtype, 2 if param is None else DTYPES[param.dtype],
          2 if shift is None else DTYPES[shift.dtype], ctx.act)
    return (dx if need[0] else None), dw, db, ds, None, None, None, None


_norm_backward_once = torch.autograd.function.once_differentiable(_norm_backward)


def _check_param(name, t, shape, device):
    if t.dtype in DTYPES and t.shape == shape and t.device == device:
        return t if t.is_contiguous() else t.contiguous()
    if t.device != device:
        raise ValueError(f"{name} must be on the input's device")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name} must be float16, bfloat16 or float32, got {t.dtype}")
    raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")


def nova_group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, activation=None, shift=None):
    """``act(group_norm(x + shift[:, :, None, None]))`` on channels-last activations.

    Args:
        x:          [B, C, H, W] float16, bfloat16 or float32 CUDA tensor in
                    channels-last layout, or a channel slice of one (channels next to
                    each other, pixels evenly spaced).
        num_groups: number of groups; divides C, at most 8192 channels each.
        weight, bias: [C] float16, bfloat16 or float32, both of one type, or None.
        eps:        added to the variance.
        activation: None or "silu".
        shift:      [B, C] float16, bfloat16 or float32 added to x before the norm (a
                    residual block's time embedding), or None.

    Returns a channels-last tensor of x's type.  Statistics and arithmetic are in 32
    bits (sums over samples in 64), with one rounding at the end; results repeat bit
    for bit.  Gradients for x, weight, bias and shift.
    """
    if x.dim() != 4:
        raise ValueError(f"x must be [B, C, H, W], got {list(x.shape)}")
    if x.dtype not in DTYPES:
        raise TypeError(f"x must be float16, bfloat16 or float32, got {x.dtype}")
    B, C, H, W = x.shape
    if num_groups < 1 or C < 1 or C % num_groups:
        raise ValueError(f"{C} channels do not divide into {num_groups} groups")
    if C // num_groups > MAX_GROUP_CHANNELS:
        raise ValueError(f"more than {MAX_GROUP_CHANNELS} channels per group: {C // num_groups}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    strides = _pixel_strides(x)
    if strides is None:
        raise ValueError("x must be channels-last (torch.channels_last, or channels of one)")
    if B * H * W > _MOST or B * num_groups > _MOST:
        raise ValueError("x must have at most 2^31 - 4096 pixels, and as many groups in all")
    if weight is not None:
        weight = _check_param("weight", weight, (C,), x.device)
    if bias is not None:
        bias = _check_param("bias", bias, (C,), x.device)
        if weight is not None and bias.dtype != weight.dtype:
            raise TypeError("weight and bias must have one type")
    if shift is not None:
        shift = _check_param("shift", shift, (B, C), x.device)
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    act = ACTIVATIONS[activation]
    if _differentiated(x, weight, bias, shift):
        return _GroupNorm.apply(x, weight, bias, shift, strides, num_groups, eps, act)
    return _norm_forward(x, strides, num_groups, weight, bias, eps, act, shift, False)[0]


class NovaGroupNorm(nn.GroupNorm):
    """``nn.GroupNorm`` of [B, C, H, W] with its activation fused in, on ``nova_group_norm``.

    Channels-last input gives channels-last output.  Contiguous NCHW input goes
    through an on-device copy to channels-last and back.
    """

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation=None,
                 device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine, device=device,
                         dtype=dtype)
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be None or 'silu', got {activation!r}")
        self.activation = activation

    def forward(self, x, shift=None):
        back = x.dim() == 4 and _pixel_strides(x) is None
        if back:
            x = x.contiguous(memory_format=torch.channels_last)
        y = nova_group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation,
                            shift)
        return y.contiguous() if back else y

    @classmethod
    def from_group_norm(cls, norm, activation=None):
        """The same norm (its parameters are shared, not copied)."""
        new = cls(norm.num_groups, norm.num_channels, eps=norm.eps, affine=False,
                  activation=activation)
        new.affine, new.weight, new.bias = norm.affine, norm.weight, norm.bias
        return new.train(norm.training)

    def extra_repr(self):
        return f"{super().extra_repr()}, activation={self.activation}"


# ---------------------------------------------------------------------------
# Cross attention
# ---------------------------------------------------------------------------

def _one_tile(D):
    """Keys that the gradient takes in one tile; with more it reads o, and what the
    rounding of o left off, for the row sums of do . o."""
    return 128 if D <= 128 else 80


def _rows(t):
    """t [B, N, H, D] with its rows' elements next to each other and every row on 16
    bytes: t itself where it lies so, else a contiguous copy (contiguous() alone may
    return t: it looks neither at the start nor at the strides of single indices)."""
    sb, sn, sh, sd = t.stride()
    if (sd == 1 and sb % 8 == 0 and sn % 8 == 0 and sh % 8 == 0 and sn and
            t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(q, k, v, mask, *more):
    vals = [*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]]
    vals += list(mask.stride()) if mask is not None else [0, 0]
    for t in more:
        vals += t.stride()[:3]
    return (ctypes.c_longlong * len(vals))(*vals)


def _mask_type(mask):
    if mask is None:
        return MASK_NONE
    return MASK_BOOL if mask.dtype == torch.bool else DTYPES[mask.dtype]


def _cross_forward(q, k, v, mask, scale, train):
    B, Nq, H, D = q.shape
    Nk = k.shape[1]
    out = torch.empty((B, Nq, H, D), dtype=q.dtype, device=q.device)
    low = lse = None
    if train:
        lse = torch.empty((B, H, Nq), dtype=torch.float32, device=q.device)
        if Nk > _one_tile(D):
            low = torch.empty((B, Nq, H, D), dtype=q.dtype, device=q.device)
    if out.numel() and Nk:
        ws, at, n = _workspace("nova_cross_attention_workspace_bytes", q.device, B, Nq, Nk, H, D, 0)
        _call("nova_cross_attention_v2", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(),
              _p(mask), out.data_ptr(), _p(low), _p(lse), at, n, B, Nq, Nk, H, D,
              _strides(q, k, v, mask), DTYPES[q.dtype], _mask_type(mask), scale)
    else:
        out.zero_()
    return out, low, lse


class _CrossAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, mask, scale):
        out, low, lse = _cross_forward(q, k, v, mask, scale, True)
        ctx.save_for_backward(q, k, v, mask, None if low is None else out, low, lse)
        ctx.scale, ctx.mask_dtype = scale, None if mask is None else mask.dtype
        return out

    @staticmethod
    def backward(ctx, do):
        return (_cross_backward_once if torch.is_grad_enabled() else _cross_backward)(ctx, do)


def _cross_backward(ctx, do):
    q, k, v, mask, *rest = ctx.saved_tensors
    B, Nq, H, D = do.shape
    Nk, dtype, device = k.shape[1], do.dtype, do.device
    out, low, lse = map(_dense, rest)
    for t in (q, out, low):
        _expect(t, dtype, do.shape, device)
    for t in (k, v):
        _expect(t, dtype, (B, Nk, H, D), device)
    _expect(mask, ctx.mask_dtype, (B, Nk), device)
    _expect(lse, torch.float32, (B, H, Nq), device)
    q, k, v = _rows(q), _rows(k), _rows(v)
    dq = torch.empty((B, Nq, H, D), dtype=q.dtype, device=q.device)
    dk = torch.empty((B, Nk, H, D), dtype=q.dtype, device=q.device)
    dv = torch.empty((B, Nk, H, D), dtype=q.dtype, device=q.device)
    if dq.numel() and Nk:
        do = _rows(do)
        ws, at, n = _workspace("nova_cross_attention_workspace_bytes", q.device, B, Nq, Nk, H, D, 1)
        _call("nova_cross_attention_grad_v2", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(),
              _p(mask), _p(out), _p(low), do.data_ptr(), lse.data_ptr(), dq.data_ptr(),
              dk.data_ptr(), dv.data_ptr(), at, n, B, Nq, Nk, H, D, _strides(q, k, v, mask, do),
              DTYPES[q.dtype], _mask_type(mask), ctx.scale)
    else:
        for t in (dq, dk, dv):
            t.zero_()
    need = ctx.needs_input_grad
    return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None)


_cross_backward_once = torch.autograd.function.once_differentiable(_cross_backward)


def nova_cross_attention(q, k, v, key_mask=None, scale=None):
    """``softmax(scale * q k^T + key_mask) v`` for every sample and head.

    Args:
        q:        [B, Nq, H, D] float16 or bfloat16 CUDA tensor, D a multiple of 8 up
                  to 160.
        k, v:     [B, Nk, H, D], of q's type.  Any strides; a tensor whose rows are
                  not contiguous on 16 bytes is copied first.
        key_mask: None, a bool [B, Nk] tensor (True: the key takes part), or a float
                  [B, Nk] tensor added to the scores (float16, bfloat16 or float32; minus
                  infinity: the key takes no part).  Not differentiable.
        scale:    default 1 / sqrt(D).

    A key that takes no part is never multiplied, whatever k and v hold there.  A
    query without keys gets zeros and passes no gradient on, whatever it and its
    gradient hold.  Finite biases count as 32-bit sums with them do: with the lowest
    value, or -1e9, for every key of a sample its rows are uniform.  Returns
    [B, Nq, H, D], contiguous.

    Products are accumulated and the softmax is computed in 32 bits.  Probabilities,
    and in the gradient their derivatives too, are rounded to q's type once, as
    operands of the products with v, k, q and the incoming gradient; what the rounding
    of the output left off goes to the gradient in q's type as well.  Gradients for q,
    k and v repeat bit for bit.

    The kernels' waits are bounded.  One that expires leaves an output that is not to
    be used, and ``nova_cross_attention_status()`` of the library (``ops.get_lib()``)
    reports it.
    """
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k and v must be [B, N, H, D], got {list(q.shape)}, {list(k.shape)} "
                         f"and {list(v.shape)}")
    dtype, device = q.dtype, q.device
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise TypeError(f"q must be float16 or bfloat16, got {dtype}")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError("q, k and v must have one type")
    if k.device != device or v.device != device:
        raise ValueError("q, k and v must be on one device")
    B, Nq, H, D = q.shape
    Nk = k.shape[1]
    if k.shape != (B, Nk, H, D) or v.shape != k.shape:
        raise ValueError(f"k and v must both be [{B}, Nk, {H}, {D}], got {list(k.shape)} and "
                         f"{list(v.shape)}")
    if D % 8 or not 8 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"head width must be a multiple of 8 up to {MAX_HEAD_DIM}, got {D}")
    if B * H * max(Nq, Nk) > _MOST:
        raise ValueError("q, k and v must have at most 2^31 - 4096 rows")
    if key_mask is not None:
        if key_mask.dtype != torch.bool and key_mask.dtype not in DTYPES:
            raise TypeError(f"key_mask must be bool, float16, bfloat16 or float32, got "
                            f"{key_mask.dtype}")
        if key_mask.shape != (B, Nk):
            raise ValueError(f"key_mask must be [{B}, {Nk}], got {list(key_mask.shape)}")
        if key_mask.device != q.device:
            raise ValueError("key_mask must be on q's device")
        if key_mask.requires_grad:
            raise ValueError("key_mask is not differentiable")
    if not q.is_cuda:
        raise ValueError("q, k and v must be CUDA tensors")
    scale = D ** -0.5 if scale is None else float(scale)
    q, k, v = _rows(q), _rows(k), _rows(v)
    if _differentiated(q, k, v):
        return _CrossAttention.apply(q, k, v, key_mask, scale)
    return _cross_forward(q, k, v, key_mask, scale, False)[0]

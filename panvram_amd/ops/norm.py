"""The residual stream's addition and root-mean-square norm (panvram_amd/csrc/pv_norm.hip)."""
import torch

from .. import _native as N
from ._call import DTYPES, call, on_gpu, once, ptr

_FORMATS = {torch.float8_e4m3fn: N.E4M3, torch.int8: N.INT8}


def _flat(t):
    """(t, the distance of its rows): `t` as rows of D neighbouring elements, itself or a view of it where its layout
    allows, else a copy."""
    if t.is_contiguous():
        return t, t.shape[-1]
    t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _forward(index, x, residual, weight, eps, keep_rstd):
    """y, the stream (None without a residual), and 1 / the root mean square of each row where it is kept"""
    shape, dtype, dev = x.shape, x.dtype, x.device
    D = shape[-1]
    count = x.numel() // D
    x, xs = _flat(x)
    residual, rs = (None, 0) if residual is None else _flat(residual)
    y = torch.empty(shape, dtype=dtype, device=dev)
    stream = torch.empty(shape, dtype=dtype, device=dev) if residual is not None else None
    rstd = torch.empty(count, dtype=torch.float32, device=dev) if keep_rstd else None
    call(N.lib().pv_add_rms_norm_hip, index, x.data_ptr(), ptr(residual), weight.data_ptr(), count, D, xs, rs, eps, DTYPES[dtype], y.data_ptr(), ptr(stream), ptr(rstd))
    return y, stream, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, stream, rstd = _forward(x.get_device(), x, residual, weight, eps, True)
        ctx.save_for_backward(x if stream is None else stream, rstd, weight)
        ctx.alone = residual is None
        ctx.set_materialize_grads(False)
        return y if stream is None else (y, stream)

    @staticmethod
    @once
    def backward(ctx, d_y, d_stream=None):
        s, rstd, weight = ctx.saved_tensors
        if d_y is None:
            return (d_stream, None if ctx.alone else d_stream, None, None)
        D, count, dtype, dev = s.shape[-1], rstd.numel(), s.dtype, s.device
        d_y = d_y.contiguous()
        d_stream = d_stream.contiguous() if d_stream is not None else None
        d = torch.empty(s.shape, dtype=dtype, device=dev)
        d_weight = torch.empty(D, dtype=torch.float32, device=dev)
        L = N.lib()
        size = L.pv_add_rms_norm_work_bytes(count, D)
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        flat, ss = _flat(s)
        call(L.pv_add_rms_norm_backward_hip, s.get_device(), flat.data_ptr(), rstd.data_ptr(), weight.data_ptr(), count, D, ss, d_y.data_ptr(), ptr(d_stream),
             DTYPES[dtype], d.data_ptr(), d_weight.data_ptr(), ptr(work), size)
        return d, None if ctx.alone else d, d_weight, None


def _checked(name, x, residual, weight):
    """The tensors' GPU, and the weight in 32 bits"""
    index = on_gpu(name, x, residual, weight)
    shape, dtype = x.shape, x.dtype
    if len(shape) < 1 or shape[-1] < 1 or dtype not in DTYPES:
        raise ValueError(f"{name}: x is float32, bfloat16 or float16 with rows of one element or more along its last dimension, got {dtype} {list(shape)}")
    if residual is not None and (residual.shape != shape or residual.dtype != dtype):
        raise ValueError(f"{name}: residual is like x, got {residual.dtype} {list(residual.shape)}")
    if weight.shape != shape[-1:] or not weight.is_floating_point():
        raise ValueError(f"{name}: weight is [{shape[-1]}], got {weight.dtype} {list(weight.shape)}")
    if weight.dtype != torch.float32:
        weight = weight.float()
    return index, weight.contiguous()


def add_rms_norm(x, residual, weight, eps=1e-6):
    """(y, stream): stream = x + residual in x's type, as the next layer adds to it, and
    y = stream / sqrt(mean(stream^2) + eps) * weight over the last dimension.

    x, residual: float32, bfloat16 or float16, alike; residual None: the norm of x itself, and x is the stream. weight: [D],
    used in 32 bits. What is normalised is the stored stream, so what the backward pass keeps is the stream and one number
    per row. Gradients flow to x, residual and weight, from y and from stream."""
    index, weight = _checked("add_rms_norm", x, residual, weight)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        got = _AddRmsNorm.apply(x, residual, weight, eps)
        return got if residual is not None else (got, x)
    y, stream, _ = _forward(index, x, residual, weight, eps, False)
    return y, x if stream is None else stream


@torch.no_grad()
def add_rms_norm_8bit(x, residual, weight, eps=1e-6, dtype=torch.float8_e4m3fn):
    """(q, scale, stream): as add_rms_norm, with y as q * scale[..., None]: scale float32 per row, max |y| over the format's
    largest value (448, or 127 for torch.int8), and q = y / scale to the nearest value, ties to even. A row of zeros has
    scale 0. A row with a NaN or an infinity has scale NaN (its q is NaN in float8, 0 in int8). No gradients."""
    index, weight = _checked("add_rms_norm_8bit", x, residual, weight)
    if dtype not in _FORMATS:
        raise ValueError(f"add_rms_norm_8bit: dtype is torch.float8_e4m3fn or torch.int8, got {dtype}")
    shape, dev, D = x.shape, x.device, x.shape[-1]
    flat, xs = _flat(x)
    res, rs = (None, 0) if residual is None else _flat(residual)
    q = torch.empty(shape, dtype=dtype, device=dev)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    stream = torch.empty(shape, dtype=x.dtype, device=dev) if res is not None else None
    call(N.lib().pv_add_rms_norm_8bit_hip, index, flat.data_ptr(), ptr(res), weight.data_ptr(), x.numel() // D, D, xs, rs, eps, DTYPES[x.dtype], _FORMATS[dtype],
         q.data_ptr(), scale.data_ptr(), ptr(stream))
    return q, scale, x if stream is None else stream

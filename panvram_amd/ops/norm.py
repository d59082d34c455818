"""The residual stream's addition and root-mean-square norm (panvram_amd/csrc/pv_norm.hip)."""
import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from ._call import DTYPES, call, need, on_gpu, ptr

_FORMATS = {torch.float8_e4m3fn: N.E4M3, torch.int8: N.INT8}


def _flat(t):
    """`t` as [rows, D] with neighbouring elements in a row: a view where its layout allows."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _forward(x, residual, weight, eps, keep_rstd):
    N_, D = x.shape
    y = torch.empty(N_, D, dtype=x.dtype, device=x.device)
    stream = torch.empty(N_, D, dtype=x.dtype, device=x.device) if residual is not None else None
    rstd = torch.empty(N_, dtype=torch.float32, device=x.device) if keep_rstd else None
    call("pv_add_rms_norm_hip", x.get_device(), x.data_ptr(), ptr(residual), weight.data_ptr(), N_, D, x.stride(0), residual.stride(0) if residual is not None else 0,
         eps, DTYPES[x.dtype], y.data_ptr(), ptr(stream), ptr(rstd))
    return y, stream, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        flat, res = _flat(x), _flat(residual) if residual is not None else None
        y, stream, rstd = _forward(flat, res, weight, eps, True)
        ctx.save_for_backward(flat if stream is None else stream, rstd, weight)
        ctx.alone = residual is None
        ctx.set_materialize_grads(False)
        y = y.view(x.shape)
        return y if stream is None else (y, stream.view(x.shape))

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y, d_stream=None):
        s, rstd, weight = ctx.saved_tensors
        if d_y is None:
            return (d_stream, None if ctx.alone else d_stream, None, None)
        rows, D = s.shape
        shape = d_y.shape
        d_y = d_y.contiguous()
        d_stream = d_stream.contiguous() if d_stream is not None else None
        d = torch.empty(shape, dtype=s.dtype, device=s.device)
        d_weight = torch.empty(D, dtype=torch.float32, device=s.device)
        work = torch.empty(N.lib().pv_add_rms_norm_work_bytes(rows, D), dtype=torch.uint8, device=s.device)
        call("pv_add_rms_norm_backward_hip", s.get_device(), s.data_ptr(), rstd.data_ptr(), weight.data_ptr(), rows, D, s.stride(0), d_y.data_ptr(), ptr(d_stream),
             DTYPES[s.dtype], d.data_ptr(), d_weight.data_ptr(), work.data_ptr(), work.numel())
        return d, None if ctx.alone else d, d_weight, None


def _checked(name, x, residual, weight):
    on_gpu(name, x, residual, weight)
    need(x.dim() >= 1 and x.dtype in DTYPES, f"{name}: x is float32, bfloat16 or float16 with rows along its last dimension, got {x.dtype} {list(x.shape)}")
    need(x.shape[-1] >= 1, f"{name}: rows of no elements")
    if residual is not None:
        need(residual.shape == x.shape and residual.dtype == x.dtype, f"{name}: residual is like x, got {residual.dtype} {list(residual.shape)}")
    need(weight.shape == x.shape[-1:] and weight.is_floating_point(), f"{name}: weight is [{x.shape[-1]}], got {weight.dtype} {list(weight.shape)}")
    return weight.float().contiguous()


def add_rms_norm(x, residual, weight, eps=1e-6):
    """(y, stream): stream = x + residual in x's type, as the next layer adds to it, and
    y = stream / sqrt(mean(stream^2) + eps) * weight over the last dimension.

    x, residual: float32, bfloat16 or float16, alike; residual None: the norm of x itself, and x is the stream. weight: [D],
    used in 32 bits. What is normalised is the stored stream, so what the backward pass keeps is the stream and one number
    per row. Gradients flow to x, residual and weight, from y and from stream."""
    weight = _checked("add_rms_norm", x, residual, weight)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        got = _AddRmsNorm.apply(x, residual, weight, float(eps))
        return got if residual is not None else (got, x)
    y, stream, _ = _forward(_flat(x), _flat(residual) if residual is not None else None, weight, float(eps), False)
    return y.view(x.shape), x if stream is None else stream.view(x.shape)


@torch.no_grad()
def add_rms_norm_8bit(x, residual, weight, eps=1e-6, dtype=torch.float8_e4m3fn):
    """(q, scale, stream): as add_rms_norm, with y as q * scale[..., None]: scale float32 per row, max |y| over the format's
    largest value (448, or 127 for torch.int8), and q = y / scale to the nearest value, ties to even. A row of zeros has
    scale 0. A row with a NaN or an infinity has scale NaN (its q is NaN in float8, 0 in int8). No gradients."""
    weight = _checked("add_rms_norm_8bit", x, residual, weight)
    need(dtype in _FORMATS, f"add_rms_norm_8bit: dtype is torch.float8_e4m3fn or torch.int8, got {dtype}")
    flat, res = _flat(x), _flat(residual) if residual is not None else None
    rows, D = flat.shape
    q = torch.empty(rows, D, dtype=dtype, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    stream = torch.empty(rows, D, dtype=x.dtype, device=x.device) if res is not None else None
    call("pv_add_rms_norm_8bit_hip", x.get_device(), flat.data_ptr(), ptr(res), weight.data_ptr(), rows, D, flat.stride(0), res.stride(0) if res is not None else 0,
         float(eps), DTYPES[x.dtype], _FORMATS[dtype], q.data_ptr(), scale.data_ptr(), ptr(stream))
    return q.view(x.shape), scale.view(x.shape[:-1]), x if stream is None else stream.view(x.shape)

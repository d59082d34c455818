"""The residual stream's addition with dropout, and its layer norm (panvram_amd/csrc/pv_layer.hip)."""
import torch

from .. import _native as N
from ._call import DTYPES, call, on_gpu, once, ptr
from .dropout import drop_args
from .norm import _flat


def _forward(index, x, residual, weight, bias, eps, drop, keep_stats):
    """y, the stream (None where it is x), and what the backward pass takes of each row where that is kept"""
    shape, dtype, dev = x.shape, x.dtype, x.device
    D = shape[-1]
    p, at, seed, site = drop
    x, xs = _flat(x)
    residual, rs = (None, 0) if residual is None else _flat(residual)
    y = torch.empty(shape, dtype=dtype, device=dev)
    stream = torch.empty(shape, dtype=dtype, device=dev) if residual is not None or p else None
    count = y.numel() // D
    stats = torch.empty((count, 3), dtype=torch.float32, device=dev) if keep_stats else None
    call(N.lib().pv_add_layer_norm_hip, index, x.data_ptr(), ptr(residual), weight.data_ptr(), ptr(bias), count, D, xs, rs, eps, p, ptr(at), seed, site,
         DTYPES[dtype], y.data_ptr(), ptr(stream), ptr(stats))
    return y, stream, stats


class _AddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, at, seed, site):
        y, stream, stats = _forward(x.get_device(), x, residual, weight, bias, eps, (p, at, seed, site), True)
        ctx.save_for_backward(x if stream is None else stream, stats, weight, at)
        ctx.alone, ctx.biased, ctx.drop = residual is None, bias is not None, (p, seed, site)
        ctx.set_materialize_grads(False)
        return y if stream is None else (y, stream)

    @staticmethod
    @once
    def backward(ctx, d_y, d_stream=None):
        s, stats, weight, at = ctx.saved_tensors
        p, seed, site = ctx.drop
        D, dtype, dev = s.shape[-1], s.dtype, s.device
        if d_y is None:
            if p and d_stream is not None:
                d_x = torch.empty(s.shape, dtype=dtype, device=dev)
                d_stream = d_stream.contiguous()
                call(N.lib().pv_dropout_hip, s.get_device(), d_stream.data_ptr(), d_x.numel(), p, ptr(at), seed, site, DTYPES[dtype], d_x.data_ptr())
            else:
                d_x = d_stream
            return d_x, None if ctx.alone else d_stream, None, None, None, None, None, None, None
        count = stats.shape[0]
        d_y = d_y.contiguous()
        d_stream = d_stream.contiguous() if d_stream is not None else None
        d = torch.empty(s.shape, dtype=dtype, device=dev)
        d_x = torch.empty(s.shape, dtype=dtype, device=dev) if p else None
        d_weight, d_bias = torch.empty(D, dtype=torch.float32, device=dev), torch.empty(D, dtype=torch.float32, device=dev)
        L = N.lib()
        size = L.pv_add_layer_norm_work_bytes(count, D)
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        flat, ss = _flat(s)
        call(L.pv_add_layer_norm_backward_hip, s.get_device(), flat.data_ptr(), stats.data_ptr(), weight.data_ptr(), count, D, ss, d_y.data_ptr(), ptr(d_stream), p,
             ptr(at), seed, site, DTYPES[dtype], d.data_ptr(), ptr(d_x), d_weight.data_ptr(), d_bias.data_ptr(), ptr(work), size)
        return d if d_x is None else d_x, None if ctx.alone else d, d_weight, d_bias if ctx.biased else None, None, None, None, None, None


def _vector(name, what, t, D):
    if t.shape != (D,) or not t.is_floating_point():
        raise ValueError(f"{name}: {what} is [{D}], got {t.dtype} {list(t.shape)}")
    return (t if t.dtype == torch.float32 else t.float()).contiguous()


def add_layer_norm(x, residual, weight, bias=None, eps=1e-5, dropout=0.0, seed=None, site=0):
    """(y, stream): stream = residual + dropout(x) in x's type, as the next layer adds to it, and
    y = (stream - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x, residual: float32, bfloat16 or float16, alike; residual None: the norm of dropout(x) itself. weight, bias: [D], used in 32
    bits; bias None: zero. dropout: the share of x's elements that is dropped before the addition; seed and site as in
    `ops.dropout`, whose elements these are (in evaluation leave dropout at 0). What is normalised is the stored stream, so what
    the backward pass keeps is the stream and three numbers per row. Gradients flow to x, residual, weight and bias, from y and
    from stream."""
    at = seed if isinstance(seed, torch.Tensor) else None
    index = on_gpu("add_layer_norm", x, residual, weight, bias, at)
    shape, dtype = x.shape, x.dtype
    if len(shape) < 1 or shape[-1] < 1 or dtype not in DTYPES:
        raise ValueError(f"add_layer_norm: x is float32, bfloat16 or float16 with rows of one element or more along its last dimension, got {dtype} {list(shape)}")
    if residual is not None and (residual.shape != shape or residual.dtype != dtype):
        raise ValueError(f"add_layer_norm: residual is like x, got {residual.dtype} {list(residual.shape)}")
    weight = _vector("add_layer_norm", "weight", weight, shape[-1])
    bias = None if bias is None else _vector("add_layer_norm", "bias", bias, shape[-1])
    drop = drop_args("add_layer_norm", dropout, seed, site)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        got = _AddLayerNorm.apply(x, residual, weight, bias, eps, *drop)
        return got if isinstance(got, tuple) else (got, x)
    y, stream, _ = _forward(index, x, residual, weight, bias, eps, drop, False)
    return y, x if stream is None else stream

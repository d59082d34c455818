"""Dropout from a counter-based generator, without a stored mask (panvram_amd/csrc/pv_dropout.hip)."""
import torch

from .. import _native as N
from ._call import DTYPES, call, on_gpu, once, ptr


def drop_args(name, p, seed, site):
    """(p, the seed's tensor or None, the seed's number, site) as the library takes them; p is 0 where nothing is dropped"""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{name}: the share that is dropped is in [0, 1], got {p}")
    if not 0 <= site < 1 << 32:
        raise ValueError(f"{name}: site is in [0, 2^32), got {site}")
    if int(p * 65536 + 0.5) == 0:
        p = 0.0
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"{name}: seed is an int64 tensor of one element, or an int, got {seed.dtype} {list(seed.shape)}")
        return p, seed if p else None, 0, site
    if seed is None:
        if p:
            raise ValueError(f"{name}: dropout takes a seed")
        seed = 0
    if not -1 << 63 <= seed < 1 << 64:
        raise ValueError(f"{name}: seed has 64 bits, got {seed}")
    return p, None, seed - (1 << 64) if seed >= 1 << 63 else seed, site


def _apply(index, x, p, at, seed, site):
    x = x.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    call(N.lib().pv_dropout_hip, index, x.data_ptr(), x.numel(), p, ptr(at), seed, site, DTYPES[x.dtype], y.data_ptr())
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, at, seed, site):
        ctx.save_for_backward(at)
        ctx.drop = (p, seed, site)
        return _apply(x.get_device(), x, p, at, seed, site)

    @staticmethod
    @once
    def backward(ctx, d_y):
        p, seed, site = ctx.drop
        return _apply(d_y.get_device(), d_y, p, ctx.saved_tensors[0], seed, site), None, None, None, None


def dropout(x, p, seed, site=0):
    """x with each element dropped (0, whatever it was) with probability p, the others divided by the share that is kept.

    x: float32, bfloat16 or float16, any shape. p in [0, 1], used to a multiple of 2^-16. seed: 64 bits, an int or an int64 tensor
    of one element on x's GPU, which is read when the kernel runs: a captured graph that draws or counts it up drops other
    elements at each replay. site: a number in [0, 2^32) for each place of a model that uses one seed, so that no two drop the
    same. Whether an element is dropped is a function of seed, site and its index in x alone; the backward pass asks that
    function again, and a seed tensor changed in between is autograd's error. Equal arguments give equal results."""
    index = on_gpu("dropout", x, seed if isinstance(seed, torch.Tensor) else None)
    if x.dtype not in DTYPES:
        raise ValueError(f"dropout: x is float32, bfloat16 or float16, got {x.dtype}")
    p, at, seed, site = drop_args("dropout", p, seed, site)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, p, at, seed, site)
    return _apply(index, x, p, at, seed, site)

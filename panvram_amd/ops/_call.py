"""What the operators' Python side shares: checks of tensors, and calls of the library on the current stream. A call of a
few rows costs its host time, so what is asked of the arguments is asked once and messages are made only where they are
raised."""
import threading

import torch
from torch.autograd import forward_ad as _fw
from torch.autograd.function import once_differentiable

from .. import _native as N
from .._streams import raw as _raw

DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}


def no_tangents(name, tensors):
    """An error if one of `tensors` carries a forward-mode derivative: the kernels would drop it without a word. (Asked for
    each tensor only while a level of dual numbers is open, of which torch keeps the number.)"""
    if getattr(_fw, "_current_level", 0) < 0:
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and _fw.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")


def on_gpu(name, first, *others):
    """The index of the GPU that all tensors (None: left out) are on; an error naming what is not there, and for forward-mode
    derivatives."""
    no_tangents(name, (first, *others))
    index = first.get_device() if isinstance(first, torch.Tensor) else -1
    for t in others:
        if t is not None and (index < 0 or not isinstance(t, torch.Tensor) or t.get_device() != index):
            index = -1
    if index >= 0:
        return index
    where = []
    for t in (first, *others):
        if t is not None:
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name}: tensors expected, got {type(t).__name__}")
            if not t.is_cuda:
                raise RuntimeError(f"{name} runs on the GPU only; got a tensor on {t.device}")
            where.append(str(t.device))
    raise ValueError(f"{name}: tensors on {' and '.join(sorted(set(where)))}")


_local = threading.local()


def call(fn, index, *args):
    """fn(*args, stream, err, errcap), a function of the library, on GPU `index`'s current stream; errors raise."""
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return call(fn, index, *args)
    try:
        err = _local.err
    except AttributeError:
        err = _local.err = N.errbuf()
    code = fn(*args, _raw.get(index), err, 4096)
    if code:
        N.raise_for(code, err)


def once(backward):
    """An autograd function's backward(ctx, *gradients) that cannot be differentiated again. Asked for a graph of the
    gradients (create_graph=True), it is torch's once_differentiable, which raises if that graph is used; else it runs as
    it is, without that wrapper's 10 us."""
    careful = once_differentiable(backward)

    def either(ctx, *gradients):
        return careful(ctx, *gradients) if torch.is_grad_enabled() else backward(ctx, *gradients)
    return either


def ptr(t):
    return None if t is None else t.data_ptr()


def rows(t):
    """`t` with neighbouring elements along its last dimension: itself, or a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()

"""What the operators' Python side shares: checks of tensors, and calls of the library on the current stream."""
import torch

from .. import _native as N

DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}


def need(ok, message):
    if not ok:
        raise ValueError(message)


def on_gpu(name, *tensors):
    """The index of the GPU that all tensors (None: left out) are on."""
    index = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: tensors expected, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"{name} runs on the GPU only; got a tensor on {t.device}")
        i = t.get_device()
        if index is not None and i != index:
            raise ValueError(f"{name}: tensors on cuda:{index} and cuda:{i}")
        index = i
    return index


def call(fn, index, *args):
    """fn(*args, stream, err, errcap) of the library on GPU `index`'s current stream; errors raise."""
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return call(fn, index, *args)
    err = N.errbuf()
    code = getattr(N.lib(), fn)(*args, torch.cuda.current_stream(index).cuda_stream, err, len(err))
    if code:
        N.raise_for(code, err)


def ptr(t):
    return None if t is None else t.data_ptr()


def rows(t):
    """`t` with neighbouring elements along its last dimension: itself, or a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()

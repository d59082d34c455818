"""The norm over many gradient tensors, and clipping to it (panvram_amd/csrc/pv_clip.hip)."""
from array import array
from operator import attrgetter, eq

import torch

from .. import _native as N
from ._call import DTYPES, call, need, on_gpu


def _dense(t):
    """Whether t's elements fill one run of memory, in whatever order of its dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


_ptr, _numel, _whole, _gpu = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.get_device
_dtype, _shape = attrgetter("dtype"), attrgetter("shape")


def _checked(name, grads):
    """The GPU that all of `grads` are on; their types are ones that the kernels take. (Many tensors: one pass of a C-level
    map for each thing that is asked, not a loop.)"""
    if not all(issubclass(c, torch.Tensor) for c in set(map(type, grads))):
        raise TypeError(f"{name}: tensors expected")
    where = set(map(_gpu, grads))
    if len(where) != 1 or -1 in where:
        on_gpu(name, *grads)
    need(set(map(_dtype, grads)) <= DTYPES.keys(), f"{name}: gradients are float32, bfloat16 or float16")
    return where.pop()


def _run(index, grads, max_norm, out):
    """grads, out: each one run of memory, each pair's elements in the same order."""
    n = len(grads)
    sizes = array("q", map(_numel, grads))
    types = array("i", map(DTYPES.__getitem__, map(_dtype, grads)))
    src = array("Q", map(_ptr, grads))
    dst = array("Q", map(_ptr, out)) if out is not None else None
    at = [a.buffer_info()[0] if a is not None else None for a in (src, dst, sizes, types)]
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    work = torch.empty(N.lib().pv_gradient_norm_work_bytes(at[2], at[3], n), dtype=torch.uint8, device=norm.device)
    call("pv_gradient_norm_hip", index, *at, n, max_norm, norm.data_ptr(), work.data_ptr(), work.numel())
    return norm


@torch.no_grad()
def gradient_norm(grads):
    """sqrt of the sum of all squares of all tensors in `grads` (on one GPU), as a float32 tensor of no dimensions. A NaN
    or an infinity anywhere shows in it; squares are summed in 64 bits."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    index = _checked("gradient_norm", grads)
    if not all(map(_whole, grads)):
        grads = [g if _dense(g) else g.contiguous() for g in grads]
    return _run(index, grads, 0.0, None)


@torch.no_grad()
def clip_gradients(grads, max_norm, out=None):
    """Scales the tensors in `grads` (float32, bfloat16, float16, mixed as they come, on one GPU) by
    min(1, max_norm / (norm + 1e-6)), in place or into the tensors of `out` (alike, for instance views of one flat buffer;
    each one grads' own tensor or apart from all of them), and returns the norm before, as gradient_norm does. Nothing is
    read back: the factor is made and used on the GPU. If the norm is not finite, neither are the scaled gradients."""
    grads = list(grads)
    max_norm = float(max_norm)
    need(max_norm >= 0, f"clip_gradients: max_norm is not negative, got {max_norm}")
    out = None if out is None else list(out)
    need(out is None or len(out) == len(grads), f"clip_gradients: {len(grads)} gradients and {len(out or ())} tensors in out")
    if not grads:
        return torch.zeros(())
    index = _checked("clip_gradients", grads)
    if out is not None:
        need(_checked("clip_gradients", out) == index, "clip_gradients: grads and out on one GPU")
        if not all(map(eq, map(_shape, grads), map(_shape, out))) or not all(map(eq, map(_dtype, grads), map(_dtype, out))):
            i = next(i for i, (g, o) in enumerate(zip(grads, out)) if g.shape != o.shape or g.dtype != o.dtype)
            raise ValueError(f"clip_gradients: out[{i}] is {out[i].dtype} {list(out[i].shape)}, its gradient {grads[i].dtype} {list(grads[i].shape)}")
    back = []           # (tensor, what its values are made in) where memory is not one run, or in another order
    if not all(map(_whole, grads)) or (out is not None and not all(map(_whole, out))):
        to = grads if out is None else out
        grads, out = list(grads), list(to)
        for i, (g, o) in enumerate(zip(grads, to)):
            if g.stride() != o.stride() or not _dense(g):
                grads[i] = g.contiguous()
                if o.is_contiguous():
                    continue
                out[i] = torch.empty_like(grads[i])
                back.append((o, out[i]))
    norm = _run(index, grads, max_norm, grads if out is None else out)
    for o, made in back:
        o.copy_(made)
    return norm

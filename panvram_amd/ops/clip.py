"""The norm over many gradient tensors, and clipping to it (panvram_amd/csrc/pv_clip.hip)."""
import ctypes
import math

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


def _run(name, grads, max_norm, out):
    index = on_gpu(name, *grads)
    for g in grads:
        need(g.dtype in DTYPES, f"{name}: gradients are float32, bfloat16 or float16, got {g.dtype}")
    n = len(grads)
    sizes = (ctypes.c_int64 * n)(*[g.numel() for g in grads])
    types = (ctypes.c_int32 * n)(*[DTYPES[g.dtype] for g in grads])
    src = (ctypes.c_void_p * n)(*[g.data_ptr() for g in grads])
    dst = (ctypes.c_void_p * n)(*[o.data_ptr() for o in out]) if out is not None else None
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    work = torch.empty(N.lib().pv_gradient_norm_work_bytes(sizes, n), dtype=torch.uint8, device=norm.device)
    call("pv_gradient_norm_hip", index, src, dst, sizes, types, n, max_norm, norm.data_ptr(), work.data_ptr(), work.numel())
    return norm


@torch.no_grad()
def gradient_norm(grads):
    """sqrt of the sum of all squares of all tensors in `grads` (on one GPU), as a float32 tensor of no dimensions. A NaN
    or an infinity anywhere shows in it; squares are summed in 64 bits."""
    grads = [g if _dense(g) else g.contiguous() for g in grads]
    return _run("gradient_norm", grads, 0.0, None) if grads else torch.zeros(())


@torch.no_grad()
def clip_gradients(grads, max_norm, out=None):
    """Scales the tensors in `grads` (float32, bfloat16, float16, mixed as they come, on one GPU) by
    min(1, max_norm / (norm + 1e-6)), in place or into the tensors of `out` (alike, for instance views of one flat buffer;
    each one grads' own tensor or apart from all of them), and returns the norm before, as gradient_norm does. Nothing is
    read back: the factor is made and used on the GPU. If the norm is not finite, neither are the scaled gradients."""
    grads = list(grads)
    max_norm = float(max_norm)
    need(max_norm >= 0 and not math.isnan(max_norm), f"clip_gradients: max_norm is not negative, got {max_norm}")
    back = []
    if out is None:
        work = [g if _dense(g) else g.contiguous() for g in grads]
        back = [(g, w) for g, w in zip(grads, work) if g is not w]
        grads, out = work, work
    else:
        out = list(out)
        need(len(out) == len(grads), f"clip_gradients: {len(grads)} gradients and {len(out)} tensors in out")
        if grads:
            on_gpu("clip_gradients", *grads, *out)
        for i, (g, o) in enumerate(zip(grads, out)):
            need(o.dtype == g.dtype and o.shape == g.shape, f"clip_gradients: out[{i}] is {o.dtype} {list(o.shape)}, its gradient {g.dtype} {list(g.shape)}")
            if g.stride() != o.stride() or not _dense(g):
                grads[i] = g = g.contiguous()
                if not o.is_contiguous():
                    out[i] = torch.empty_like(g)
                    back.append((o, out[i]))
    if not grads:
        return torch.zeros(())
    norm = _run("clip_gradients", grads, max_norm, out)
    for to, made in back:
        to.copy_(made)
    return norm

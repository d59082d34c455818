"""The norm over many gradient tensors, and clipping to it (panvram_amd/csrc/pv_clip.hip)."""
from array import array
from operator import attrgetter

import torch

from .. import _native as N
from ._call import DTYPES, call, no_tangents, on_gpu


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
_dtype = attrgetter("dtype")
_written = torch.autograd.graph.increment_version        # autograd does not see the kernels' writes by itself


class _List:
    """Many tensors as the library takes them: addresses, sizes, types. (One pass of a C-level map for each thing that is
    asked, not a loop: 150 tensors cost 40 us.)"""

    def __init__(self, name, tensors):
        self.tensors, self.name = tensors, name
        if not all(issubclass(c, torch.Tensor) for c in set(map(type, tensors))):
            raise TypeError(f"{name}: tensors expected")
        no_tangents(name, tensors)
        where = set(map(_gpu, tensors))
        if len(where) != 1 or -1 in where:
            on_gpu(name, *tensors)
        self.index = where.pop()
        self.dtypes = list(map(_dtype, tensors))
        kinds = set(self.dtypes)
        if not kinds <= DTYPES.keys():
            raise ValueError(f"{name}: gradients are float32, bfloat16 or float16, got {[k for k in kinds if k not in DTYPES]}")
        self.types = array("i", [DTYPES[kinds.pop()]]) * len(tensors) if len(kinds) == 1 else array("i", map(DTYPES.__getitem__, self.dtypes))
        self.sizes = array("q", map(_numel, tensors))
        self.whole = all(map(_whole, tensors))
        self.made = []                     # copies, kept until the call is made

    def replace(self, i, t):
        if not self.made:
            self.tensors = list(self.tensors)
        self.made.append(t)
        self.tensors[i] = t

    def pointers(self):
        return array("Q", map(_ptr, self.tensors))


def _at(a):
    return a.buffer_info()[0]


def _norm(g, src):
    """The norm of g's tensors, which are at the addresses src"""
    norm = torch.empty((), dtype=torch.float32, device=g.tensors[0].device)
    L, n = N.lib(), len(g.tensors)
    size = L.pv_gradient_norm_work_bytes(_at(g.sizes), _at(g.types), n)
    work = torch.empty(size, dtype=torch.uint8, device=norm.device)
    call(L.pv_gradient_norm_hip, g.index, _at(src), _at(g.sizes), _at(g.types), n, norm.data_ptr(), work.data_ptr(), size)
    return norm


@torch.no_grad()
def gradient_norm(grads):
    """sqrt of the sum of all squares of all tensors in `grads` (on one GPU), as a float32 tensor of no dimensions. A NaN
    or an infinity anywhere shows in it; squares are summed in 64 bits."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    g = _List("gradient_norm", grads)
    if not g.whole:
        for i, t in enumerate(grads):
            if not _dense(t):
                g.replace(i, t.contiguous())
    return _norm(g, g.pointers())


@torch.no_grad()
def clip_gradients(grads, max_norm, out=None):
    """Scales the tensors in `grads` (float32, bfloat16, float16, mixed as they come, on one GPU) by
    min(1, max_norm / (norm + 1e-6)), in place or into the tensors of `out`, and returns the norm before, as gradient_norm
    does. out: for each gradient a tensor of its type and size, for instance views of one flat buffer; the gradient itself,
    or memory apart from all of them; no memory twice. Nothing is read back: the factor is made and used on the GPU. A norm
    of NaN makes NaN of all elements. An infinite one, of an infinite element or of a sum whose root float32 does not hold,
    makes a factor of 0: NaN of infinite elements, 0 of finite ones. A loop that is to skip such steps asks the norm."""
    grads = list(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_gradients: max_norm is not negative, got {max_norm}")
    out = None if out is None else list(out)
    if out is not None and len(out) != len(grads):
        raise ValueError(f"clip_gradients: {len(grads)} gradients and {len(out)} tensors in out")
    if not grads:
        return torch.zeros(())
    g = _List("clip_gradients", grads)
    o = g if out is None else _List("clip_gradients", out)
    if o is not g and (o.index != g.index or o.dtypes != g.dtypes or o.sizes != g.sizes):
        for i, (a, b) in enumerate(zip(grads, out)):
            if a.dtype != b.dtype or a.numel() != b.numel() or a.device != b.device:
                raise ValueError(f"clip_gradients: out[{i}] is {b.dtype} {list(b.shape)} on {b.device}, its gradient {a.dtype} {list(a.shape)} on {a.device}")
    back = []           # (tensor, what its values are made in) where memory is not one run, or in another order
    if not (g.whole and o.whole):
        to = grads if out is None else out
        if o is g:
            o = _List("clip_gradients", grads)
        for i, (a, b) in enumerate(zip(grads, to)):
            if (a.is_contiguous() and b.is_contiguous()) or (a.stride() == b.stride() and a.shape == b.shape and _dense(a)):
                continue
            if a.shape != b.shape:
                raise ValueError(f"clip_gradients: out[{i}] is {list(b.shape)}, its gradient {list(a.shape)}, and one of them is not contiguous")
            if not a.is_contiguous():
                g.replace(i, a.contiguous())
            if not b.is_contiguous():
                o.replace(i, torch.empty_like(a, memory_format=torch.contiguous_format))
                back.append((b, o.made[-1]))
    src = g.pointers()
    dst = src if o is g else o.pointers()
    if len(set(dst)) < len(dst):
        to = [p for p in dst if p]                  # (empty tensors have no address)
        if len(set(to)) < len(to):
            raise ValueError("clip_gradients: the same memory twice among the tensors to write")
    norm = _norm(g, src)
    call(N.lib().pv_scale_gradients_hip, g.index, _at(src), _at(dst), _at(g.sizes), _at(g.types), len(grads), max_norm, norm.data_ptr())
    _written(grads if out is None else out)
    for b, made in back:
        b.copy_(made)
    return norm

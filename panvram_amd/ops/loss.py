"""The head and loss over a small alphabet (panvram_amd/csrc/pv_loss.hip)."""
import torch

from .. import _native as N
from ._call import DTYPES, call, on_gpu, once, ptr, rows


def _run(hidden, weight, tokens, ignore, want_each, want_loss, grads, scale=None, factor=None):
    B, T, D = hidden.shape
    V = weight.shape[0]
    dev = hidden.device
    each = torch.empty((B, T), dtype=torch.float32, device=dev) if want_each else None
    loss = torch.empty((), dtype=torch.float32, device=dev) if want_loss else None
    d_hidden = torch.empty((B, T, D), dtype=hidden.dtype, device=dev) if grads else None
    d_weight = torch.empty((V, D), dtype=weight.dtype, device=dev) if grads else None
    L = N.lib()
    size = L.pv_next_base_loss_work_bytes(B, T, D, V, grads)
    work = torch.empty(size, dtype=torch.uint8, device=dev)
    hb, ht, _ = hidden.stride()
    call(L.pv_next_base_loss_hip, hidden.get_device(), hidden.data_ptr(), weight.data_ptr(), tokens.data_ptr(), B, T, D, V, hb, ht, tokens.stride(0), ignore,
         DTYPES[hidden.dtype], DTYPES[weight.dtype], tokens.element_size(), ptr(scale), ptr(factor), ptr(each), ptr(loss), ptr(d_hidden), ptr(d_weight),
         work.data_ptr(), size)
    return each, loss, d_hidden, d_weight


class _NextBaseLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, tokens, ignore, mean):
        each, loss, _, _ = _run(hidden, weight, tokens, ignore, not mean, mean, False)
        ctx.save_for_backward(hidden, weight, tokens)
        ctx.ignore, ctx.mean = ignore, mean
        return loss if mean else each

    @staticmethod
    @once
    def backward(ctx, d):
        hidden, weight, tokens = ctx.saved_tensors
        d = d.contiguous()
        _, _, d_hidden, d_weight = _run(hidden, weight, tokens, ctx.ignore, False, False, True, scale=d if ctx.mean else None, factor=None if ctx.mean else d)
        return d_hidden, d_weight, None, None, None


def _checked(name, hidden, weight, tokens, ignore):
    on_gpu(name, hidden, weight, tokens)
    if hidden.dim() != 3 or hidden.dtype not in DTYPES or hidden.numel() == 0:
        raise ValueError(f"{name}: hidden is [B, T, D] in float32, bfloat16 or float16 and not empty, got {hidden.dtype} {list(hidden.shape)}")
    B, T, D = hidden.shape
    if weight.dim() != 2 or weight.shape[1] != D or not 1 <= weight.shape[0] <= 16:
        raise ValueError(f"{name}: weight is [V, {D}] with 1 to 16 ids, got {list(weight.shape)}")
    if weight.dtype != hidden.dtype and weight.dtype != torch.float32:
        raise ValueError(f"{name}: weight is in hidden's type or float32, got {weight.dtype}")
    if tokens.shape != (B, T) or tokens.dtype not in (torch.uint8, torch.int64):
        raise ValueError(f"{name}: tokens are uint8 or int64 {[B, T]}, got {tokens.dtype} {list(tokens.shape)}")
    return rows(hidden), weight.contiguous(), rows(tokens), -1 if ignore is None else int(ignore)


def next_base_loss(hidden, weight, tokens, ignore=4, reduction="mean"):
    """The cross-entropy of each next token under softmax(hidden @ weight.T), the head's logits never stored.

    hidden: [B, T, D], float32, bfloat16 or float16. weight: [V, D] with V up to 16, in hidden's type or float32. tokens:
    uint8 or int64 [B, T] as Cohort.sample returns them; hidden[:, t] predicts tokens[:, t + 1]. Places whose next token is
    `ignore` (4: every byte other than A, C, G, T; None: no such id) or no id of [0, V) do not count, nor does the last of
    a row: windows packed in a row go in as rows of their own (a view where they are of one length), or else the last place of
    each predicts the next one's first token. reduction: "mean" over the places that count (0 where there are none), or
    "none": float32 [B, T] with 0 at places that do not count. Gradients flow to hidden and weight; what stands in hidden where nothing counts reaches neither."""
    hidden, weight, tokens, ignore = _checked("next_base_loss", hidden, weight, tokens, ignore)
    if reduction not in ("mean", "none"):
        raise ValueError(f'next_base_loss: reduction is "mean" or "none", got {reduction!r}')
    mean = reduction == "mean"
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _NextBaseLoss.apply(hidden, weight, tokens, ignore, mean)
    each, loss, _, _ = _run(hidden, weight, tokens, ignore, not mean, mean, False)
    return loss if mean else each


@torch.no_grad()
def next_base_loss_grad(hidden, weight, tokens, ignore=4, scale=None):
    """(loss, d_hidden, d_weight): next_base_loss's mean and its gradients, times `scale` (None, or a float32 tensor of one
    element on the GPU, as a loss scaler keeps it), from one pass over hidden - where autograd makes two, one for the loss
    and one for the gradients. `hidden.backward(d_hidden)` goes on from it."""
    hidden, weight, tokens, ignore = _checked("next_base_loss_grad", hidden, weight, tokens, ignore)
    if scale is not None:
        on_gpu("next_base_loss_grad", hidden, scale)
        if scale.dtype != torch.float32 or scale.numel() != 1:
            raise ValueError(f"next_base_loss_grad: scale is one float32, got {scale.dtype} {list(scale.shape)}")
    _, loss, d_hidden, d_weight = _run(hidden, weight, tokens, ignore, False, True, True, scale=scale)
    return loss, d_hidden, d_weight

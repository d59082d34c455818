"""The gated linear recurrence over sequences (panvram_amd/csrc/pv_scan.hip)."""
import torch

from .. import _native as N
from ._call import DTYPES, call, on_gpu, once, ptr, rows


def _steps(t):
    """(t, its batch and time strides) with neighbouring channels, and steps at most 64 MiB apart (the kernels' offsets
    within a chunk): itself, or a copy."""
    b, s, d = t.stride()
    if (d != 1 and t.shape[2] != 1) or s > 1 << 24:
        t = t.contiguous()
        b, s, _ = t.stride()
    return t, b, s


def _work(L, B, T, D, dev):
    n = L.pv_gated_scan_work_bytes(B, T, D)
    return (torch.empty(n, dtype=torch.uint8, device=dev) if n else None), n


def _forward(index, gate, value, state, reset, keep_carry):
    B, T, D = gate.shape
    dev, dtype = gate.device, gate.dtype
    gate, gb, gt = _steps(gate)
    value, vb, vt = _steps(value)
    out = torch.empty((B, T, D), dtype=dtype, device=dev)
    last = torch.empty((B, D), dtype=torch.float32, device=dev)
    L = N.lib()
    carry = torch.empty((B, L.pv_gated_scan_spans(T), D), dtype=torch.float32, device=dev) if keep_carry else None
    work, size = _work(L, B, T, D, dev)
    call(L.pv_gated_scan_hip, index, gate.data_ptr(), value.data_ptr(), ptr(state), ptr(reset), B, T, D, gb, gt, vb, vt, DTYPES[dtype], out.data_ptr(),
         last.data_ptr(), ptr(carry), ptr(work), size)
    return out, last, carry


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, value, state, reset):
        index = gate.get_device()
        out, last, carry = _forward(index, gate, value, state, reset, True)
        ctx.save_for_backward(gate, value, carry, reset)
        ctx.has_state = state is not None
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once
    def backward(ctx, d_out, d_last):
        gate, value, carry, reset = ctx.saved_tensors
        B, T, D = gate.shape
        dev, dtype, index = gate.device, gate.dtype, gate.get_device()
        d_gate = torch.empty((B, T, D), dtype=dtype, device=dev)
        d_value = torch.empty((B, T, D), dtype=dtype, device=dev)
        d_state = torch.empty((B, D), dtype=torch.float32, device=dev) if ctx.has_state else None
        d_out = torch.zeros((B, T, D), dtype=dtype, device=dev) if d_out is None else d_out
        gate, gb, gt = _steps(gate)
        value, vb, vt = _steps(value)
        d_out, ob, ot = _steps(d_out)
        d_last = None if d_last is None else d_last.contiguous()
        L = N.lib()
        work, size = _work(L, B, T, D, dev)
        call(L.pv_gated_scan_backward_hip, index, gate.data_ptr(), value.data_ptr(), carry.data_ptr(), ptr(reset), B, T, D, gb, gt, vb, vt, d_out.data_ptr(),
             ob, ot, ptr(d_last), DTYPES[dtype], d_gate.data_ptr(), d_value.data_ptr(), ptr(d_state), ptr(work), size)
        return d_gate, d_value, d_state, None


def gated_scan(gate, value, state=None, reset=None):
    """h[t] = (1 - z[t]) h[t-1] + z[t] value[t] with z = sigmoid(gate), for each of the [B, T, D] channels by itself.

    gate, value: [B, T, D], float32, bfloat16 or float16; halves of one projection (`gate, value = p.chunk(2, -1)`) are
    read where they are. state: float32 [B, D], the h before the first step (None: zero). reset: bool or uint8 [B, T];
    where it is set, the h of the step before is dropped, as at the first base of a window packed behind another.
    Returns (out [B, T, D] in gate's type, last float32 [B, D]); `last` is the next call's state, so generation calls it
    with T = 1. Gradients flow to gate, value and state, from out and from last."""
    index = on_gpu("gated_scan", gate, value, state, reset)
    if gate.dim() != 3 or gate.shape != value.shape:
        raise ValueError(f"gated_scan: gate and value are [B, T, D] alike, got {list(gate.shape)} and {list(value.shape)}")
    if gate.dtype not in DTYPES or gate.dtype != value.dtype:
        raise ValueError(f"gated_scan: gate and value are float32, bfloat16 or float16 alike, got {gate.dtype} and {value.dtype}")
    B, T, D = gate.shape
    grad = gate.requires_grad or value.requires_grad
    if state is not None:
        if state.dtype != torch.float32 or state.shape != (B, D):
            raise ValueError(f"gated_scan: state is float32 {[B, D]}, got {state.dtype} {list(state.shape)}")
        grad = grad or state.requires_grad
        state = state.contiguous()
    if reset is not None:
        if reset.dtype not in (torch.bool, torch.uint8) or reset.shape != (B, T):
            raise ValueError(f"gated_scan: reset is bool or uint8 {[B, T]}, got {reset.dtype} {list(reset.shape)}")
        reset = reset.contiguous()
    if T == 0:
        return gate * value, state.clone() if state is not None else torch.zeros(B, D, dtype=torch.float32, device=gate.device)
    if grad and torch.is_grad_enabled():
        return _GatedScan.apply(gate, value, state, reset)
    return _forward(index, gate, value, state, reset, False)[:2]

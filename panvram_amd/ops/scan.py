"""The gated linear recurrence over sequences (panvram_amd/csrc/pv_scan.hip)."""
import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from ._call import DTYPES, call, need, on_gpu, ptr, rows


def _steps(t):
    """`t` with neighbouring channels, and steps at most 64 MiB apart (the kernels' offsets within a chunk): itself, or a copy."""
    t = rows(t)
    return t if t.stride(1) * t.element_size() <= 1 << 26 else t.contiguous()


def _forward(gate, value, state, reset, keep_carry):
    B, T, D = gate.shape
    dev = gate.device
    out = torch.empty(B, T, D, dtype=gate.dtype, device=dev)
    last = torch.empty(B, D, dtype=torch.float32, device=dev)
    L = N.lib()
    carry = torch.empty(B, L.pv_gated_scan_chunks(T), D, dtype=torch.float32, device=dev) if keep_carry else None
    work = torch.empty(L.pv_gated_scan_work_bytes(B, T, D), dtype=torch.uint8, device=dev)
    call("pv_gated_scan_hip", gate.get_device(), gate.data_ptr(), value.data_ptr(), ptr(state), ptr(reset), B, T, D, gate.stride(0), gate.stride(1),
         value.stride(0), value.stride(1), DTYPES[gate.dtype], out.data_ptr(), last.data_ptr(), ptr(carry), work.data_ptr(), work.numel())
    return out, last, carry


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, value, state, reset):
        out, last, carry = _forward(gate, value, state, reset, True)
        ctx.save_for_backward(gate, value, carry, reset)
        ctx.has_state = state is not None
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_last):
        gate, value, carry, reset = ctx.saved_tensors
        B, T, D = gate.shape
        dev = gate.device
        d_out, d_last = _steps(d_out), d_last.contiguous()
        d_gate = torch.empty(B, T, D, dtype=gate.dtype, device=dev)
        d_value = torch.empty(B, T, D, dtype=gate.dtype, device=dev)
        d_state = torch.empty(B, D, dtype=torch.float32, device=dev) if ctx.has_state else None
        work = torch.empty(N.lib().pv_gated_scan_work_bytes(B, T, D), dtype=torch.uint8, device=dev)
        call("pv_gated_scan_backward_hip", gate.get_device(), gate.data_ptr(), value.data_ptr(), carry.data_ptr(), ptr(reset), B, T, D, gate.stride(0),
             gate.stride(1), value.stride(0), value.stride(1), d_out.data_ptr(), d_out.stride(0), d_out.stride(1), d_last.data_ptr(), DTYPES[gate.dtype],
             d_gate.data_ptr(), d_value.data_ptr(), ptr(d_state), work.data_ptr(), work.numel())
        return d_gate, d_value, d_state, None


def gated_scan(gate, value, state=None, reset=None):
    """h[t] = (1 - z[t]) h[t-1] + z[t] value[t] with z = sigmoid(gate), for each of the [B, T, D] channels by itself.

    gate, value: [B, T, D], float32, bfloat16 or float16; halves of one projection (`gate, value = p.chunk(2, -1)`) are
    read where they are. state: float32 [B, D], the h before the first step (None: zero). reset: bool or uint8 [B, T];
    where it is set, the h of the step before is dropped, as at the first base of a window packed behind another.
    Returns (out [B, T, D] in gate's type, last float32 [B, D]); `last` is the next call's state, so generation calls it
    with T = 1. Gradients flow to gate, value and state, from out and from last."""
    index = on_gpu("gated_scan", gate, value, state, reset)
    need(gate.dim() == 3 and gate.shape == value.shape, f"gated_scan: gate and value are [B, T, D] alike, got {list(gate.shape)} and {list(value.shape)}")
    need(gate.dtype in DTYPES and gate.dtype == value.dtype, f"gated_scan: gate and value are float32, bfloat16 or float16 alike, got {gate.dtype} and {value.dtype}")
    B, T, D = gate.shape
    if state is not None:
        need(state.dtype == torch.float32 and state.shape == (B, D), f"gated_scan: state is float32 {[B, D]}, got {state.dtype} {list(state.shape)}")
        state = state.contiguous()
    if reset is not None:
        need(reset.dtype in (torch.bool, torch.uint8) and reset.shape == (B, T), f"gated_scan: reset is bool or uint8 {[B, T]}, got {reset.dtype} {list(reset.shape)}")
        reset = reset.contiguous()
    if T == 0:
        return gate * value, state.clone() if state is not None else torch.zeros(B, D, dtype=torch.float32, device=gate.device)
    gate, value = _steps(gate), _steps(value)
    if torch.is_grad_enabled() and (gate.requires_grad or value.requires_grad or (state is not None and state.requires_grad)):
        return _GatedScan.apply(gate, value, state, reset)
    return _forward(gate, value, state, reset, False)[:2]

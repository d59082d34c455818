"""The gated delta rule over sequences (panvram_amd/csrc/pv_delta.hip)."""
import ctypes

import torch

from .. import _native as N
from ._call import DTYPES, call, on_gpu, once, ptr


_FORWARD, _BACKWARD = ctypes.c_int64 * 15, ctypes.c_int64 * 9         # strides of a sequence, a step and a head of each tensor


def _strided(t):
    """`t` with neighbouring elements in a head, and steps at most 2^22 elements apart: itself, or a copy; and its strides. (A single
    step has no stride, whatever the tensor says of it and keeps saying when it is made contiguous.)"""
    s = t.stride()
    if s[1] > 1 << 22 or (len(s) == 4 and s[3] != 1 and t.shape[3] != 1):
        if t.shape[1] != 1 or (len(s) == 4 and s[3] != 1):
            t = t.contiguous()
            s = t.stride()
        s = (s[0], s[1] if t.shape[1] != 1 else 0, s[2])
    return t, *s[:3]


def _forward(index, query, key, value, gate, write, state, reset, eps, keep):
    """out, last, and for the backward pass the states before the chunks and the chunks' records"""
    B, T, H, K = query.shape
    G, V = value.shape[2:]
    dev, dtype = query.device, query.dtype
    query, *qs = _strided(query)
    key, *ks = _strided(key)
    value, *vs = _strided(value)
    gate, *gs = _strided(gate)
    write, *ws = _strided(write)
    out = torch.empty((B, T, G, V), dtype=dtype, device=dev)
    last = torch.empty((B, G, K, V), dtype=torch.float32, device=dev)
    L, code = N.lib(), DTYPES[dtype]
    kept = torch.empty(L.pv_gated_delta_kept_bytes(B, T, G, K, V, code), dtype=torch.uint8, device=dev) if keep else None
    size = L.pv_gated_delta_work_bytes(B, T, H, G, K, V, code, int(keep))
    work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    call(L.pv_gated_delta_hip, index, query.data_ptr(), key.data_ptr(), value.data_ptr(), gate.data_ptr(), write.data_ptr(), ptr(state), ptr(reset), B, T, H, G, K, V,
         _FORWARD(*qs, *ks, *vs, *gs, *ws), eps, code, out.data_ptr(), last.data_ptr(), ptr(kept), ptr(work), size)
    return out, last, kept, work


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, gate, write, state, reset, eps):
        out, last, kept, records = _forward(query.get_device(), query, key, value, gate, write, state, reset, eps, True)
        ctx.save_for_backward(gate, write, kept, records)          # (queries and keys are among the records)
        ctx.shape, ctx.has_state = (*query.shape, *value.shape[2:]), state is not None
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once
    def backward(ctx, d_out, d_last):
        gate, write, kept, records = ctx.saved_tensors
        B, T, H, K, G, V = ctx.shape
        dev, dtype = gate.device, gate.dtype
        d_out, *os = _strided(torch.zeros((B, T, G, V), dtype=dtype, device=dev) if d_out is None else d_out)
        d_last = None if d_last is None else d_last.contiguous()
        d_query, d_key, d_value, d_gate, d_write = (torch.empty(s, dtype=dtype, device=dev) for s in ((B, T, H, K), (B, T, H, K), (B, T, G, V), (B, T, G), (B, T, G)))
        d_state = torch.empty((B, G, K, V), dtype=torch.float32, device=dev) if ctx.has_state else None
        L, code = N.lib(), DTYPES[dtype]
        size = L.pv_gated_delta_backward_work_bytes(B, T, G, K, V, code)
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        gate, *gs = _strided(gate)
        write, *ws = _strided(write)
        call(L.pv_gated_delta_backward_hip, gate.get_device(), gate.data_ptr(), write.data_ptr(), d_out.data_ptr(), ptr(d_last), B, T, H, G, K, V,
             _BACKWARD(*gs, *ws, *os), code, kept.data_ptr(), records.data_ptr(), d_query.data_ptr(), d_key.data_ptr(), d_value.data_ptr(), d_gate.data_ptr(),
             d_write.data_ptr(), ptr(d_state), work.data_ptr(), size)
        return d_query, d_key, d_value, d_gate, d_write, d_state, None, None


def gated_delta(query, key, value, gate, write, state=None, reset=None, eps=1e-6):
    """The gated delta rule: each value head has a matrix S as its state, and with keep = 1 - sigmoid(gate),
    rate = sigmoid(write), and query and key divided by sqrt(the sum of their squares + eps),

        S[t] = keep[t] S[t-1] + key[t] u[t]^T,  u[t] = rate[t] (value[t] - keep[t] S[t-1]^T key[t]),  out[t] = S[t]^T query[t]:

    what S holds for the direction of key[t] is replaced by value[t], in the share that rate says.

    query, key: [B, T, H, K] with K up to 128; value: [B, T, G, V]; gate, write: [B, T, G]; float32, bfloat16 or float16, alike. G is
    a multiple of H: value head g goes with query and key head g // (G // H). Parts of one projection are read where they are.
    state: float32 [B, G, K, V], the S before the first step (None: zero). reset: bool or uint8 [B, T]; where it is set, the S of the
    step before is dropped, as at the first base of a window packed behind another. Returns (out [B, T, G, V] in query's type,
    last float32 [B, G, K, V]); `last` is the next call's state, so generation calls it with T = 1. Gradients flow to query, key,
    value, gate, write and state, from out and from last.

    For its gradients a call keeps, beside gate and write, some 2.9 KB a step of each head of 128 x 128 in 16 bits, 3.3 in float32:
    states and updates of each chunk, and what the chunks' steps do to each other. Queries, keys and values need not be kept.

    B G ceil(T / 64) and B G ceil(V / 32), the chunks and the columns' groups of a call, are below 2^23, H K and G V at most 2^22.

    Calls of up to 8 steps without gradients go step by step, others in chunks of 64 by matrix products, long ones of few heads in
    pieces: the same up to roundings, and equal from run to run, not from one of these ways to another. A NaN or an infinity among a
    step's inputs reaches what it reaches in the formulas above, its own output and those after it up to the next reset, and is NaN there where
    steps go in chunks; gradients that it reaches are NaN, and so may be those of gate at steps before it in its chunk, back to a reset. Queries
    and keys have squares whose sum is a float32."""
    index = on_gpu("gated_delta", query, key, value, gate, write, state, reset)
    if query.dim() != 4 or query.shape != key.shape:
        raise ValueError(f"gated_delta: query and key are [B, T, H, K] alike, got {list(query.shape)} and {list(key.shape)}")
    dtype = query.dtype
    if dtype not in DTYPES or not (dtype == key.dtype == value.dtype == gate.dtype == write.dtype):
        raise ValueError(f"gated_delta: query, key, value, gate and write are float32, bfloat16 or float16 alike, got {[str(t.dtype) for t in (query, key, value, gate, write)]}")
    B, T, H, K = query.shape
    if value.dim() != 4 or value.shape[:2] != (B, T) or H < 1 or value.shape[2] < 1 or value.shape[2] % H:
        raise ValueError(f"gated_delta: value is [{B}, {T}, G, V] with G a multiple of {H}, got {list(value.shape)}")
    G, V = value.shape[2:]
    if not 1 <= K <= 128 or not 1 <= V <= 1 << 16:
        raise ValueError(f"gated_delta: keys have 1 to 128 elements and values 1 to 65,536, got {K} and {V}")
    if G * V > 1 << 22 or H * K > 1 << 22:
        raise ValueError(f"gated_delta: a step's values, and its keys, are 2^22 at most, got {G} x {V} and {H} x {K}")
    if gate.shape != (B, T, G) or write.shape != (B, T, G):
        raise ValueError(f"gated_delta: gate and write are {[B, T, G]}, got {list(gate.shape)} and {list(write.shape)}")
    if not eps >= 0:
        raise ValueError(f"gated_delta: eps is not negative, got {eps}")
    if state is not None:
        if state.dtype != torch.float32 or state.shape != (B, G, K, V):
            raise ValueError(f"gated_delta: state is float32 {[B, G, K, V]}, got {state.dtype} {list(state.shape)}")
        state = state.contiguous()
    if reset is not None:
        if reset.dtype not in (torch.bool, torch.uint8) or reset.shape != (B, T):
            raise ValueError(f"gated_delta: reset is bool or uint8 {[B, T]}, got {reset.dtype} {list(reset.shape)}")
        reset = reset.contiguous()
    if B == 0 or T == 0:
        return value * 1, state.clone() if state is not None else torch.zeros(B, G, K, V, dtype=torch.float32, device=query.device)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (query, key, value, gate, write, state)):
        return _GatedDelta.apply(query, key, value, gate, write, state, reset, eps)
    return _forward(index, query, key, value, gate, write, state, reset, eps, False)[:2]

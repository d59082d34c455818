"""The gated scan's forms for tensors that the caches do not hold, for a single step of more channels than 32-bit byte offsets
reach, and what it leaves alone: memory behind a sequence's end. Run with -m gpu."""
import ctypes

import pytest
import torch

from panvram_amd import _native as N
from tests.test_gpu_scan import check, cpu, make
from tests import ops_plain as P

pytestmark = pytest.mark.gpu
KIND = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}


@pytest.mark.parametrize("dtype,B,D", [(torch.float32, 33, 1024), (torch.bfloat16, 64, 1024), (torch.float16, 132, 512)])
@pytest.mark.parametrize("reset", [0.0, 0.01])
def test_larger_than_the_caches_hold(dtype, B, D, reset):
    """64 MiB a tensor and more, rows of whole 128-byte lines: three chunks of the forward pass, five of the backward one."""
    assert B * 530 * D * torch.empty(0, dtype=dtype).element_size() >= 64 << 20
    check(*make(B, 530, D, dtype, seed=D + B, reset=reset))


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, (1 << 30) + 1), (torch.float32, (1 << 30) + 1), (torch.bfloat16, (1 << 30) + 128)])
def test_a_step_of_many_channels(dtype, D):
    """One step whose row is over 2 or 4 GiB: each channel's own value in its place (compared at both ends and in between)."""
    from panvram_amd import ops
    gate = torch.empty(1, 1, D, dtype=dtype, device="cuda")
    gate.view(-1)[:] = 100.0                         # z = 1: out = value
    value = torch.empty(1, 1, D, dtype=dtype, device="cuda")
    flat = value.view(-1)
    for at in range(0, D, 1 << 26):
        n = min(1 << 26, D - at)
        flat[at:at + n] = ((torch.arange(n, device="cuda") + at // 7) % 251).to(dtype)
    out, last = ops.gated_scan(gate, value)
    for at in range(0, D, 1 << 26):
        n = min(1 << 26, D - at)
        assert torch.equal(out.view(-1)[at:at + n], flat[at:at + n]) and torch.equal(last.view(-1)[at:at + n], flat[at:at + n].float())


@pytest.mark.parametrize("dtype", list(KIND))
@pytest.mark.parametrize("T,D", [(1, 130), (3, 64), (5, 129), (33, 66), (257, 130), (523, 7)])
def test_nothing_behind_the_end(T, D, dtype):
    """Inputs and outputs in the middle of larger buffers: what stands behind a sequence's last step (NaN) is not read into any
    result, and what stands around the outputs is as it was."""
    gate, value, state, _, d_out, d_last = make(2, T, D, dtype, seed=T + D)
    plain = P.scan(*cpu(gate, value, state), None, *cpu(d_out, d_last))
    pad = 300 * D            # more than a chunk of steps

    def inside(t):           # a batch's steps, then `pad` elements of NaN, and as many before
        room = torch.full((2, T * D + 2 * pad), float("nan"), dtype=t.dtype, device="cuda")
        room[:, pad:pad + T * D] = t.reshape(2, T * D)
        return room, room.data_ptr() + pad * room.element_size()

    def outside(dtype, count):
        room = torch.full((count + 2 * pad,), -77.0, dtype=dtype, device="cuda")
        return room, room.data_ptr() + pad * room.element_size()

    def held(room):
        return bool((room[:pad] == -77.0).all() and (room[-pad:] == -77.0).all())

    L, err, st = N.lib(), N.errbuf(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    rows = T * D + 2 * pad
    g, gp = inside(gate)
    v, vp = inside(value)
    d, dp = inside(d_out)
    out, op = outside(dtype, 2 * T * D)
    last, lp = outside(torch.float32, 2 * D)
    carry, cp = outside(torch.float32, 2 * D * L.pv_gated_scan_spans(T))
    size = L.pv_gated_scan_work_bytes(2, T, D)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    code = L.pv_gated_scan_hip(gp, vp, state.data_ptr(), None, 2, T, D, rows, D, rows, D, KIND[dtype], op, lp, cp, work.data_ptr(), size, st, err, len(err))
    assert code == N.PV_OK, err.value
    assert held(out) and held(last) and held(carry)
    P.inside(out[pad:-pad].view(2, T, D), plain["out"][0], plain["out"][1] + P.rounded(plain["out"][0], dtype))
    P.inside(last[pad:-pad].view(2, D), plain["last"][0], plain["last"][1] + P.rounded(plain["last"][0], torch.float32))
    dg, dgp = outside(dtype, 2 * T * D)
    dv, dvp = outside(dtype, 2 * T * D)
    ds, dsp = outside(torch.float32, 2 * D)
    code = L.pv_gated_scan_backward_hip(gp, vp, cp, None, 2, T, D, rows, D, rows, D, dp, rows, D, d_last.data_ptr(), KIND[dtype], dgp, dvp, dsp, work.data_ptr(),
                                        size, st, err, len(err))
    assert code == N.PV_OK, err.value
    assert held(dg) and held(dv) and held(ds)
    for room, name, shape, kind in ((dg, "d_gate", (2, T, D), dtype), (dv, "d_value", (2, T, D), dtype), (ds, "d_state", (2, D), torch.float32)):
        P.inside(room[pad:-pad].view(shape), plain[name][0], plain[name][1] + P.rounded(plain[name][0], kind))

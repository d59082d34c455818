"""Sizes past what one launch takes (below 2^32 work items in a grid): refused by the C entries before any launch, or worked on
in several."""
import ctypes

import pytest
import torch

from panvram_amd import _native as N
from tests.test_ops_refusals import FAKE, refused


def test_scan_workgroups():
    """512 work items for a chunk of a sequence's channels: 2^23 of them are too many."""
    def scan(B, T, D, dtype=N.F32):
        return refused("pv_gated_scan_hip", FAKE, FAKE, None, None, B, T, D, D * T, D, D * T, D, dtype, FAKE, FAKE, None, FAKE, 1 << 50)

    def back(B, T, D, dtype=N.F32):
        return refused("pv_gated_scan_backward_hip", FAKE, FAKE, FAKE, None, B, T, D, D * T, D, D * T, D, FAKE, D * T, D, None, dtype, FAKE, FAKE, None, FAKE, 1 << 50)
    for fn in (scan, back):
        assert "too many chunks" in fn(1 << 23, 33, 1)
        assert "too many chunks" in fn(1 << 23, 33, 128, N.BF16)
        assert "too many chunks" in fn(1, (1 << 31) - 1, 1)
        assert "too many chunks" in fn(1 << 26, 1, 1)


def test_loss_columns():
    def loss(D):
        return refused("pv_next_base_loss_hip", FAKE, FAKE, FAKE, 1, 2, D, 4, 2 * D, D, 2, 4, N.F32, N.F32, 1, None, None, None, FAKE, None, None, FAKE, 1 << 50)
    assert "shape" in loss((1 << 23) + 1)


def test_clip_sizes():
    vp, i64, i32 = ctypes.c_void_p * 1, ctypes.c_int64 * 1, ctypes.c_int32 * 1
    for size, dtype in (((1 << 36), N.F32), ((1 << 37), N.BF16)):
        assert "size" in refused("pv_gradient_norm_hip", vp(FAKE), i64(size), i32(dtype), 1, FAKE, FAKE, 1 << 40)
        assert "size" in refused("pv_scale_gradients_hip", vp(FAKE), vp(FAKE), i64(size), i32(dtype), 1, 1.0, FAKE)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [(1 << 29) + 7, (1 << 29)])
def test_norm_of_many_rows(count):
    """More rows than one launch's work items: in the stream's type, in 8 bits, and backwards."""
    from panvram_amd import ops
    x = torch.full((count, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    x[-1] = -3.0
    x[1 << 28] = -5.0
    w = torch.tensor([1.5], device="cuda")

    def right(y, low):
        assert float(y[-1]) == -low and float(y[1 << 28]) == -low
        y[-1] = y[1 << 28] = low
        assert bool((y == low).all())

    right(ops.add_rms_norm(x, None, w, eps=0.0)[0], 1.5)
    q, scale, _ = ops.add_rms_norm_8bit(x, None, w, eps=0.0, dtype=torch.int8)
    right(q, 127)
    assert float((scale - 1.5 / 127).abs().max()) <= 1e-8
    del q, scale
    v = w.clone().requires_grad_()
    y, _ = ops.add_rms_norm(x, None, v, eps=0.0)
    d_y = torch.zeros_like(y)
    d_y[-1] = d_y[0] = d_y[1 << 28] = 1.0
    (d,) = torch.autograd.grad(y, (v,), d_y)
    assert abs(float(d) - (1 - 1 - 1)) <= 1e-5


@pytest.mark.gpu
def test_norm_of_one_long_row():
    """A row of over 2^28 elements and its weight's gradient."""
    from panvram_amd import ops
    D = (1 << 28) + 65
    x = torch.full((1, D), 2.0, device="cuda")
    x[0, -1] = -2.0
    w = torch.full((D,), 1.5, device="cuda").requires_grad_()
    y, _ = ops.add_rms_norm(x.expand(3, D), None, w, eps=0.0)
    assert float((y[1].abs() - 1.5).abs().max()) <= 1e-5 and float(y[2, -1]) < 0
    (d,) = torch.autograd.grad(y, (w,), torch.ones(1, 1, device="cuda").expand(3, D))
    assert float((d[:-1] - 3).abs().max()) <= 1e-4 and abs(float(d[-1]) + 3) <= 1e-4

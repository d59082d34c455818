"""What the operators refuse: the C entries' checks (before any launch, so without a GPU) and the Python functions'."""
import ctypes

import pytest
import torch

from panvram_amd import _native as N
from panvram_amd import ops

FAKE = 0x1000          # not null, never followed: every call here is refused first


def refused(fn, *args):
    err = N.errbuf()
    code = getattr(N.lib(), fn)(*args, None, err, len(err))
    assert code == N.PV_EARG, (fn, code)
    return err.value.decode()


def scan(B=1, T=8, D=4, dtype=N.F32, gate=FAKE, out=FAKE, work=FAKE, work_bytes=1 << 20):
    return refused("pv_gated_scan_hip", gate, FAKE, None, None, B, T, D, D * T, D, D * T, D, dtype, out, FAKE, None, work, work_bytes)


def test_scan_entry():
    assert "dtype" in scan(dtype=7)
    assert "shape" in scan(B=-1)
    assert "shape" in scan(T=0)
    assert "work" in scan(T=5000, work_bytes=8)
    assert "stride" in refused("pv_gated_scan_hip", FAKE, FAKE, None, None, 1, 8, 4, 32, 1 << 25, 32, 4, N.F32, FAKE, FAKE, None, FAKE, 1 << 20)
    assert "null" in scan(gate=None)
    assert "null" in scan(out=None)
    m = refused("pv_gated_scan_backward_hip", FAKE, FAKE, None, None, 1, 8, 4, 32, 4, 32, 4, FAKE, 32, 4, None, N.F32, FAKE, FAKE, None, FAKE, 1 << 20)
    assert "null" in m


@pytest.mark.parametrize("call", [
    lambda t: ops.gated_scan(t, t), lambda t: ops.add_rms_norm(t, t, t[0, 0]), lambda t: ops.add_rms_norm_8bit(t, t, t[0, 0]),
    lambda t: ops.next_base_loss(t, t[0], t[:, :, 0]), lambda t: ops.clip_gradients([t], 1.0), lambda t: ops.gradient_norm([t])])
def test_no_cpu_tensors(call):
    with pytest.raises(RuntimeError, match="GPU only"):
        call(torch.zeros(2, 3, 4))


def test_not_tensors():
    with pytest.raises(TypeError):
        ops.gated_scan([1.0], [2.0])


@pytest.mark.gpu
def test_scan_arguments():
    g = torch.zeros(2, 3, 4, device="cuda")
    for bad in (dict(gate=g[0], value=g[0]), dict(gate=g, value=g[:, :2]), dict(gate=g, value=g.bfloat16()), dict(gate=g.double(), value=g.double()),
                dict(gate=g, value=g, state=g[0]), dict(gate=g, value=g, state=g[:, 0].bfloat16()), dict(gate=g, value=g, reset=g[:, :, 0]),
                dict(gate=g, value=g, reset=torch.zeros(2, 4, dtype=torch.bool, device="cuda"))):
        with pytest.raises(ValueError):
            ops.gated_scan(**bad)


def test_norm_entries():
    def norm(N_=4, D=8, dtype=N.F32, x=FAKE, residual=FAKE, weight=FAKE, y=FAKE, stream=FAKE):
        return refused("pv_add_rms_norm_hip", x, residual, weight, N_, D, D, D, 1e-6, dtype, y, stream, None)
    assert "dtype" in norm(dtype=3)
    assert "shape" in norm(N_=-1) and "shape" in norm(D=0)
    for name in ("x", "weight", "y", "stream"):
        assert "null" in norm(**{name: None})

    def bits8(format=N.E4M3, q=FAKE, scale=FAKE):
        return refused("pv_add_rms_norm_8bit_hip", FAKE, FAKE, FAKE, 4, 8, 8, 8, 1e-6, N.BF16, format, q, scale, FAKE)
    assert "format" in bits8(format=2)
    assert "null" in bits8(q=None) and "null" in bits8(scale=None)

    def back(work=FAKE, work_bytes=1 << 20, d=FAKE):
        return refused("pv_add_rms_norm_backward_hip", FAKE, FAKE, FAKE, 4000, 8, 8, FAKE, None, N.F32, d, FAKE, work, work_bytes)
    assert "work" in back(work=None) and "work" in back(work_bytes=16)
    assert "null" in back(d=None)


def test_loss_entry():
    def loss(B=2, T=5, D=8, V=5, dtype=N.BF16, wdtype=N.BF16, token_bytes=1, hidden=FAKE, d_hidden=None, d_weight=None, work=FAKE, work_bytes=1 << 20):
        return refused("pv_next_base_loss_hip", hidden, FAKE, FAKE, B, T, D, V, T * D, D, T, 4, dtype, wdtype, token_bytes, None, None, None, FAKE, d_hidden, d_weight,
                       work, work_bytes)
    assert "dtype" in loss(dtype=9)
    assert "weight_dtype" in loss(wdtype=N.F16)
    assert "token_bytes" in loss(token_bytes=4)
    for k in ("B", "T", "D"):
        assert "shape" in loss(**{k: 0})
    assert "V" in loss(V=0) and "V" in loss(V=17)
    assert "null" in loss(hidden=None) and "null" in loss(d_hidden=FAKE) and "null" in loss(d_weight=FAKE)
    assert "work" in loss(work=None) and "work" in loss(work_bytes=8)


def test_gradients_entries():
    vp, i64, i32 = ctypes.c_void_p * 1, ctypes.c_int64 * 1, ctypes.c_int32 * 1

    def norm(grad=FAKE, size=100, dtype=N.F32, norm=FAKE, work=FAKE, work_bytes=1 << 20):
        return refused("pv_gradient_norm_hip", vp(grad), i64(size), i32(dtype), 1, norm, work, work_bytes)

    def scale(grad=FAKE, out=FAKE, size=100, dtype=N.F32, norm=FAKE):
        return refused("pv_scale_gradients_hip", vp(grad), vp(out), i64(size), i32(dtype), 1, 1.0, norm)
    for fn in (norm, scale):
        assert "dtype" in fn(dtype=5)
        assert "size" in fn(size=-1) and "size" in fn(size=1 << 41)
        assert "null" in fn(grad=None) and "null" in fn(norm=None)
        assert "address" in fn(grad=FAKE + 2)
    assert "null" in scale(out=None)
    assert "work" in norm(work=None) and "work" in norm(work_bytes=4)


@pytest.mark.gpu
def test_norm_arguments():
    x, w = torch.zeros(2, 8, device="cuda"), torch.ones(8, device="cuda")
    for fn in (ops.add_rms_norm, ops.add_rms_norm_8bit):
        for bad in ((x, x[:1], w), (x, x.bfloat16(), w), (x, x, w[:4]), (x, x, w.int()), (x.double(), None, w), (x[:, :0], None, w[:0])):
            with pytest.raises(ValueError):
                fn(*bad)
    with pytest.raises(ValueError):
        ops.add_rms_norm_8bit(x, x, w, dtype=torch.float8_e5m2)


@pytest.mark.gpu
def test_loss_arguments():
    h, w, t = torch.zeros(2, 6, 8, device="cuda"), torch.zeros(5, 8, device="cuda"), torch.zeros(2, 6, dtype=torch.uint8, device="cuda")
    for fn in (ops.next_base_loss, ops.next_base_loss_grad):
        for bad in ((h[0], w, t), (h, w[:, :4], t), (h, w.bfloat16(), t), (h, torch.zeros(17, 8, device="cuda"), t), (h, w, t[:, :5]), (h, w, t.int()),
                    (h[:0], w, t[:0]), (h.double(), w, t)):
            with pytest.raises(ValueError):
                fn(*bad)
    with pytest.raises(ValueError):
        ops.next_base_loss(h, w, t, reduction="sum")
    with pytest.raises(ValueError):
        ops.next_base_loss_grad(h, w, t, scale=torch.ones(2, device="cuda"))


@pytest.mark.gpu
def test_clip_arguments():
    g = torch.zeros(5, device="cuda")
    for bad in (dict(grads=[g], max_norm=-1.0), dict(grads=[g], max_norm=float("nan")), dict(grads=[g.double()], max_norm=1.0), dict(grads=[g], max_norm=1.0, out=[]),
                dict(grads=[g], max_norm=1.0, out=[g[:3]]), dict(grads=[g], max_norm=1.0, out=[g.bfloat16()]), dict(grads=[g[::2]], max_norm=1.0, out=[torch.zeros(3, 1, device="cuda")])):
        with pytest.raises(ValueError):
            ops.clip_gradients(**bad)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.clip_gradients([g, torch.zeros(3)], 1.0)

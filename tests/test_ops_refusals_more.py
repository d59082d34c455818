"""What the gated delta rule, the layer norm and dropout refuse: the C entries' checks (before any launch, so without a GPU) and the
Python functions'; and that neither has forward-mode derivatives."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw

from panvram_amd import _native as N
from panvram_amd import ops
from tests.test_ops_refusals import FAKE, refused


def strides(*values):
    return (ctypes.c_int64 * len(values))(*values)


def delta(B=2, T=70, H=2, G=4, K=16, V=24, dtype=N.BF16, given=None, out=FAKE, kept=None, work=FAKE, work_bytes=1 << 40, query=FAKE, last=FAKE):
    s = given or strides(*([T * 64, 64, 16] * 5))
    return refused("pv_gated_delta_hip", query, FAKE, FAKE, FAKE, FAKE, None, None, B, T, H, G, K, V, s, 1e-6, dtype, out, last, kept, work, work_bytes)


def test_delta_entry():
    assert "dtype" in delta(dtype=5)
    for bad in (dict(B=0), dict(T=0), dict(H=0), dict(G=3), dict(G=1), dict(V=0), dict(V=(1 << 16) + 1), dict(K=0), dict(K=129)):
        assert "shape" in delta(**bad), bad
    assert "shape" in delta(H=1 << 16, G=1 << 16, K=128, B=1)
    assert "too many" in delta(B=1 << 22) and "too many" in delta(T=(1 << 31) - 1, B=64) and "too many" in delta(T=1 << 31)
    assert "stride" in delta(given=strides(0, (1 << 22) + 1, 0, *([64, 64, 16] * 4))) and "stride" in delta(given=strides(*([64, 64, 16] * 4), 0, -1, 0))
    for bad in (dict(out=None), dict(query=None), dict(last=None)):
        assert "null" in delta(**bad)
    assert "work" in delta(work=None) and "work" in delta(work_bytes=100) and "work" in delta(work=FAKE + 8)
    assert "kept" in delta(kept=FAKE + 8)
    assert "work" in delta(T=1, kept=FAKE, work=None)          # (kept for a backward pass, a single step goes by way of a chunk too)


def test_delta_backward_entry():
    def back(T=70, dtype=N.BF16, gate=FAKE, kept=FAKE, records=FAKE, d_key=FAKE, work=FAKE, work_bytes=1 << 40, step=64):
        return refused("pv_gated_delta_backward_hip", gate, FAKE, FAKE, None, 2, T, 2, 4, 16, 24, strides(640, 64, 1, 640, 64, 1, 640, step, 24), dtype, kept, records, FAKE,
                       d_key, FAKE, FAKE, FAKE, None, work, work_bytes)
    assert "dtype" in back(dtype=4) and "shape" in back(T=0) and "stride" in back(step=(1 << 22) + 1)
    for bad in (dict(gate=None), dict(kept=None), dict(records=None), dict(d_key=None)):
        assert "null" in back(**bad)
    assert "aligned" in back(kept=FAKE + 4) and "aligned" in back(records=FAKE + 8)
    assert "work" in back(work=None) and "work" in back(work_bytes=64) and "work" in back(work=FAKE + 8)


def test_delta_work_sizes():
    """Scratch memory grows with the sequence, and a pieces' share of it comes with few heads and many chunks."""
    f = N.lib().pv_gated_delta_work_bytes
    assert f(2, 8, 1, 1, 16, 16, N.BF16, 0) == 0 < f(2, 8, 1, 1, 16, 16, N.BF16, 1)
    assert f(1, 128, 1, 1, 16, 16, N.BF16, 0) == 2 * f(1, 64, 1, 1, 16, 16, N.BF16, 0)
    assert f(1, 4096, 1, 1, 128, 128, N.BF16, 0) > 64 * f(1, 64, 1, 1, 128, 128, N.BF16, 0)
    assert f(64, 4096, 8, 8, 128, 128, N.BF16, 0) == 64 * 8 * 64 * f(1, 64, 1, 1, 128, 128, N.BF16, 0)


def test_layer_entries():
    def layer(N_=4, D=8, dtype=N.F32, x=FAKE, residual=FAKE, weight=FAKE, y=FAKE, stream=FAKE, p=0.0, seed_at=None):
        return refused("pv_add_layer_norm_hip", x, residual, weight, None, N_, D, D, D, 1e-5, p, seed_at, 0, 0, dtype, y, stream, None)
    assert "dtype" in layer(dtype=3)
    assert "shape" in layer(N_=-1) and "shape" in layer(D=0) and "shape" in layer(N_=1 << 31) and "shape" in layer(D=1 << 31)
    for name in ("x", "weight", "y", "stream"):
        assert "null" in layer(**{name: None})
    assert "null" in layer(residual=None, stream=None, p=0.5)
    for p in (-0.1, 1.1, float("nan")):
        assert "p:" in layer(p=p)
    assert "seed" in layer(seed_at=FAKE + 4)

    def back(d=FAKE, d_x=FAKE, d_bias=FAKE, work=FAKE, work_bytes=1 << 30, p=0.5, seed_at=None):
        return refused("pv_add_layer_norm_backward_hip", FAKE, FAKE, FAKE, 4000, 8, 8, FAKE, None, p, seed_at, 0, 0, N.F32, d, d_x, FAKE, d_bias, work, work_bytes)
    assert "null" in back(d=None) and "null" in back(d_x=None) and "null" in back(d_bias=None)
    assert "work" in back(work=None) and "work" in back(work_bytes=16) and "work" in back(work=FAKE + 8)
    assert "seed" in back(seed_at=FAKE + 4) and "p:" in back(p=2.0)


def test_dropout_entry():
    def drop(x=FAKE, n=10, p=0.5, seed_at=None, dtype=N.F32, y=FAKE):
        return refused("pv_dropout_hip", x, n, p, seed_at, 0, 0, dtype, y)
    assert "dtype" in drop(dtype=3) and "shape" in drop(n=-1) and "shape" in drop(n=(1 << 48) + 1)
    for p in (-0.5, 1.5, float("nan")):
        assert "p:" in drop(p=p)
    assert "null" in drop(x=None) and "null" in drop(y=None)
    assert "address" in drop(x=FAKE + 2) and "address" in drop(y=FAKE + 1) and "address" in drop(seed_at=FAKE + 4)


CALLS = {
    "gated_delta": lambda t: ops.gated_delta(t, t, t, t[..., 0], t[..., 0]), "add_layer_norm": lambda t: ops.add_layer_norm(t, t, t[0, 0, 0], t[0, 0, 0]),
    "dropout": lambda t: ops.dropout(t, 0.5, 1),
}


@pytest.mark.parametrize("name", CALLS)
def test_no_cpu_tensors(name):
    with pytest.raises(RuntimeError, match=f"{name}.*GPU only"):
        CALLS[name](torch.zeros(2, 3, 4, 5))
    with fw.dual_level():
        t = fw.make_dual(torch.ones(2, 3, 4, 5), torch.ones(2, 3, 4, 5))
        with pytest.raises(NotImplementedError, match=f"{name}.*forward-mode"):
            CALLS[name](t)


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_gradients_of_gradients(name):
    t = torch.ones(2, 3, 4, 5, device="cuda", requires_grad=True)
    out = CALLS[name](t)
    out = out[0] if isinstance(out, tuple) else out
    (d,) = torch.autograd.grad(out.square().sum(), (t,), create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


@pytest.mark.gpu
def test_delta_arguments():
    r = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    good = dict(query=r(2, 5, 2, 8), key=r(2, 5, 2, 8), value=r(2, 5, 4, 6), gate=r(2, 5, 4), write=r(2, 5, 4))
    ops.gated_delta(**good)
    for bad in (dict(query=r(2, 5, 8)), dict(key=r(2, 5, 2, 7)), dict(value=r(2, 5, 3, 6)), dict(value=r(2, 4, 4, 6)), dict(value=r(2, 5, 4)), dict(gate=r(2, 5, 2)),
                dict(write=r(2, 5, 4, 1)), dict(gate=r(2, 5, 4).bfloat16()), dict(state=r(2, 4, 8, 5)), dict(state=r(2, 4, 8, 6).bfloat16()), dict(reset=r(2, 5)),
                dict(reset=torch.zeros(2, 4, dtype=torch.bool, device="cuda")), dict(query=r(2, 5, 2, 129), key=r(2, 5, 2, 129)), dict(value=r(2, 5, 4, 0)),
                dict(query=r(2, 5, 2, 0), key=r(2, 5, 2, 0)), dict(eps=-1.0), dict(eps=float("nan")), {k: v.double() for k, v in good.items()}):
        with pytest.raises(ValueError):
            ops.gated_delta(**(good | bad))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.gated_delta(**(good | dict(gate=torch.zeros(2, 5, 4))))
    with pytest.raises(ValueError, match="2\\^22"):
        big = torch.zeros(1, 1, 1, 1, device="cuda")
        ops.gated_delta(big.expand(1, 9, 1, 128), big.expand(1, 9, 1, 128), big.expand(1, 9, 1 << 16, 128), big[..., 0].expand(1, 9, 1 << 16), big[..., 0].expand(1, 9, 1 << 16))


@pytest.mark.gpu
def test_layer_arguments():
    x, w = torch.zeros(2, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (dict(residual=x[:1]), dict(residual=x.bfloat16()), dict(weight=w[:4]), dict(weight=w.int()), dict(bias=w[:4]), dict(bias=w.int()), dict(x=x.double(), residual=None),
                dict(x=x[:, :0], residual=None, weight=w[:0], bias=None), dict(dropout=-0.1, seed=1), dict(dropout=1.1, seed=1), dict(dropout=0.5), dict(dropout=0.5, seed=1 << 64),
                dict(dropout=0.5, seed=1, site=-1), dict(dropout=0.5, seed=1, site=1 << 32), dict(dropout=0.5, seed=torch.zeros(2, dtype=torch.int64, device="cuda")),
                dict(dropout=0.5, seed=torch.zeros(1, device="cuda"))):
        with pytest.raises(ValueError):
            ops.add_layer_norm(**(dict(x=x, residual=x, weight=w, bias=w) | bad))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.add_layer_norm(x, x, w, w, dropout=0.5, seed=torch.zeros(1, dtype=torch.int64))


@pytest.mark.gpu
def test_dropout_arguments():
    x = torch.zeros(5, device="cuda")
    for bad in (dict(p=-1e-3), dict(p=1.001), dict(p=float("nan")), dict(seed=None), dict(seed=1 << 64), dict(seed=-(1 << 63) - 1), dict(site=1 << 32), dict(x=x.double()), dict(x=x.int()),
                dict(seed=torch.zeros(1, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            ops.dropout(**(dict(x=x, p=0.5, seed=1) | bad))

"""ops.gated_delta where inputs are not finite: what a step's NaN or infinity reaches is what it reaches in the recurrence, not the steps before
it and not what lies behind a reset. And the gradients."""
import pytest
import torch

from panvram_amd import ops
from tests.ops_plain_more import delta, delta_off, near
from tests.test_gpu_delta import NAMES, made, wide

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAN, INF = float("nan"), float("inf")
WHERE = [("query", NAN), ("key", NAN), ("value", NAN), ("gate", NAN), ("write", NAN), ("query", INF), ("key", -INF), ("value", INF), ("value", -INF)]


def spoil(a, name, fill, at):
    t = a[name] = a[name].clone()
    t[0, at, 0, ...] = fill if t.dim() == 3 else t[0, at, 0]
    if t.dim() == 4:
        t[0, at, 0, 3] = fill


def same_places(got, want, off, dtype):
    """Finite where the recurrence is, and right there"""
    got, want = got.detach().cpu().double(), want.detach()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    near(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0), off, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name, fill", WHERE)
@pytest.mark.parametrize("T, at, reset", [(5, 2, 4), (70, 0, None), (70, 40, 50), (200, 70, 130), (200, 127, None), (200, 100, 100), (200, 63, 64), (1700, 600, 1100)])
def test_outputs(dtype, name, fill, T, at, reset):
    a, _, _ = made(2, T, 1, 2, 20, 24, dtype, seed=at)
    if reset is not None:
        a["reset"] = torch.zeros(2, T, dtype=torch.bool, device="cuda")
        a["reset"][:, reset] = True
    spoil(a, name, fill, at)
    if name == "gate" and reset == at:         # (a reset's gate has nothing to keep)
        a["gate"][0, at] = NAN
    out, last = delta(**wide(a))
    with torch.no_grad():
        got = ops.gated_delta(**a)
    same_places(got[0], out, delta_off("out", dtype), dtype)
    same_places(got[1], last, delta_off("last", dtype), torch.float32)
    if T <= 8:                                 # (by steps without gradients, in chunks with them)
        return
    a["value"].requires_grad_()
    for x, y in zip(ops.gated_delta(**a), got):        # with what is kept for gradients
        assert torch.equal(torch.nan_to_num(x.detach()), torch.nan_to_num(y))


@pytest.mark.parametrize("B, T, H, G, K, V", [(2, 300, 2, 4, 32, 40), (8, 130, 8, 16, 100, 70), (1, 2113, 1, 2, 128, 72)])
def test_several(B, T, H, G, K, V):
    """Some of each, resets between them, in all columns and heads; of few heads, many, and in pieces"""
    a, _, _ = made(B, T, H, G, K, V, torch.bfloat16, reset=0.04)
    gen = torch.Generator(device="cuda").manual_seed(2)
    for name, fill in WHERE:
        t = a[name]
        t[torch.rand(t.shape, generator=gen, device="cuda") < (0.004 if t.dim() == 3 else 0.0064 / t.shape[3])] = fill
    out, last = delta(**wide(a))
    assert 0.1 < torch.isfinite(out).double().mean() < 0.9
    with torch.no_grad():
        got = ops.gated_delta(**a)
    same_places(got[0], out, delta_off("out", torch.bfloat16), torch.bfloat16)
    same_places(got[1], last, delta_off("last", torch.bfloat16), torch.float32)


def test_a_key_of_zeros_without_eps():
    """0 / 0 in one step, where nothing is added to the squares: it reaches nothing before it."""
    a, _, _ = made(1, 100, 1, 1, 16, 24, torch.float32, state=False)
    a["key"][:, 50] = 0.0
    out, last = delta(**wide(a), eps=0.0)
    with torch.no_grad():
        got = ops.gated_delta(**a, eps=0.0)
    same_places(got[0], out, delta_off("out", torch.float32), torch.float32)
    assert torch.isfinite(got[0][:, :50]).all() and not torch.isfinite(got[1]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name, fill", WHERE + [("d_out", NAN), ("d_out", INF), ("state", NAN)])
@pytest.mark.parametrize("T, at, lo, hi", [(70, 40, 30, 50), (200, 100, 70, 130), (200, 64, 64, 128), (1700, 800, 500, 1100)])
def test_gradients_of_windows(dtype, name, fill, T, at, lo, hi):
    """Three windows behind each other, something in the middle one (or before the first): the others' gradients are what they are without it."""
    a, d_out, _ = made(1, T, 1, 2, 20, 24, dtype, seed=at, state=name == "state")
    a["reset"] = torch.zeros(1, T, dtype=torch.bool, device="cuda")
    a["reset"][:, [0, lo, hi]] = True
    names = [k for k in NAMES if a[k] is not None]

    def both(a, d):
        a = {k: t.detach().clone().requires_grad_() if k in names else t for k, t in a.items()}
        out, last = ops.gated_delta(**a)
        return dict(zip(names, torch.autograd.grad(out, [a[k] for k in names], d)))
    want = both(a, d_out)
    if name == "state":
        a["state"] = torch.full_like(a["state"], fill)
        assert all(torch.equal(x, y) for x, y in zip(both(a, d_out).values(), want.values()))
        return
    bad = a | {"d_out": d_out}
    spoil(bad, name, fill, at)
    have = both({k: bad[k] for k in a}, bad["d_out"])
    if name == "gate" and at == lo:            # (a reset's gate has nothing to keep)
        assert all(torch.equal(have[k], want[k]) for k in NAMES[:5] if k != "gate")
        return
    for k in NAMES[:5]:
        for x, y in ((have[k][:, :lo], want[k][:, :lo]), (have[k][:, hi:], want[k][:, hi:])):
            near(x, y, 2 * delta_off("d_" + k, dtype), dtype)
    # in the window itself the first head's are not finite wherever the recurrence's are not, and the other value head's are as they were
    # but for what it shares with it
    inner = {k: bad[k][:, lo:hi].detach().double().cpu().requires_grad_() for k in NAMES[:5]}
    ref = torch.autograd.grad(delta(**inner)[0], list(inner.values()), bad["d_out"][:, lo:hi].double().cpu())
    for k, r in zip(NAMES[:5], ref):
        h = have[k][:, lo:hi].cpu()
        if k == "gate":                        # (the first step's keeps nothing; in the window by itself it keeps a state of zeros)
            h, r = h[:, 1:], r[:, 1:]
        assert not torch.isfinite(h[~torch.isfinite(r)]).any(), k
    if name in ("value", "gate", "write", "d_out"):
        for k in ("value", "gate", "write"):
            assert torch.equal(have[k][:, :, 1], want[k][:, :, 1]), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_that_overlap(dtype):
    """Values, and gradients of out, whose steps are windows of one run of numbers: what a step has in one column, another has in the next."""
    T, V = 70, 24
    a, d_out, _ = made(1, T, 1, 1, 16, V, dtype, state=False)
    run, d_run = a["value"].flatten()[:T + V], d_out.flatten()[:T + V]
    run[T] = d_run[T] = NAN                        # columns 1 .. V - 1 of steps T - 1 .. T - V + 1, and column 0 of none
    a["value"], d_out = run.as_strided((1, T, 1, V), (0, 1, 0, 1)), d_run.as_strided((1, T, 1, V), (0, 1, 0, 1))
    out, last = delta(**wide(a))
    with torch.no_grad():
        got = ops.gated_delta(**a)
    same_places(got[0], out, delta_off("out", dtype), dtype)
    same_places(got[1], last, delta_off("last", dtype), torch.float32)
    assert torch.isfinite(got[1][..., 0]).all()
    a["value"] = a["value"].nan_to_num()
    leaves = {k: a[k].detach().requires_grad_() for k in NAMES[:5]}
    (d_value,) = torch.autograd.grad(ops.gated_delta(**leaves)[0], (leaves["value"],), d_out)
    assert torch.isfinite(d_value[..., 0]).all() and not torch.isfinite(d_value[:, :T - V + 1, :, 1:]).any()

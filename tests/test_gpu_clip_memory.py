"""What clipping does to the memory it writes: autograd knows of it, no gradient is scaled twice, and what an infinite or
undefined norm leaves of each element. Run with -m gpu."""
import pytest
import torch

from tests import ops_plain as P

pytestmark = pytest.mark.gpu


def test_autograd_knows_of_the_writing():
    """A gradient that a later operation has saved and that is then clipped: the second gradient is refused, as after any of
    torch's own in-place operations, and not made from other numbers."""
    from panvram_amd import ops
    for apart in (False, True):
        x = torch.randn(50, device="cuda", requires_grad=True)
        (g,) = torch.autograd.grad(x.pow(3).sum(), (x,), create_graph=True)
        y = (g * g).sum()                       # saves g
        if apart:
            ops.clip_gradients([torch.randn(50, device="cuda")], 1e-3, out=[g])
        else:
            ops.clip_gradients([g], 1e-3)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.parametrize("gaps", [False, True])
def test_versions(gaps):
    """Each written tensor's version goes up; those that are only read keep theirs."""
    from panvram_amd import ops
    make = lambda: [torch.randn(40, 6, device="cuda")[:, :3 if gaps else 6], torch.randn(5, device="cuda"), torch.randn(0, device="cuda")]  # noqa: E731
    grads, out = make(), make()
    was = [[t._version for t in ts] for ts in (grads, out)]
    ops.gradient_norm(grads)
    ops.clip_gradients(grads, 1.0, out=out)
    assert [t._version for t in grads] == was[0] and all(t._version > v for t, v in zip(out[:2], was[1]))
    ops.clip_gradients(grads, 1.0)
    assert all(t._version > v for t, v in zip(grads[:2], was[0]))


def test_inference_tensors():
    """Tensors made under inference_mode have no version and are clipped all the same."""
    from panvram_amd import ops
    with torch.inference_mode():
        g = [torch.full((100,), 2.0, device="cuda")]
        norm = ops.clip_gradients(g, 1.0)
        assert abs(float(norm) - 20) <= 1e-5 and float((g[0] - 0.1).abs().max()) <= 1e-6


def test_the_same_memory_twice_is_refused():
    """Two workgroups would scale the same elements, some once and some twice."""
    from panvram_amd import ops
    g, h = torch.randn(100, device="cuda"), torch.randn(100, device="cuda")
    keep = g.clone()
    with pytest.raises(ValueError, match="twice"):
        ops.clip_gradients([g, h, g], 1.0)
    with pytest.raises(ValueError, match="twice"):
        ops.clip_gradients([g, h], 1.0, out=[g, g])
    assert torch.equal(g, keep)
    empty = torch.zeros(0, device="cuda")
    norm = ops.clip_gradients([empty, g, empty, g[:0]], 1e-3)
    assert abs(float(norm) / float(keep.norm()) - 1) <= 1e-6
    assert abs(float(ops.gradient_norm([keep, keep])) / float(keep.double().norm() * 2 ** 0.5) - 1) <= 4 * P.U


def test_infinite_norms():
    """factor = min(1, max_norm / (norm + 1e-6)) throughout: an infinite norm makes 0 of finite elements and NaN of infinite
    ones, a norm of NaN makes NaN of all; a sum of squares whose root 32 bits do not hold is an infinite norm."""
    from panvram_amd import ops
    for apart in (False, True):
        for bad in (float("nan"), float("inf"), -float("inf"), 3e38):
            grads = [torch.randn(100, device="cuda"), torch.randn(5000, device="cuda")]
            grads[1][4321] = bad
            if bad == 3e38:
                grads[0][7] = bad
            out = [torch.zeros_like(g) for g in grads] if apart else None
            norm = ops.clip_gradients(grads, 1.0, out=out)
            got = torch.cat(out or grads)
            if bad != bad:
                assert torch.isnan(norm) and torch.isnan(got).all()
            else:
                assert float(norm) == float("inf")
                at = torch.zeros(5100, dtype=torch.bool, device="cuda")
                at[4421] = bad != 3e38
                assert torch.equal(torch.isnan(got), at) and not got[~at].any()

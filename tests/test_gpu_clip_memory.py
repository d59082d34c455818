"""What clipping does to the memory it writes: autograd knows of it. Run with -m gpu."""
import pytest
import torch

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

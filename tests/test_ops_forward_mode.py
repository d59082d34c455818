"""Forward-mode derivatives: no operator has one, so each says so instead of returning outputs without a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from panvram_amd import ops

CALLS = {
    "gated_scan": lambda t: ops.gated_scan(t, t), "add_rms_norm": lambda t: ops.add_rms_norm(t, t, t[0, 0]),
    "add_rms_norm_8bit": lambda t: ops.add_rms_norm_8bit(t, t, t[0, 0]),
    "next_base_loss": lambda t: ops.next_base_loss(t, t[0], torch.zeros(2, 3, dtype=torch.uint8, device=t.device)),
    "next_base_loss_grad": lambda t: ops.next_base_loss_grad(t, t[0], torch.zeros(2, 3, dtype=torch.uint8, device=t.device)),
    "clip_gradients": lambda t: ops.clip_gradients([torch.zeros_like(t), t], 1.0), "gradient_norm": lambda t: ops.gradient_norm([t]),
}


@pytest.mark.parametrize("name", CALLS)
def test_refused(name):
    with fw.dual_level():
        t = fw.make_dual(torch.ones(2, 3, 4), torch.ones(2, 3, 4))
        with pytest.raises(NotImplementedError, match=f"{name}.*forward-mode"):
            CALLS[name](t)


def test_refused_under_jvp():
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: ops.gated_scan(t, t)[0], (torch.ones(2, 3, 4),), (torch.ones(2, 3, 4),))


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_refused_on_the_gpu(name):
    with fw.dual_level():
        t = fw.make_dual(torch.ones(2, 3, 4, device="cuda"), torch.ones(2, 3, 4, device="cuda"))
        with pytest.raises(NotImplementedError, match=f"{name}.*forward-mode"):
            CALLS[name](t)


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_others_run_beside_dual_numbers(name):
    """Tensors without a tangent, where a level of dual numbers is open."""
    with fw.dual_level():
        CALLS[name](torch.ones(2, 3, 4, device="cuda"))

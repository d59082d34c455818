"""The gradient of ops.gated_delta's gate where states and their gradients are large in different rows."""
import pytest
import torch

from panvram_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 64, 130])
def test_large_states(dtype, T):
    """A state of 1e30 in one row and a gradient of 1e30 in another: their product, which is all that the gates get where nothing is written,
    is 0. Keys and queries are of the third row."""
    K, V = 16, 8
    a = {k: torch.zeros(1, T, 1, K, device="cuda", dtype=dtype) for k in ("query", "key")}
    for t in a.values():
        t[..., 2] = 1.0
    a["value"] = torch.zeros(1, T, 1, V, device="cuda", dtype=dtype)
    a["gate"] = torch.full((1, T, 1), -4.0, device="cuda", dtype=dtype)
    a["write"] = torch.full((1, T, 1), float("-inf"), device="cuda", dtype=dtype)
    a["state"] = torch.zeros(1, 1, K, V, device="cuda")
    a["state"][0, 0, 0] = 1e30
    d_last = torch.zeros_like(a["state"])
    d_last[0, 0, 1] = 1e30
    leaves = {k: t.requires_grad_() for k, t in a.items()}
    _, last = ops.gated_delta(**leaves)
    grads = dict(zip(leaves, torch.autograd.grad(last, list(leaves.values()), d_last)))
    assert all(torch.isfinite(g).all() for g in grads.values()), [k for k, g in grads.items() if not torch.isfinite(g).all()]
    assert not grads["gate"].any()

"""The gated scan of a single step of more channels than 32-bit byte offsets reach. Run with -m gpu."""
import pytest
import torch

pytestmark = pytest.mark.gpu


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

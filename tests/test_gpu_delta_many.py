"""ops.gated_delta in the forms that take many heads, whose walks have workgroups of four waves, or long keys in pieces."""
import pytest
import torch

from panvram_amd import ops
from tests.test_gpu_delta import NAMES, compare, made

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, T, H, G, K, V, reset", [(16, 70, 16, 16, 20, 24, 0.02), (8, 100, 8, 16, 64, 70, None), (8, 70, 16, 16, 100, 70, 0.02), (16, 65, 4, 8, 128, 128, None)])
def test_many_heads(dtype, B, T, H, G, K, V, reset):
    """256 workgroups of 64 columns and more, the last one of a head full or not"""
    assert B * G * (((V + 31) // 32 * 32 + 63) // 64) >= 256
    a, d_out, d_last = made(B, T, H, G, K, V, dtype, seed=K, reset=reset)
    compare(a, d_out, d_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, G, K, V, reset", [(2113, 2, 65, 40, 0.002), (2100, 1, 100, 128, None), (1600, 1, 128, 128, 0.002)])
def test_long_keys_in_pieces(dtype, T, G, K, V, reset):
    a, d_out, d_last = made(1, T, 1, G, K, V, dtype, seed=T, reset=reset, keep=-6.0)
    compare(a, d_out, d_last)


@pytest.mark.parametrize("B, T, G, K, V", [(1, 2113, 2, 128, 72), (16, 130, 16, 128, 40)])
def test_memory_that_held_something(B, T, G, K, V):
    """Workspaces and records that lie where NaN lay: nothing is read before it is written."""
    a, d_out, d_last = made(B, T, G, G, K, V, torch.bfloat16)
    leaves = [a[k].requires_grad_() for k in NAMES]

    def run():
        got = ops.gated_delta(**a)
        return [*(t.detach().clone() for t in got), *torch.autograd.grad(got, leaves, (d_out, d_last))]

    first = run()
    held = [torch.full((size,), float("nan"), device="cuda") for size in [1 << 26] * 8 + [1 << 22] * 8 + [1 << 16] * 64 + [1 << 10] * 64]
    del held
    for x, y in zip(first, run()):
        assert torch.isfinite(x).all() and torch.equal(x, y)

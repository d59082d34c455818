"""ops.gated_delta on tensors of 16 bits: its arithmetic is that of 32 bits, so that a result is the exact one rounded, but for the few
whose exact value lies next to a border between two numbers of the type."""
import pytest
import torch

from panvram_amd import ops
from tests.ops_plain import U
from tests.ops_plain_more import delta
from tests.test_gpu_delta import NAMES, made, wide

pytestmark = pytest.mark.gpu
SHAPES = [(2, 130, 2, 4, 38, 109), (1, 300, 2, 2, 128, 128), (1, 1300, 1, 2, 24, 64), (2, 70, 2, 2, 64, 72)]


def flips(name, got, want, chains=1.0):
    """Asserts that `got` is `want` rounded to its type but for flips to the other side of a border. With e what arithmetic is off by, a
    value x flips with a chance of 2 |e| / step and is a step off then, a step being eps |x| at most: the flips have a 2-norm of
    sqrt(sum 2 |e| step) <= sqrt(2 eps |e| |x|) together. Of e: four sums of 256 terms each, whose roundings in 32 bits add up as the
    root of their number, 16 U, and eight roundings of operands to 22 bits; `chains` times that."""
    eps, off = torch.finfo(got.dtype).eps, chains * (4 * 16 * U + 8 * 2.0 ** -23)
    got, want = got.detach().cpu(), want.detach()
    found = float((got.double() - want.to(got.dtype).double()).norm() / want.norm())
    assert found <= (2 * eps * off) ** 0.5, (name, found, (2 * eps * off) ** 0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B, T, H, G, K, V", SHAPES)
def test_outputs(dtype, B, T, H, G, K, V):
    a, _, _ = made(B, T, H, G, K, V, dtype, seed=T)
    with torch.no_grad():
        flips("out", ops.gated_delta(**a)[0], delta(**wide(a))[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B, T, H, G, K, V", SHAPES)
def test_gradients(dtype, B, T, H, G, K, V):
    """A gradient's chain of sums is twice an output's."""
    a, d_out, d_last = made(B, T, H, G, K, V, dtype, seed=T)
    ref = wide(a)
    leaves = {k: ref[k].requires_grad_() for k in NAMES}
    want = torch.autograd.grad(delta(**ref), list(leaves.values()), (d_out.double().cpu(), d_last.double().cpu()))
    own = a | {k: a[k].detach().requires_grad_() for k in NAMES}
    have = torch.autograd.grad(ops.gated_delta(**own), [own[k] for k in NAMES], (d_out, d_last))
    for name, h, w in zip(NAMES, have, want):
        if name != "state":
            flips("d_" + name, h, w, 2.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B, T, H, G, K, V", SHAPES)
def test_with_and_without_gradients(dtype, B, T, H, G, K, V):
    """Whether gradients will be asked for does not change results."""
    a, _, _ = made(B, T, H, G, K, V, dtype, seed=T)
    with torch.no_grad():
        want = ops.gated_delta(**a)
    a["value"].requires_grad_()
    got = ops.gated_delta(**a)
    assert got[0].requires_grad and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

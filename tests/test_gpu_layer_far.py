"""ops.add_layer_norm of rows whose sums leave 32 bits and whose elements are all alike."""
import pytest
import torch

from panvram_amd import ops
from tests.ops_plain import U, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, value", [(torch.float32, 1.75 * 2.0 ** 127), (torch.float32, -1.25 * 2.0 ** 127), (torch.bfloat16, 1.5 * 2.0 ** 127)])
@pytest.mark.parametrize("D", [64, 1024, 65536])
def test_rows_of_one_value(dtype, value, D):
    """Nothing is left of such a row around its mean, which is exact where D is a power of two and the value's bits and D's are 24 together: y is the
    bias, and gradients are those of a row of zeros."""
    x = torch.full((3, D), value, device="cuda", dtype=dtype).requires_grad_()
    zero = torch.zeros_like(x).detach().requires_grad_()
    gen = torch.Generator(device="cuda").manual_seed(D)
    w, b = (torch.randn(D, generator=gen, device="cuda") for _ in range(2))
    d = torch.randn(3, D, generator=gen, device="cuda").to(dtype)
    y, _ = ops.add_layer_norm(x, None, w, b)
    assert torch.equal(y, b.to(dtype).expand(3, D))
    (got,), (want,) = (torch.autograd.grad(ops.add_layer_norm(t, None, w, b)[0], (t,), d) for t in (x, zero))
    # one over the root of eps is made in a few last places either way
    assert bool(((got.double() - want.double()).abs() <= 16 * U * want.double().abs() + 2 * rounded(want.double(), dtype)).all())

"""The gradients of the logits enter the next-base loss's products with the bits that 32-bit arithmetic has, whatever the
type of hidden and head: sums of them that are zero in the definition come out as zero but for 32-bit roundings. Run with
-m gpu."""
import pytest
import torch

from tests import ops_plain as P

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [60, 512, 2100])
def test_d_hidden_where_all_ids_weigh_the_same(D, dtype):
    """A column in which the head has the same weight c for every id: d_hidden = c (sum of softmax - 1) = 0. Off by, in
    last places (U) of c: V + 3 for the softmax's sum and reciprocal, 2 each for the subtraction, the factor and what the
    products leave out of each gradient, and 2 V + 2 for the products' sum, whose partial sums are at most 1."""
    from panvram_amd import ops
    V = 5
    gen = torch.Generator().manual_seed(D)
    hidden = torch.randn(3, 700, D, generator=gen).to(dtype).cuda()
    weight = torch.randn(V, D, generator=gen) * D ** -0.5 * 2
    weight[:, ::2] = 1.0
    tokens = torch.randint(V, (3, 700), generator=gen, dtype=torch.uint8).cuda()
    h = hidden.requires_grad_()
    each = ops.next_base_loss(h, weight.to(dtype).cuda(), tokens, ignore=None, reduction="none")
    (d,) = torch.autograd.grad(each, (h,), torch.ones(3, 700, device="cuda"))
    d = d[..., ::2].double().abs()
    assert float(d.max()) <= (3 * V + 11) * P.U + P.TINY[dtype]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [60, 512, 2100])
def test_d_weight_of_factors_that_cancel(D, dtype):
    """Three places with the same hidden values and next id, and factors a, b and -(a + b): d_weight = 0. Off by, in last
    places of (a + b) |hidden|: 2 for the three products with the factors, 2 for what is left out of each gradient, 12 for
    the sum (three additions, of parts, with partial sums of at most 1 of it)."""
    from panvram_amd import ops
    V = 16
    gen = torch.Generator().manual_seed(D + 1)
    for _ in range(12):
        hidden = torch.randn(1, 1, D, generator=gen).to(dtype).expand(1, 4, D).contiguous().cuda()
        weight = (torch.randn(V, D, generator=gen) * D ** -0.5 * 2).to(dtype).cuda().requires_grad_()
        tokens = torch.full((1, 4), 3, dtype=torch.uint8, device="cuda")
        a, b = (torch.randint(1, 1 << 20, (2,), generator=gen) / 2.0 ** 21).tolist()
        each = ops.next_base_loss(hidden, weight, tokens, ignore=None, reduction="none")
        (d,) = torch.autograd.grad(each, (weight,), torch.tensor([[a, b, -(a + b), 0.0]], device="cuda"))
        over = d.double().abs() - 16 * P.U * (a + b) * hidden[0, 0].double().abs() - P.TINY[dtype]
        assert float(over.max()) <= 0

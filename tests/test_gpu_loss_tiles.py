"""The next-base loss where a workgroup works on several tiles of places, the last of them a part of one: more tiles than
workgroups on every path, with and without gradients, in each type. Run with -m gpu."""
import pytest
import torch

from tests import ops_plain as P
from tests.test_gpu_loss import check, make

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]

# (B, T, D): a row of D columns is cut into slabs of 128 (16-bit products) or 64 (32-bit), a wave each. With gradients there
# are at most 256 * (16 // waves) workgroups of 16 places a tile; rows of more than 16 slabs go by 256 workgroups a column block.
MANY = [(2, 4111, 1024), (3, 1800, 2048), (1, 4500, 2100), (2, 9000, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D", MANY)
def test_sizes(B, T, D, dtype):
    check(*make(B, T, D, 5, dtype, seed=T + D))


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_weight_in_32_bits(dtype):
    check(*make(2, 2500, 1000, 6, dtype, seed=1, wtype=torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_narrow_rows(dtype):
    """One wave a workgroup: up to 4,096 workgroups with gradients and 6,144 without."""
    check(*make(3, 33_001, 24, 4, dtype, seed=2))


@pytest.mark.parametrize("T,D,dtype", [(t, d, k) for k in TYPES for t, d in ((30_011, 512), (14_007, 1024), (132_001, 1030) if k == torch.float32 else (131_501, 2051))])
def test_scores(T, D, dtype):
    """Losses alone: 256 * (24 // waves) workgroups, or 2,048 of four tiles where the row has more than 16 slabs (1,030
    columns of 32 bits, 2,051 of 16). Compared at every 13th place and at the last ones."""
    from panvram_amd import ops
    hidden, weight, tokens = make(1, T, D, 5, dtype, seed=T)
    each = ops.next_base_loss(hidden, weight, tokens, reduction="none").cpu()
    at = torch.cat([torch.arange(0, T - 300, 13), torch.arange(T - 300, T - 1)])
    pairs = torch.stack([tokens.cpu()[0, at], tokens.cpu()[0, at + 1]], 1)          # rows of two: a place and its next token
    two = torch.stack([hidden.cpu()[0, at], torch.zeros(len(at), D, dtype=dtype)], 1)
    want, bound = P.loss(two, weight.cpu(), pairs, 4)["each"]
    P.inside(each[0, at], want[:, 0], bound[:, 0] + P.rounded(want[:, 0], torch.float32))
    assert float(each[0, -1]) == 0
    mean = ops.next_base_loss(hidden, weight, tokens)
    counted = int((tokens[0, 1:] < 4).sum())
    total = float(each.double().sum()) / counted
    assert abs(float(mean) - total) <= 4 * P.U * total


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D", [(1, 8900, 1024), (1, 4700, 2100), (1, 70_000, 24)])
def test_factors_of_all_sizes(B, T, D, dtype):
    """Gradients of the places' losses from 2^-46 to 2^4, rising and falling from tile to tile of a workgroup: sums that began
    small go on as large ones, and the other way round. (All sums are within float16's range.)"""
    from panvram_amd import ops
    hidden, weight, tokens = make(B, T, D, 7, dtype, seed=D)
    tokens %= 7
    rising = torch.exp2(torch.linspace(-46, 4, T)).view(B, T)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    for factor in (rising, rising.flip(1), torch.where(torch.arange(T) % 5 == 0, rising, rising.flip(1))):
        d = torch.autograd.grad(ops.next_base_loss(h, w, tokens, ignore=None, reduction="none"), (h, w), factor.cuda())
        plain = P.loss(hidden.detach().cpu(), weight.detach().cpu(), tokens.cpu(), None, factor=factor)
        for got, name in zip(d, ("d_hidden", "d_weight")):
            P.inside(got, plain[name][0], plain[name][1] + P.rounded(plain[name][0], dtype))


def test_growing_sums_in_float16():
    """Each tile of a workgroup's has gradients far larger than all before it, and d_weight is the definition's in every
    tile's share: the sums are scaled again whenever a tile needs it, and keep what they hold."""
    from panvram_amd import ops
    hidden, weight, tokens = make(1, 3 * 4096 + 5, 2048, 4, torch.float16, seed=5)
    tokens %= 4
    T = tokens.shape[1]
    w = weight.requires_grad_()
    for step in (7, 12, -9):
        power = (torch.arange(T) // 4096 * step).float()
        factor = torch.exp2(power - power.max() - 4).view(1, T)
        (d,) = torch.autograd.grad(ops.next_base_loss(hidden, w, tokens, ignore=None, reduction="none"), (w,), factor.cuda())
        want, bound = P.loss(hidden.cpu(), weight.detach().cpu(), tokens.cpu(), None, factor=factor)["d_weight"]
        P.inside(d, want, bound + P.rounded(want, torch.float16))


def test_same_from_run_to_run():
    from panvram_amd import ops
    hidden, weight, tokens = make(2, 8200, 1024, 5, torch.bfloat16, seed=6)
    want = ops.next_base_loss_grad(hidden, weight, tokens)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, ops.next_base_loss_grad(hidden, weight, tokens)))

"""ops.dropout against the definition of its bits, element by element."""
import pytest
import torch

from panvram_amd import ops
from tests.ops_plain import U, inside, rounded
from tests.ops_plain_more import kept

pytestmark = pytest.mark.gpu


def check(y, x, p, seed, site=0):
    keep, up = kept(x.numel(), p, seed, site)
    want = torch.where(keep.view(x.shape), x.double().cpu() * up, 0.0)
    assert torch.equal(y.cpu() == 0, want == 0)
    inside(y, want, 2 * U * want.abs() + rounded(want, x.dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9, 1), (3, 5, 7), (257, 500), (1030, 1024)])
def test_elements(dtype, shape):
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = torch.randn(shape, generator=gen, device="cuda").add_(5).to(dtype).requires_grad_()
    seed = torch.tensor([0x0123456789ABCDEF], device="cuda")
    y = ops.dropout(x, 0.25, seed, site=3)
    check(y, x.detach(), 0.25, int(seed), 3)
    d = torch.randn(shape, generator=gen, device="cuda").sub_(5).to(dtype)
    (d_x,) = torch.autograd.grad(y, (x,), d)
    check(d_x, d, 0.25, int(seed), 3)
    assert torch.equal(y, ops.dropout(x, 0.25, int(seed), 3))


@pytest.mark.parametrize("seed", [0, 1, 2 ** 32, 2 ** 63, 2 ** 64 - 1, -1])
def test_seeds(seed):
    x = torch.ones(999, device="cuda")
    check(ops.dropout(x, 0.4, seed, (1 << 32) - 1), x, 0.4, seed, (1 << 32) - 1)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -16, 0.5, 1 - 2.0 ** -16, 1.0])
def test_shares(p):
    x = torch.full((70001,), -2.0, device="cuda", dtype=torch.bfloat16)
    check(ops.dropout(x, p, 5), x, p, 5)


def test_dropped_whatever_it_was():
    x = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda").repeat(500).requires_grad_()
    y = ops.dropout(x, 0.5, 11)
    keep, _ = kept(x.numel(), 0.5, 11)
    assert bool((y.detach().cpu()[~keep] == 0).all()) and not torch.isfinite(y.detach().cpu()[keep][:2]).all()
    (d,) = torch.autograd.grad(y, (x,), torch.full_like(y, float("nan")))
    assert bool((d.cpu()[~keep] == 0).all()) and bool(torch.isnan(d.cpu()[keep]).all())


def test_layouts():
    """Views of any strides are dropped by their own index; a tensor that begins off 16 bytes; none at all."""
    base = torch.randn(40, 130, device="cuda").add_(4)
    for x in (base.T, base[:, 3:60], base[::2], base.view(-1)[1:], base[:0], base[:1].expand(40, 130)):
        check(ops.dropout(x, 0.3, 9), x, 0.3, 9)


def test_replayed():
    """A captured call reads its seed at each replay, which the graph counts up."""
    x = torch.randn(5000, device="cuda").add_(4).requires_grad_()
    seed = torch.tensor([100], device="cuda")
    d = torch.ones(5000, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.dropout(x, 0.5, seed), (x,), d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout(x, 0.5, seed)
        (g,) = torch.autograd.grad(y, (x,), d)
        seed += 1
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        now = int(seed) - 1
        assert now == 100 + k
        check(y, x.detach(), 0.5, now)
        check(g, d, 0.5, now)


def test_seed_changed_before_backward():
    x = torch.randn(50, device="cuda").requires_grad_()
    seed = torch.tensor([1], device="cuda")
    y = ops.dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_past_32_bit_indexes():
    """Elements behind index 2^32, in more than one launch's reach of 32-bit offsets."""
    n = (1 << 32) + 1000
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = ops.dropout(x, 0.5, 77)
    for first in (0, (1 << 31) - 8, (1 << 32) - 504, n - 1000):
        count = min(1000, n - first)
        keep, up = kept(count, 0.5, 77, first=first)
        assert torch.equal(y[first:first + count].cpu().double(), keep.double() * up)
    del x, y


def test_other_stream():
    x = torch.ones(1 << 20, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.dropout(x, 0.5, 1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ops.dropout(x, 0.5, 1))

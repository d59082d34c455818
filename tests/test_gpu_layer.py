"""ops.add_layer_norm and its gradients against definitions in 64 bits."""
import pytest
import torch

from panvram_amd import ops
from tests.ops_plain import inside, rounded
from tests.ops_plain_more import kept, layer

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def made(N, D, dtype, seed=0, mean=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, std=1.0, mean=0.0, kind=dtype: torch.randn(*s, generator=gen, device="cuda").mul_(std).add_(mean).to(kind)  # noqa: E731
    return (r(N, D), r(N, D, std=2.0, mean=mean), r(D, std=0.3, mean=1.0, kind=torch.float32), r(D, std=0.5, kind=torch.float32), r(N, D, std=0.1), r(N, D, std=0.1))


def compare(x, residual, w, b, d_y, d_stream, eps=1e-5, p=0.0, seed=None, site=0):
    dtype, N, D = x.dtype, x.shape[0], x.shape[1]
    wanted = [t.detach().requires_grad_() for t in (x, residual, w, b) if t is not None]
    it = iter(wanted)
    x, residual, w, b = (None if t is None else next(it) for t in (x, residual, w, b))
    y, stream = ops.add_layer_norm(x, residual, w, b, eps=eps, dropout=p, seed=seed, site=site)
    assert y.dtype == stream.dtype == dtype and y.shape == stream.shape == x.shape
    keep, up = kept(N * D, p, seed or 0, site) if p else (torch.ones(N * D, dtype=torch.bool), 1.0)
    keep = keep.view(N, D)
    dropped = torch.where(keep, x.detach().double().cpu() * up, 0.0)
    want = dropped + (residual.detach().double().cpu() if residual is not None else 0.0)
    inside(stream, want, 2 * 2.0 ** -24 * (dropped.abs() + want.abs()) + rounded(want, dtype))
    cpu = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    plain = layer(cpu(stream), cpu(w), cpu(b), eps, cpu(d_y), cpu(d_stream))
    inside(y, plain["y"][0], plain["y"][1] + rounded(plain["y"][0], dtype))
    outs, ds = ((y, stream), (d_y, d_stream)) if d_stream is not None else ((y,), (d_y,))
    got = list(torch.autograd.grad(outs, wanted, ds))
    d, e = plain["d"]
    dx, ex = torch.where(keep, d * up, 0.0), torch.where(keep, e * up, 0.0)
    # where x itself is the stream, autograd adds d_stream to the norm's part d - d_stream after that has been rounded by itself:
    # half a step of the part (UNIT |d - d_stream|) beside half a step of the sum, of (1 + UNIT) |sum| at most
    twice = rounded(d - d_stream.double().cpu(), dtype) * (1 + 2.0 ** -8) if residual is None and not p and d_stream is not None else 0.0
    inside(got.pop(0), dx, ex + rounded(dx, dtype) + twice)
    if residual is not None:
        inside(got.pop(0), d, e + rounded(d, dtype))
    inside(got.pop(0), *plain["d_weight"])
    if b is not None:
        inside(got.pop(0), *plain["d_bias"])
    with torch.no_grad():
        again = ops.add_layer_norm(x, residual, w, b, eps=eps, dropout=p, seed=seed, site=site)
    assert torch.equal(again[0], y) and torch.equal(again[1], stream)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N, D", [(1, 1), (3, 2), (5, 63), (33, 64), (70, 129), (9, 500), (4, 513), (17, 1024), (5, 2047), (3, 4100), (2, 8200), (3, 20011), (2, 33000)])
def test_rows(dtype, N, D):
    compare(*made(N, D, dtype, seed=D))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N, D", [(1, 1), (7, 61), (13, 500), (6, 1024), (3, 4100), (2, 40000)])
def test_dropout(dtype, N, D):
    compare(*made(N, D, dtype, seed=D), p=0.3, seed=12345678901234567, site=2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_forms(dtype):
    """Without a residual, a bias, or a gradient of the stream; dropout without a residual; nearly and really everything dropped."""
    x, residual, w, b, d_y, d_stream = made(19, 300, dtype)
    compare(x, None, w, b, d_y, d_stream)
    compare(x, None, w, None, d_y, None)
    compare(x, residual, w, None, d_y, None)
    compare(x, None, w, b, d_y, d_stream, p=0.25, seed=4)
    compare(x, residual, w, b, d_y, None, p=1.0, seed=4)
    compare(x, residual, w, b, d_y, d_stream, p=2.0 ** -20, seed=4)


def test_only_the_stream():
    """A gradient that comes from the stream alone."""
    x, residual, w, b, _, d = made(9, 130, torch.float32)
    x.requires_grad_(), residual.requires_grad_()
    _, stream = ops.add_layer_norm(x, residual, w, b, dropout=0.5, seed=3)
    dx, dr = torch.autograd.grad(stream, (x, residual), d)
    keep, up = kept(9 * 130, 0.5, 3)
    assert torch.equal(dr, d) and torch.equal(dx.cpu(), torch.where(keep.view(9, 130), d.cpu() * up, 0.0))


@pytest.mark.parametrize("rows", [1, 8000, 70001])
def test_many_rows(rows):
    """Several groups of rows in a workgroup: the sums of the weight's and the bias's gradients."""
    compare(*made(rows, 40, torch.bfloat16, seed=rows))
    compare(*made(rows // 8 + 1, 300, torch.float32, seed=rows), p=0.1, seed=rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mean", [30.0, -1000.0])
def test_far_from_zero(dtype, mean):
    x, residual, w, b, d_y, d_stream = made(6, 777, dtype, mean=mean)
    compare(x, residual, w, b, d_y, d_stream)


@pytest.mark.parametrize("scale", [1e-36, 1e-25, 1e25, 2e37])
def test_range(scale):
    """Squares and sums past 32 bits and below them, without an eps that covers them."""
    x, _, w, b, d_y, _ = made(7, 600, torch.float32)
    y, _ = ops.add_layer_norm(x * scale, None, w, b, eps=0.0)
    want, bound = layer((x * scale).cpu(), w.cpu(), b.cpu(), 0.0)["y"]
    inside(y, want, bound + 2.0 ** -20)            # (of numbers below 2^-126 the last places are gone)


def test_largest_numbers():
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[big, -big] * 50, [big] * 99 + [-big], [0.0] * 100], device="cuda").requires_grad_()
    w, b = torch.ones(100, device="cuda"), torch.zeros(100, device="cuda")
    y, _ = ops.add_layer_norm(x, None, w, b)
    want, bound = layer(x.detach().cpu(), w.cpu(), b.cpu(), 1e-5)["y"]
    inside(y, want, bound)
    (d,) = torch.autograd.grad(y, (x,), torch.ones_like(y))
    assert torch.isfinite(d).all()


def test_not_finite_rows():
    """A NaN or an infinity takes its own row and no other."""
    x = torch.randn(6, 90, device="cuda")
    x[1, 3], x[4, 89] = float("nan"), float("inf")
    w, b = torch.ones(90, device="cuda"), torch.zeros(90, device="cuda")
    y, _ = ops.add_layer_norm(x, None, w, b)
    assert torch.isnan(y[1]).all() and torch.isnan(y[4]).all() and torch.isfinite(y[[0, 2, 3, 5]]).all()


def test_layouts():
    """Row strides, rows off 16 bytes, transposed and broadcast tensors, leading dimensions."""
    base = torch.randn(30, 2 * 101 + 1, device="cuda").bfloat16()
    w, b = torch.rand(101, device="cuda") + 0.5, torch.randn(101, device="cuda")
    d = torch.randn(30, 101, device="cuda").bfloat16()
    a, c = base[:, 1:102], base[:, 102:]
    compare(a, c, w, b, d, None)
    compare(a, base[:1, :101].expand(30, 101), w, b, d, d, p=0.2, seed=8)
    t = torch.randn(101, 30, device="cuda").bfloat16().T
    compare(t, t, w, b, d, None)
    y, s = ops.add_layer_norm(a.unflatten(0, (5, 6)), c.unflatten(0, (5, 6)), w, b, dropout=0.2, seed=1)
    y2, s2 = ops.add_layer_norm(a, c, w, b, dropout=0.2, seed=1)
    assert torch.equal(y.flatten(0, 1), y2) and torch.equal(s.flatten(0, 1), s2)
    empty = ops.add_layer_norm(a[:0], c[:0], w, b)[0]
    assert empty.shape == (0, 101)
    wb = w.bfloat16().requires_grad_()
    y, _ = ops.add_layer_norm(a, c, wb, None)
    (g,) = torch.autograd.grad(y, (wb,), d)
    assert g.dtype == torch.bfloat16


def test_no_rows_gradients():
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    y, _ = ops.add_layer_norm(x, x, w, b)
    for g in torch.autograd.grad(y, (w, b), torch.zeros_like(y)):
        assert torch.equal(g, torch.zeros(8, device="cuda"))


def test_differences():
    """The gradients against differences of the function itself, in 32 bits."""
    x, residual, w, b, d_y, d_stream = (t.detach() for t in made(3, 37, torch.float32))
    leaves = [t.requires_grad_() for t in (x, residual, w, b)]

    def value(*ts):
        y, stream = ops.add_layer_norm(*ts, dropout=0.3, seed=2)
        return (y.double() * d_y).sum() + (stream.double() * d_stream).sum()
    got = torch.autograd.grad(value(*leaves), leaves)
    h = 2.0 ** -7
    for k, g in enumerate(got):
        step = torch.randn(leaves[k].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k))
        with torch.no_grad():
            at = lambda e: value(*(t + e * step if j == k else t for j, t in enumerate(leaves)))  # noqa: E731
            slope = (at(h) - at(-h)) / (2 * h)
        # third derivatives h^2 and roundings of some 200 values / h
        assert abs(float(slope) - float((g * step).sum())) < 20 * h * h + 200 * 2.0 ** -22 / h


def test_captured():
    """Forwards and backwards in a graph, replayed with other inputs and a seed counted up, between eager calls."""
    x, residual, w, b, d_y, d_stream = made(300, 256, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, residual, w, b)]
    seed = torch.tensor([5], device="cuda")

    def both(seed):
        out = ops.add_layer_norm(x, residual, w, b, dropout=0.1, seed=seed, site=1)
        return (*out, *torch.autograd.grad(out, leaves, (d_y, d_stream)))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both(seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(seed)
        seed += 1
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, both(int(seed) - 1)):
            assert torch.equal(a, c)

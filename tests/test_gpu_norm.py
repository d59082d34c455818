"""The residual addition and norm against the definition in 64 bits (tests/ops_plain.py), in the stream's type and in 8 bits,
and the gradients against the formula's and against differences. Run with -m gpu."""
import pytest
import torch

from tests import ops_plain as P

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-6


def make(N, D, dtype, seed, residual=True):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return (n(N, D).to(dtype).cuda(), (2 * n(N, D)).to(dtype).cuda() if residual else None, (1 + 0.3 * n(D)).cuda(), n(N, D).to(dtype).cuda(), n(N, D).to(dtype).cuda())


def check(x, residual, weight, d_y=None, d_stream=None):
    from panvram_amd import ops
    wanted = [t.detach().requires_grad_() for t in (x, residual, weight) if t is not None]
    a, w = wanted[0], wanted[-1]
    y, stream = ops.add_rms_norm(a, wanted[1] if residual is not None else None, w, eps=EPS)
    want_stream = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    assert torch.equal(stream, want_stream) and y.dtype == x.dtype and y.shape == x.shape
    flat = lambda t: None if t is None else t.detach().cpu().reshape(-1, x.shape[-1])  # noqa: E731
    plain = P.norm(flat(want_stream), weight.cpu(), EPS, flat(d_y), flat(d_stream) if residual is not None else None)
    P.inside(y.reshape(-1, x.shape[-1]), plain["y"][0], plain["y"][1] + P.rounded(plain["y"][0], x.dtype))
    if d_y is not None:
        outs, ds = ((y, stream), (d_y, d_stream)) if residual is not None else ((y,), (d_y,))
        d = torch.autograd.grad(outs, wanted, ds)
        for got in d[:-1]:
            P.inside(got.reshape(-1, x.shape[-1]), plain["d"][0], plain["d"][1] + P.rounded(plain["d"][0], x.dtype))
        P.inside(d[-1], plain["d_weight"][0], plain["d_weight"][1] + P.rounded(plain["d_weight"][0], torch.float32))
    with torch.no_grad():
        again, s2 = ops.add_rms_norm(x, residual, weight, eps=EPS)
    assert torch.equal(again, y) and torch.equal(s2, stream)


SIZES = [(1, 1), (5, 3), (1, 64), (3, 63), (7, 65), (2, 128), (4, 500), (33, 512), (16, 1000), (9, 1024), (3, 1025), (5, 2048), (3, 2056), (2, 4096), (2, 5000),
         (3, 8192), (1, 20000), (2, 20001), (1100, 72), (2, 65536)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D", SIZES)
def test_sizes(N, D, dtype):
    check(*make(N, D, dtype, seed=N * 100000 + D))


@pytest.mark.parametrize("dtype", TYPES)
def test_without_residual(dtype):
    for N, D in ((3, 70), (5, 1024), (2, 9000)):
        check(*make(N, D, dtype, seed=D, residual=False))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [512, 515])
def test_strided_and_shaped(D, dtype):
    """Rows of a wider matrix, three dimensions, a start off the wide loads' alignment, columns apart, a shared gradient."""
    x, residual, weight, d_y, d_s = make(6, 2 * D, dtype, seed=D)
    w = weight[:D].contiguous()
    check(x[:, :D], residual[:, D:], w, d_y[:, :D], d_s[:, D:])
    check(x[:, 1:D + 1], residual[:, :D], w, d_y[:, :D], d_s[:, :D])
    check(x.view(2, 3, 2 * D)[..., :D], residual.view(2, 3, 2 * D)[..., :D], w, d_y.view(2, 3, 2 * D)[..., :D], d_s.view(2, 3, 2 * D)[..., D:])
    check(x[:, ::2], residual[:, 1::2], w, d_y[:, ::2], d_s[:, ::2])
    check(x[:, :D], residual[:, :D], w, torch.full((1, 1), 0.5, device="cuda", dtype=dtype).expand(6, D), d_s[:, :D])


def quantised(x, residual, weight, kind):
    from panvram_amd import ops
    q, scale, stream = ops.add_rms_norm_8bit(x, residual, weight, eps=EPS, dtype=kind)
    want = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    assert torch.equal(stream, want) and q.dtype == kind and q.shape == x.shape and scale.shape == x.shape[:-1]
    y, bound = P.norm(want.cpu(), weight.cpu(), EPS)["y"]
    most = 448.0 if kind == torch.float8_e4m3fn else 127.0
    s = y.abs().amax(-1) / most
    c = (x.shape[-1] / 64 + 24) * P.U
    P.inside(scale, s, c * s)
    v = torch.where(s[:, None] > 0, y / s[:, None], torch.zeros(()).double())
    if kind == torch.int8:
        half = torch.full_like(v, 0.5)
    else:       # half the distance of neighbours: 3 bits behind the leading one, down to 2^-9
        half = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4)
    P.inside(q.float(), v, half * (1 + 1e-6) + 2 * c * v.abs())
    return q, scale


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D", SIZES)
def test_8bit(N, D, dtype, kind):
    x, residual, weight, _, _ = make(N, D, dtype, seed=N + D)
    quantised(x, residual, weight, kind)
    quantised(x, None, weight, kind)


@pytest.mark.parametrize("D", [70, 1024, 5000])
def test_odd_values(D):
    """Rows of zeros, of tiny and of huge numbers, one number in a row, a NaN or an infinity in one row only."""
    from panvram_amd import ops
    gen = torch.Generator().manual_seed(D)
    x = torch.randn(8, D, generator=gen)
    x[0] = 0
    x[1] *= 1e-18
    x[2] *= 1e18
    x[3] = 0
    x[3, D // 2] = 5.0
    weight = (1 + 0.1 * torch.randn(D, generator=gen)).cuda()
    ok = x.cuda()
    check(ok, torch.zeros_like(ok), weight, torch.randn(8, D, generator=gen).cuda(), torch.randn(8, D, generator=gen).cuda())
    for kind in (torch.float8_e4m3fn, torch.int8):
        q, scale = quantised(ok, None, weight, kind)
        assert float(scale[0]) == 0 and not q[0].float().any()
        for bad in (float("nan"), float("inf")):
            b = ok.clone()
            b[5, D - 1] = bad
            q2, scale2, _ = ops.add_rms_norm_8bit(b, None, weight, eps=EPS, dtype=kind)
            assert torch.isnan(scale2[5])
            assert torch.isnan(q2[5].float()).all() if kind == torch.float8_e4m3fn else not q2[5].any()
            keep = [0, 1, 2, 3, 4, 6, 7]
            assert torch.equal(q2[keep].float(), q[keep].float()) and torch.equal(scale2[keep], scale[keep])
            y, _ = ops.add_rms_norm(b, None, weight, eps=EPS)
            assert torch.isnan(y[5, D - 1]) and torch.isfinite(y[keep]).all()


def test_weight_of_another_type():
    """A bfloat16 weight is used in 32 bits; its gradient comes back in its type."""
    from panvram_amd import ops
    x, residual, weight, d_y, d_s = make(40, 256, torch.bfloat16, seed=4)
    w = weight.bfloat16().requires_grad_()
    y, stream = ops.add_rms_norm(x, residual, w, eps=EPS)
    (d,) = torch.autograd.grad((y, stream), (w,), (d_y, d_s))
    plain = P.norm(stream.cpu(), w.detach().float().cpu(), EPS, d_y.cpu(), d_s.cpu())
    assert d.dtype == torch.bfloat16
    P.inside(d, plain["d_weight"][0], plain["d_weight"][1] + P.rounded(plain["d_weight"][0], torch.bfloat16))


def test_one_output_wanted():
    from panvram_amd import ops
    x, residual, weight, d_y, d_s = make(20, 100, torch.float32, seed=5)
    a, b = x.clone().requires_grad_(), residual.clone().requires_grad_()
    y, stream = ops.add_rms_norm(a, b, weight, eps=EPS)
    plain = P.norm(stream.detach().cpu(), weight.cpu(), EPS, d_y.cpu(), None)
    got = torch.autograd.grad(y, (a, b), d_y, retain_graph=True)
    P.inside(got[1], plain["d"][0], plain["d"][1] + P.rounded(plain["d"][0], torch.float32))
    got = torch.autograd.grad(stream, (a, b), d_s)
    assert torch.equal(got[0], d_s) and torch.equal(got[1], d_s)


def test_gradients_against_differences():
    from panvram_amd import ops
    x, residual, weight, d_y, d_s = make(6, 40, torch.float32, seed=7)
    wanted = [t.clone().requires_grad_() for t in (x, residual, weight)]
    d = torch.autograd.grad(ops.add_rms_norm(*wanted, eps=EPS), wanted, (d_y, d_s))
    at = [t.double().cpu() for t in (x, residual, weight)]
    gen = torch.Generator().manual_seed(8)

    def value(a, b, w):
        s = a + b
        return float((s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * w * d_y.double().cpu()).sum() + (s * d_s.double().cpu()).sum())

    for k in range(3):
        way = torch.randn(at[k].shape, generator=gen, dtype=torch.float64)
        want = (value(*[t + 1e-5 * way if j == k else t for j, t in enumerate(at)]) - value(*[t - 1e-5 * way if j == k else t for j, t in enumerate(at)])) / 2e-5
        got = d[k].double().cpu()
        assert abs(float((got * way).sum()) - want) <= 1e-5 * float((got * way).abs().sum()) + 1e-6


def test_gradients_of_gradients_are_refused():
    """A graph of the gradients may be asked for (create_graph=True), but not differentiated."""
    from panvram_amd import ops
    x, _, weight, d_y, _ = make(4, 64, torch.float32, seed=6, residual=False)
    a = x.clone().requires_grad_()
    y, _ = ops.add_rms_norm(a, None, weight, eps=EPS)
    (plain,) = torch.autograd.grad(y, (a,), d_y, retain_graph=True)
    (d,) = torch.autograd.grad(y, (a,), d_y, create_graph=True)
    assert torch.equal(plain, d)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), (a,))


def test_empty():
    from panvram_amd import ops
    x = torch.zeros(0, 12, device="cuda", requires_grad=True)
    w = torch.ones(12, device="cuda", requires_grad=True)
    y, stream = ops.add_rms_norm(x, x, w)
    assert y.shape == (0, 12) and stream.shape == (0, 12)
    y.sum().backward()
    assert not w.grad.any()
    q, scale, _ = ops.add_rms_norm_8bit(x.detach(), None, w)
    assert q.shape == (0, 12) and scale.shape == (0,)


def test_capture():
    from panvram_amd import ops
    x, residual, weight, d_y, d_s = make(300, 1000, torch.bfloat16, seed=9)
    a, b, w = (t.clone().requires_grad_() for t in (x, residual, weight))

    def step():
        outs = ops.add_rms_norm(a, b, w, eps=EPS)
        return (*outs, *torch.autograd.grad(outs, (a, b, w), (d_y, d_s)), *(t.float() for t in ops.add_rms_norm_8bit(a, b, w, eps=EPS)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step()
    for k in range(4):
        with torch.no_grad():
            a.copy_(make(300, 1000, torch.bfloat16, seed=30 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step()))

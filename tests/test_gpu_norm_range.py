"""The norm of rows at either end of what the stream's type holds: finite rows whose squares leave 32 bits, up to the type's
largest value, and rows of the smallest numbers without an eps. Run with -m gpu."""
import pytest
import torch

from tests import ops_plain as P

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16]          # (float16's squares stay within 32 bits)


def compare(x, weight, eps, gradients=True):
    from panvram_amd import ops
    gen = torch.Generator().manual_seed(1)
    d_y = torch.randn(x.shape, generator=gen).to(x.dtype)
    a, w = x.cuda().requires_grad_(), weight.cuda().requires_grad_()
    y, _ = ops.add_rms_norm(a, None, w, eps=eps)
    plain = P.norm(x, weight, eps, d_y)
    P.inside(y, plain["y"][0], plain["y"][1] + P.rounded(plain["y"][0], x.dtype))
    if gradients:
        d = torch.autograd.grad(y, (a, w), d_y.cuda())
        P.inside(d[0], plain["d"][0], plain["d"][1] + P.rounded(plain["d"][0], x.dtype))
        P.inside(d[1], plain["d_weight"][0], plain["d_weight"][1] + P.rounded(plain["d_weight"][0], torch.float32))
    for kind, most in ((torch.float8_e4m3fn, 448.0), (torch.int8, 127.0)):
        q, scale, _ = ops.add_rms_norm_8bit(x.cuda(), None, weight.cuda(), eps=eps, dtype=kind)
        want, c = plain["y"][0], (x.shape[1] / 64 + 24) * P.U
        s = want.abs().amax(-1) / most
        P.inside(scale, s, c * s + 2.0 ** -149)
        v = torch.where(s[:, None] > 0, want / s[:, None], torch.zeros(()).double())
        half = torch.full_like(v, 0.5) if kind == torch.int8 else torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4)
        P.inside(q.float(), v, half * (1 + 1e-6) + 2 * c * v.abs())


def rows(D, dtype, *scales):
    gen = torch.Generator().manual_seed(D)
    return torch.cat([(torch.randn(1, D, generator=gen, dtype=torch.float64).clamp(-3.5, 3.5) * s) for s in scales]).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 1024, 4096, 70_000])
def test_large_rows(D, dtype):
    most = torch.finfo(dtype).max
    x = rows(D, dtype, 1.0, 1e18, 5e18, 1e19, 1e20, 1e30, 5e36, 1.5e37, most / 4, 1e-3)
    x = torch.cat([x, torch.full((1, D), most, dtype=dtype) * torch.where(torch.arange(D) % 3 == 0, -1, 1).to(dtype), torch.zeros(2, D, dtype=dtype)])
    x[-2, D // 3] = most
    weight = 1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(2))
    compare(x, weight, 1e-6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 1024, 70_000])
def test_small_rows(D, dtype):
    """Without an eps, and with one that is of the rows' own size."""
    weight = 1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(3))
    x = rows(D, dtype, 1.0, 1e-10, 1e-15, 1e-18, 1e-20, 1e-25, 1e-30, 1e-35)
    compare(x, weight, 0.0)
    for eps in (1e-10, 1e-18, 1e-20, 1e-21, 1e-30, 1e-36):
        compare(x, weight, eps)
    least = rows(D, dtype, 1e-37, 1e-38, 1e-39, 1e-40)
    compare(least, weight, 0.0, gradients=False)         # (1 / their root mean square is past 32 bits)


@pytest.mark.parametrize("dtype", TYPES)
def test_small_rows_and_weights(dtype):
    """8 bits, where the products of both leave 32 bits downwards."""
    x = rows(1000, dtype, 1e-12, 1e-20, 1e-30, 1e-36)
    weight = torch.randn(1000, generator=torch.Generator().manual_seed(4)) * 1e-18
    compare(x, weight, 0.0, gradients=False)

"""The norm over many tensors and clipping to it, against sums in 64 bits. Run with -m gpu."""
import math

import pytest
import torch

from tests import ops_plain as P

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def true_norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def check(grads, max_norm, apart):
    """In place, or into tensors of their own: the norm to one rounding, each gradient to its factor's three and its own."""
    from panvram_amd import ops
    before = [g.clone() for g in grads]
    want = true_norm(before)
    out = [torch.full_like(g, float("nan")) for g in grads] if apart else None
    assert abs(float(ops.gradient_norm(grads)) - want) <= 2 * P.U * want
    norm = ops.clip_gradients(grads, max_norm, out=out)
    assert norm.shape == () and norm.dtype == torch.float32 and abs(float(norm) - want) <= 2 * P.U * want
    factor = min(1.0, max_norm / (want + 1e-6))
    for b, g, o in zip(before, grads, out if apart else grads):
        w = b.double().cpu() * factor
        P.inside(o, w, 6 * P.U * w.abs() + P.rounded(w, o.dtype))
        if apart:
            assert torch.equal(b, g)


def make(sizes, seed, types=TYPES, std=0.1):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * std).to(types[i % len(types)]).cuda() for i, n in enumerate(sizes)]


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("sizes", [[1], [7], [0, 5, 0], [1 << 20], [100_003, 1, 2, 3, 64, 65, 255, 4097, 16384, 16385, 32769], [5] * 700, [300_001, 70_000] * 3])
def test_sizes(sizes, apart):
    for k, types in enumerate(([torch.float32], [torch.bfloat16], [torch.float16], TYPES)):
        check(make(sizes, len(sizes) + k, types), 0.05, apart)


@pytest.mark.parametrize("apart", [False, True])
def test_below_the_limit(apart):
    grads = make([1000, 33], 1, std=1e-4)
    before = [g.clone() for g in grads]
    check(grads, 10.0, apart)
    if not apart:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_shapes_and_strides():
    """Matrices, transposed ones, slices with gaps, starts off the wide loads' alignment, into other layouts."""
    from panvram_amd import ops
    gen = torch.Generator().manual_seed(2)
    for dtype in TYPES:
        n = lambda *s: torch.randn(*s, generator=gen).to(dtype).cuda()  # noqa: E731, B023
        grads = [n(30, 50), n(40, 20).t(), n(30, 90)[:, 11:60], n(1001)[1:], n(5, 6, 7).permute(2, 0, 1), n(()), n(1, 1), n(65)[::3]]
        check(grads, 0.5, False)
        grads = [n(30, 50), n(40, 20).t(), n(30, 90)[:, 11:60], n(1001)[1:], n(5, 6, 7).permute(2, 0, 1), n(())]
        check(grads, 0.5, True)
        flat = torch.zeros(30 * 50 + 17, dtype=dtype, device="cuda")
        a = n(50, 30)
        want = true_norm([a])
        ops.clip_gradients([a.t()], 0.5, out=[flat[17:].view(30, 50)])
        w = a.t().double().cpu() * (0.5 / (want + 1e-6))
        P.inside(flat[17:].view(30, 50), w, 6 * P.U * w.abs() + P.rounded(w, dtype))
        assert not flat[:17].any()
        wide = torch.zeros(30, 100, dtype=dtype, device="cuda")
        ops.clip_gradients([a.t()], 0.5, out=[wide[:, ::2]])
        P.inside(wide[:, ::2], w, 6 * P.U * w.abs() + P.rounded(w, dtype))
        assert not wide[:, 1::2].any()


def test_every_start_and_length():
    """Each start within 16 bytes and each short length: nothing before or behind is read into the norm or written."""
    from panvram_amd import ops
    for dtype in TYPES:
        room = torch.full((80,), float("nan"), dtype=dtype, device="cuda")
        for start in range(0, 9):
            for n in (1, 2, 3, 7, 8, 9, 15, 16, 17, 40):
                room[start:start + n] = 2.0
                norm = ops.clip_gradients([room[start:start + n]], 1.0)
                assert abs(float(norm) - 2 * math.sqrt(n)) <= 1e-5
                assert float((room[start:start + n].float() - 1 / math.sqrt(n)).abs().max()) <= 1e-2
                room[start:start + n] = float("nan")
                assert torch.isnan(room).all()


def test_far_values():
    """Squares that 32 bits could not hold, both ways; NaN and infinity reach the norm and the gradients."""
    from panvram_amd import ops
    big, tiny = torch.full((1000,), 1e30, device="cuda"), torch.full((1000,), 1e-30, device="cuda")
    assert abs(float(ops.gradient_norm([big])) / (1e30 * math.sqrt(1000)) - 1) <= 1e-6
    assert abs(float(ops.gradient_norm([tiny])) / (1e-30 * math.sqrt(1000)) - 1) <= 1e-6
    check([big.clone(), tiny.clone()], 1.0, False)
    for bad in (float("nan"), float("inf")):
        grads = make([100, 5000], 3, [torch.float32])
        grads[1][4321] = bad
        norm = ops.clip_gradients(grads, 1.0)
        assert not torch.isfinite(norm)
        assert not torch.isfinite(grads[1][4321])
    zero = [torch.zeros(500, device="cuda")]
    assert float(ops.clip_gradients(zero, 1.0)) == 0 and not zero[0].any()
    grads = make([100], 4, [torch.float32])
    ops.clip_gradients(grads, 0.0)
    assert not grads[0].any()


def test_generator_and_none():
    from panvram_amd import ops
    model = torch.nn.Linear(20, 30).cuda()
    model(torch.randn(5, 20, device="cuda")).square().sum().backward()
    want = true_norm([p.grad for p in model.parameters()])
    norm = ops.clip_gradients((p.grad for p in model.parameters() if p.grad is not None), 0.25)
    assert abs(float(norm) - want) <= 2 * P.U * want
    assert abs(true_norm([p.grad for p in model.parameters()]) - 0.25) <= 1e-5
    assert float(ops.clip_gradients([], 1.0)) == 0 and float(ops.gradient_norm([])) == 0


def test_capture():
    from panvram_amd import ops
    grads = make([70_001, 12, 300_000] * 50, 5)
    out = [torch.zeros_like(g) for g in grads]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = ops.clip_gradients(grads, 1.0, out=out)
    for k in range(4):
        for g in grads:
            g.mul_(1.0 + k)
        graph.replay()
        torch.cuda.synchronize()
        other = [torch.zeros_like(g) for g in grads]
        norm = ops.clip_gradients(grads, 1.0, out=other)
        assert torch.equal(norm, held) and all(torch.equal(a, b) for a, b in zip(out, other))


def test_large():
    """A tensor of over 2^31 elements."""
    from panvram_amd import ops
    n = (1 << 31) + 12345
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    g[-1] = 3.0
    want = math.sqrt((n - 1) * 0.25 + 9.0)
    norm = ops.clip_gradients([g], want / 2)
    assert abs(float(norm) - want) <= 2 * P.U * want
    assert float(g[-1]) == 1.5 and float(g[0]) == 0.25 and float((g[:-1] - 0.25).abs().max()) == 0

"""The gated recurrence against its definition in 64 bits (tests/ops_plain.py), its gradients against the formula's and
against differences. Run with -m gpu."""
import pytest
import torch

from tests import ops_plain as P

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(B, T, D, dtype, seed, state=True, reset=0.0, joined=False, mean=-1.0):
    gen = torch.Generator().manual_seed(seed)
    p = torch.randn(B, T, 2 * D, generator=gen)
    p[..., :D] = p[..., :D] * 2 + mean
    p = p.to(dtype).cuda()
    gate, value = p.chunk(2, -1)
    if not joined:
        gate, value = gate.contiguous(), value.contiguous()
    s = torch.randn(B, D, generator=gen).cuda() if state else None
    r = (torch.rand(B, T, generator=gen) < reset).cuda() if reset else None
    d_out = torch.randn(B, T, D, generator=gen).to(dtype).cuda()
    d_last = torch.randn(B, D, generator=gen).cuda()
    return gate, value, s, r, d_out, d_last


def cpu(*ts):
    return [None if t is None else t.detach().cpu() for t in ts]


def same(a, b):
    return torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)


def check(gate, value, state, reset, d_out=None, d_last=None):
    from panvram_amd import ops
    wanted = [t.detach().requires_grad_() for t in (gate, value, state) if t is not None]
    g, v = wanted[:2]
    s = wanted[2] if state is not None else None
    out, last = ops.gated_scan(g, v, state=s, reset=reset)
    plain = P.scan(*cpu(gate, value, state, reset, d_out, d_last))
    assert out.dtype == gate.dtype and out.shape == gate.shape and last.dtype == torch.float32
    got = {"out": out, "last": last}
    if d_out is not None:
        d = torch.autograd.grad((out, last), wanted, (d_out, d_last))
        got |= dict(zip(("d_gate", "d_value", "d_state"), d))
    for name, x in got.items():
        want, bound = plain[name]
        P.inside(x, want, bound + P.rounded(want, x.dtype))
    with torch.no_grad():
        again, last2 = ops.gated_scan(gate, value, state=state, reset=reset)
    assert same(again, out) and same(last2, last)      # with and without gradients: the same numbers


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (3, 1, 130), (2, 2, 64), (1, 15, 33), (2, 16, 128), (1, 17, 6), (2, 63, 65), (1, 64, 256), (3, 65, 10), (2, 127, 66),
                                   (1, 128, 500), (2, 129, 130), (1, 255, 64), (1, 257, 129), (2, 700, 40), (1, 2049, 70)])
def test_sizes(B, T, D, dtype):
    check(*make(B, T, D, dtype, seed=B * 10000 + T * 10 + D))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 40, 129, 600])
def test_resets_and_no_state(T, dtype):
    check(*make(2, T, 36, dtype, seed=T, state=False, reset=0.05))
    gate, value, state, _, d_out, d_last = make(2, T, 36, dtype, seed=T + 1)
    every = torch.ones(2, T, dtype=torch.uint8, device="cuda")
    check(gate, value, state, every, d_out, d_last)
    first = torch.zeros(2, T, dtype=torch.uint8, device="cuda")
    first[0, 0] = 7
    check(gate, value, state, first, d_out, d_last)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 65, 130])
def test_strided_inputs(D, dtype):
    """Halves of one projection, a transposed batch, every other channel, a gradient that is one number seen everywhere."""
    check(*make(2, 150, D, dtype, seed=D, joined=True))
    gate, value, state, _, d_out, d_last = make(3, 140, D, dtype, seed=D + 1)
    swap = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    check(swap(gate), value, state, None, swap(d_out), d_last)
    wide = torch.randn(3, 140, 2 * D, device="cuda").to(dtype)
    check(wide[..., ::2], wide[..., 1::2], state, None, d_out, d_last)
    check(gate, value, state, None, torch.full((1, 1, 1), 0.5, device="cuda", dtype=dtype).expand(3, 140, D), d_last)
    shifted = torch.randn(3 * 140 * D + 1, device="cuda").to(dtype)[1:].view(3, 140, D)
    check(shifted, value, state, None, d_out, d_last)


@pytest.mark.parametrize("dtype", TYPES)
def test_far_gates(dtype):
    """Gates that keep everything, drop everything, and infinite ones."""
    gate, value, state, _, d_out, d_last = make(2, 300, 70, dtype, seed=3)
    for far in (30.0, -30.0, 300.0, -300.0, float("inf"), float("-inf")):
        gate[:, ::7] = far
        check(gate, value, state, None, d_out, d_last)


def test_reset_stops_nan_and_infinity():
    """What stands before a reset reaches nothing behind it, forward, and nothing before it, backward."""
    from panvram_amd import ops
    for T, at in ((40, 20), (700, 333), (700, 640)):
        gate, value, state, _, d_out, d_last = make(1, T, 66, torch.float32, seed=T)
        reset = torch.zeros(1, T, dtype=torch.bool, device="cuda")
        reset[0, at] = True
        for bad in (float("nan"), float("inf")):
            v = value.clone()
            v[0, at - 3] = bad
            check(gate, v, state, reset)
            d = d_out.clone()
            d[0, at + 5] = bad
            g, w = gate.clone().requires_grad_(), value.clone().requires_grad_()
            out, _ = ops.gated_scan(g, w, state=state, reset=reset)
            dg, dw = torch.autograd.grad(out, (g, w), d)
            assert torch.isfinite(dg[0, :at]).all() and torch.isfinite(dw[0, :at]).all()
            assert not torch.isfinite(dw[0, at:at + 6]).any()


def test_continued_over_calls():
    """A sequence in pieces, the state handed on (generation's single steps among them), is the sequence in one."""
    from panvram_amd import ops
    gate, value, state, _, _, _ = make(2, 400, 96, torch.float32, seed=9)
    whole, end = ops.gated_scan(gate, value, state=state)
    s, parts, at = state, [], 0
    for n in (1, 1, 1, 130, 64, 1, 202):
        o, s = ops.gated_scan(gate[:, at:at + n], value[:, at:at + n], state=s)
        parts.append(o)
        at += n
    plain = P.scan(*cpu(gate, value, state))
    P.inside(torch.cat(parts, 1), plain["out"][0], plain["out"][1] + P.rounded(plain["out"][0], torch.float32))
    P.inside(s, end.double().cpu(), 2 * plain["last"][1] + P.rounded(plain["last"][0], torch.float32))


def test_gradients_against_differences():
    """d_gate, d_value and d_state against central differences of the 64-bit definition along random directions."""
    from panvram_amd import ops
    gate, value, state, reset, d_out, d_last = make(2, 90, 34, torch.float32, seed=5, reset=0.03)
    wanted = [t.clone().requires_grad_() for t in (gate, value, state)]
    d = torch.autograd.grad(ops.gated_scan(*wanted, reset=reset), wanted, (d_out, d_last))
    gen = torch.Generator().manual_seed(6)
    x = [t.double().cpu() for t in (gate, value, state)]
    for k in range(3):
        way = torch.randn(x[k].shape, generator=gen, dtype=torch.float64)
        at = []
        for h in (1e-4, -1e-4):
            y = [t + h * way if j == k else t for j, t in enumerate(x)]
            p = P.scan(*y, reset.cpu())
            at.append(float((p["out"][0] * d_out.double().cpu()).sum() + (p["last"][0] * d_last.double().cpu()).sum()))
        want, got = (at[0] - at[1]) / 2e-4, float((d[k].double().cpu() * way).sum())
        # the difference is good to h^2 times the third derivative (1e-8, of sums of 6,000 numbers of order 1), the gradient to 1e-5
        assert abs(got - want) <= 1e-5 * float((d[k].double().cpu() * way).abs().sum()) + 1e-5


def test_only_last_or_only_value_wanted():
    from panvram_amd import ops
    gate, value, state, _, _, d_last = make(2, 130, 20, torch.float32, seed=8)
    v = value.clone().requires_grad_()
    _, last = ops.gated_scan(gate, v, state=state)
    (d,) = torch.autograd.grad(last, (v,), d_last)
    want, bound = P.scan(*cpu(gate, value, state), None, torch.zeros(2, 130, 20), d_last.cpu())["d_value"]
    P.inside(d, want, bound + P.rounded(want, torch.float32))


def test_empty():
    from panvram_amd import ops
    for B, T, D in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        gate = torch.zeros(B, T, D, device="cuda", requires_grad=True)
        state = torch.randn(B, D, device="cuda")
        out, last = ops.gated_scan(gate, gate, state=state)
        assert out.shape == (B, T, D) and last.shape == (B, D)
        if T == 0:
            assert torch.equal(last, state)
        out.sum().backward()
        assert gate.grad is None or gate.grad.shape == gate.shape


def test_steps_far_apart():
    """Steps 128 MiB apart in memory."""
    room = torch.zeros(3, 1 << 26, dtype=torch.bfloat16, device="cuda")
    gate, value, state, _, _, _ = make(1, 3, 64, torch.bfloat16, seed=30)
    room[:, :64] = gate[0]
    check(room[None, :, :64], value, state, None)


def test_other_stream_and_capture():
    """On a stream of its own, and captured into a graph that is replayed on new inputs between eager work."""
    from panvram_amd import ops
    gate, value, state, reset, _, _ = make(2, 500, 130, torch.bfloat16, seed=12, reset=0.01)
    want = ops.gated_scan(gate, value, state=state, reset=reset)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.gated_scan(gate, value, state=state, reset=reset)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g, v = gate.clone(), value.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = ops.gated_scan(g, v, state=state, reset=reset)
    for k in range(4):
        more = make(2, 500, 130, torch.bfloat16, seed=20 + k)
        g.copy_(more[0])
        v.copy_(more[1])
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.gated_scan(g, v, state=state, reset=reset)
        assert torch.equal(held[0], eager[0]) and torch.equal(held[1], eager[1])


def test_long():
    """A sequence of many chunks per channel against the definition, and the last state of 3 * 2^20 steps."""
    check(*make(1, 40_000, 3, torch.float32, seed=15, reset=1e-4, mean=-4.0))
    check(*make(1, 33_000, 130, torch.bfloat16, seed=16, mean=-3.0))
    from panvram_amd import ops
    T = 3 << 20
    gate = torch.full((1, T, 2), -3.0, device="cuda")
    value = torch.ones(1, T, 2, device="cuda")
    out, last = ops.gated_scan(gate, value)
    assert float((last - 1).abs().max()) <= 1e-5 and float((out[0, -1] - 1).abs().max()) <= 1e-5

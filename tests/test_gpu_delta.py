"""ops.gated_delta and its gradients against the recurrence step by step in 64 bits."""
import pytest
import torch

from panvram_amd import ops
from tests.ops_plain_more import delta, delta_off, near

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("query", "key", "value", "gate", "write", "state")


def made(B, T, H, G, K, V, dtype, seed=0, state=True, reset=None, keep=-3.0, alike=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, std=1.0, mean=0.0, kind=dtype: torch.randn(*s, generator=gen, device="cuda").mul_(std).add_(mean).to(kind)  # noqa: E731
    a = dict(query=r(B, T, H, K, mean=alike), key=r(B, T, H, K, mean=alike), value=r(B, T, G, V), gate=r(B, T, G, mean=keep, std=1.5), write=r(B, T, G))
    a["state"] = r(B, G, K, V, std=0.5, kind=torch.float32) if state else None
    a["reset"] = torch.rand(B, T, generator=gen, device="cuda") < reset if reset else None
    return a, r(B, T, G, V, std=0.1), r(B, G, K, V, std=0.1, kind=torch.float32)


def wide(a):
    return {k: t if t is None or t.dtype in (torch.bool, torch.uint8) else t.detach().double().cpu() for k, t in a.items()} | (
        {"reset": a["reset"].cpu()} if a.get("reset") is not None else {})


def compare(a, d_out, d_last=None, skip=(), **more):
    """Outputs without gradients, then outputs and gradients"""
    dtype = a["query"].dtype
    ref = wide(a)
    leaves = {k: ref[k].requires_grad_() for k in NAMES if ref.get(k) is not None}
    out, last = delta(**ref, **more)
    with torch.no_grad():
        got = ops.gated_delta(**a, **more)
    near(got[0], out, delta_off("out", dtype), dtype)
    near(got[1], last, delta_off("last", dtype), torch.float32)
    a = {k: t.detach().requires_grad_() if k in leaves else t for k, t in a.items()}
    got = ops.gated_delta(**a, **more)
    near(got[0], out, delta_off("out", dtype), dtype)
    near(got[1], last, delta_off("last", dtype), torch.float32)
    ends, grads = [out], [d_out.double().cpu()]
    own, given = [got[0]], [d_out]
    if d_last is not None:
        ends, grads, own, given = ends + [last], grads + [d_last.double().cpu()], own + [got[1]], given + [d_last]
    want = torch.autograd.grad(ends, list(leaves.values()), grads)
    have = torch.autograd.grad(own, [a[k] for k in leaves], given)
    for k, w, h in zip(leaves, want, have):
        assert h.dtype == a[k].dtype
        if k not in skip:
            near(h, w, delta_off("d_" + k, dtype), a[k].dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 8, 9, 63, 64, 65, 127, 128, 200])
def test_lengths(dtype, T):
    a, d_out, d_last = made(2, T, 2, 2, 24, 40, dtype, seed=T)
    compare(a, d_out, d_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K, V", [(2, 1), (3, 5), (7, 31), (8, 32), (17, 33), (31, 64), (32, 16), (33, 72), (64, 130), (65, 96), (100, 17), (127, 129), (128, 128)])
def test_widths(dtype, K, V):
    a, d_out, d_last = made(1, 75, 1, 2, K, V, dtype, seed=K)
    compare(a, d_out, d_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_key_element(dtype):
    """A key of one element is 1 or -1: its own gradient is nothing but what roundings leave."""
    a, d_out, d_last = made(2, 70, 1, 2, 1, 6, dtype)
    compare(a, d_out, d_last, skip=("query", "key"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, G", [(1, 1), (1, 3), (2, 4), (3, 3), (3, 9)])
def test_shared_heads(dtype, H, G):
    a, d_out, d_last = made(2, 100, H, G, 20, 36, dtype, seed=G, reset=0.02)
    compare(a, d_out, d_last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("share", [0.01, 0.2, 1.0])
def test_resets(dtype, share):
    """Some, many in a chunk, and at every step"""
    a, d_out, d_last = made(3, 150, 1, 2, 16, 24, dtype, seed=5, reset=share)
    compare(a, d_out, d_last)
    a["reset"] = a["reset"].to(torch.uint8) * 7
    compare(a | {"state": None}, d_out)


@pytest.mark.parametrize("T, at", [(1, 0), (5, 0), (5, 3), (70, 0), (70, 1), (70, 40), (70, 64), (200, 130)])
def test_reset_drops_what_there_was(T, at):
    """A state that is not finite, under a reset at the first step or later: nothing before a reset matters behind it."""
    a, _, _ = made(2, T, 1, 1, 16, 24, torch.bfloat16)
    a["reset"] = torch.zeros(2, T, dtype=torch.bool, device="cuda")
    a["reset"][:, at] = True
    want = ops.gated_delta(**(a | {"state": None}))
    for fill in (float("nan"), float("inf"), -float("inf")):
        got = ops.gated_delta(**(a | {"state": torch.full_like(a["state"], fill)}))
        assert torch.equal(got[0][:, at:], want[0][:, at:]) and torch.equal(got[1], want[1])
        assert not torch.isfinite(got[0][:, :at]).any()
    one = a["state"].clone()                                    # one column of it, and one element
    one[0, 0, 3, 5] = float("nan")
    got = ops.gated_delta(**(a | {"state": one}))
    assert torch.equal(got[0][:, at:], want[0][:, at:]) and torch.equal(got[1], want[1])
    assert torch.isnan(got[0][0, :at, 0, 5]).all() and torch.isfinite(got[0][:, :at, :, :5]).all()


def test_packed_windows():
    """Windows packed behind each other, with resets, are the windows by themselves."""
    a, _, _ = made(1, 300, 2, 2, 32, 32, torch.float32, state=False)
    a["reset"] = torch.zeros(1, 300, dtype=torch.bool, device="cuda")
    cuts = [0, 50, 128, 129, 260, 300]
    a["reset"][0, cuts[1:-1]] = True
    out, last = ops.gated_delta(**a)
    for lo, hi in zip(cuts, cuts[1:]):
        o, s = ops.gated_delta(*(a[k][:, lo:hi] for k in NAMES[:5]))
        near(out[:, lo:hi], o, delta_off("out", torch.float32), torch.float32)
    near(last, s, delta_off("last", torch.float32), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_and_sequences(dtype):
    """A sequence at once, in two calls, and step by step: the state is carried along."""
    a, _, _ = made(2, 90, 2, 4, 48, 56, dtype)
    out, last = ops.gated_delta(**a)
    state, outs = a["state"], []
    for t in range(90):
        o, state = ops.gated_delta(*(a[k][:, t:t + 1] for k in NAMES[:5]), state=state)
        outs.append(o)
    near(torch.cat(outs, 1), out, 2 * delta_off("out", dtype), dtype)
    near(state, last, 2 * delta_off("last", dtype), torch.float32)
    o1, s = ops.gated_delta(*(a[k][:, :37] for k in NAMES[:5]), state=a["state"])
    o2, s = ops.gated_delta(*(a[k][:, 37:] for k in NAMES[:5]), state=s)
    near(torch.cat([o1, o2], 1), out, 2 * delta_off("out", dtype), dtype)
    near(s, last, 2 * delta_off("last", dtype), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate, write", [(-30.0, 30.0), (30.0, -3.0), (120.0, 0.0), (float("inf"), 2.0), (float("-inf"), float("inf")), (0.0, float("-inf"))])
def test_gates_at_their_ends(dtype, gate, write):
    """Everything kept, next to nothing kept (and exactly nothing), everything replaced, nothing written"""
    a, d_out, d_last = made(1, 80, 1, 2, 16, 24, dtype)
    a["gate"][:, ::2] = gate
    a["write"][:, ::3] = write
    compare(a, d_out, d_last)


@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_that_are_alike(dtype):
    """One key all along, nothing forgotten and everything replaced: sums of powers in place of the inverse would be lost here."""
    a, d_out, _ = made(1, 128, 1, 1, 32, 24, dtype, state=False)
    a["key"][:] = a["key"][:, :1]
    a["key"][:, 70:] = a["key"][:, :1] + (0.01 * torch.randn(1, 58, 1, 32, device="cuda")).to(dtype)
    a["gate"][:] = -20.0
    a["write"][:] = 6.0
    ref = wide(a)
    out, last = delta(**ref)
    got = ops.gated_delta(**a)
    near(got[0], out, 4 * delta_off("out", dtype), dtype)          # (a step's part of the sums is as large as the sums)
    near(got[1], last, 4 * delta_off("last", dtype), torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e25])
def test_sizes_of_values(dtype, size):
    """Values, states and gradients of any size: everything is linear in them."""
    a, d_out, d_last = made(1, 100, 1, 1, 24, 40, dtype)
    a["value"], a["state"] = (a["value"].float() * size).to(dtype), a["state"] * size
    d = (d_out.float() / size).to(dtype)
    compare(a, d, d_last / size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-15, 1e15])
def test_sizes_of_keys(dtype, size):
    """Lengths do not matter as long as their squares are float32 and above eps."""
    a, d_out, d_last = made(1, 100, 1, 1, 24, 40, dtype)
    for k in ("query", "key"):
        a[k] = (a[k].float() * size).to(dtype)
    compare(a, d_out, d_last, eps=0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_columns_of_different_sizes(dtype):
    """Each column of values by itself: its results are as exact as if the others were not there."""
    a, d_out, _ = made(1, 100, 1, 1, 24, 40, dtype)
    sizes = torch.logspace(-12, 12, 40, device="cuda")
    a["value"], a["state"] = (a["value"].float() * sizes).to(dtype), a["state"] * sizes
    d_out = (d_out.float() / sizes).to(dtype)
    ref = wide(a)
    leaves = {k: ref[k].requires_grad_() for k in NAMES}
    out, last = delta(**ref)
    b = {k: t.detach().requires_grad_() if k in leaves else t for k, t in a.items()}
    got = ops.gated_delta(**b)
    want = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), d_out.double().cpu())))
    have = dict(zip(leaves, torch.autograd.grad(got[0], [b[k] for k in leaves], d_out)))
    for c in range(40):
        near(got[0][..., c], out[..., c], delta_off("out", dtype), dtype)
        near(got[1][..., c], last[..., c], delta_off("last", dtype), torch.float32)
        near(have["value"][..., c], want["value"][..., c], delta_off("d_value", dtype), dtype)
        near(have["state"][..., c], want["state"][..., c], delta_off("d_state", dtype), torch.float32)
    for k in ("query", "key", "gate", "write"):
        near(have[k], want[k], delta_off("d_" + k, dtype), dtype)


def test_zero_keys():
    """A key of zeros reads and writes nothing; its gradient is finite."""
    a, d_out, d_last = made(1, 70, 1, 1, 16, 24, torch.float32)
    a["key"][:, ::2] = 0.0
    a["query"][:, 5] = 0.0
    compare(a, d_out, d_last, eps=1e-2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Parts of one projection, heads and steps in other orders, tensors that begin off 16 bytes, broadcast ones."""
    B, T, H, G, K, V = 2, 70, 2, 4, 19, 21
    a, d_out, d_last = made(B, T, H, G, K, V, dtype)
    joined = torch.randn(B, T, 2 * H * K + G * V + 3, device="cuda").to(dtype)[..., 3:]
    q, k, v = joined.split([H * K, H * K, G * V], -1)
    compare(a | dict(query=q.unflatten(-1, (H, K)), key=k.unflatten(-1, (H, K)), value=v.unflatten(-1, (G, V))), d_out)
    swapped = {n: a[n].transpose(1, 2).contiguous().transpose(1, 2) for n in NAMES[:5]}
    compare(a | swapped, d_out.transpose(1, 2).contiguous().transpose(1, 2), d_last)
    compare(a | dict(gate=a["gate"][:, :, :1].expand(B, T, G), write=a["write"][:1, :1].expand(B, T, G), key=a["key"].transpose(2, 3).contiguous().transpose(2, 3)), d_out)
    compare(a | dict(query=a["query"][:, :1].expand(B, T, H, K)), d_out[:, :1].expand(B, T, G, V), d_last)


def test_one_end_only():
    """Gradients from `last` alone, and of some inputs alone"""
    a, d_out, d_last = made(1, 90, 1, 2, 16, 24, torch.float32)
    ref = wide(a)
    leaves = [ref[k].requires_grad_() for k in ("key", "value")]
    want = torch.autograd.grad(delta(**ref)[1], leaves, d_last.double().cpu())
    b = a | {k: a[k].detach().requires_grad_() for k in ("key", "value")}
    have = torch.autograd.grad(ops.gated_delta(**b)[1], [b["key"], b["value"]], d_last)
    for h, w in zip(have, want):
        near(h, w, delta_off("d_key", torch.float32), torch.float32)


def test_against_differences():
    a, d_out, d_last = made(1, 70, 1, 2, 8, 8, torch.float32)
    names = list(NAMES)
    leaves = [a[k].requires_grad_() for k in names]

    def value(ts):
        out, last = ops.gated_delta(**dict(zip(names, ts)))
        return (out.double() * d_out).sum() + (last.double() * d_last).sum()
    got = torch.autograd.grad(value(leaves), leaves)
    h = 2.0 ** -7
    for j, g in enumerate(got):
        step = torch.randn(leaves[j].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(j))
        step /= step.norm()
        with torch.no_grad():
            at = lambda e: value([t + e * step if i == j else t for i, t in enumerate(leaves)])  # noqa: E731
            slope = (at(h) - at(-h)) / (2 * h)
        # a third derivative along a direction of length 1, and roundings of two sums of some 1,300 products of size 0.1
        assert abs(float(slope) - float((g * step).sum())) < 30 * h * h + 40 * 0.1 * 256 * 2.0 ** -24 / h


def test_empty():
    a, _, _ = made(2, 0, 1, 2, 8, 8, torch.float32)
    out, last = ops.gated_delta(**a)
    assert out.shape == (2, 0, 2, 8) and torch.equal(last, a["state"])
    a, _, _ = made(0, 5, 1, 2, 8, 8, torch.float32, state=False)
    out, last = ops.gated_delta(**a)
    assert out.shape == (0, 5, 2, 8) and last.shape == (0, 2, 8, 8)


def test_the_same_again():
    a, d_out, _ = made(3, 200, 2, 4, 64, 64, torch.bfloat16)
    b = {k: t.detach().requires_grad_() if k in NAMES else t for k, t in a.items()}

    def both():
        out, last = ops.gated_delta(**b)
        return (out, last, *torch.autograd.grad(out, [b[k] for k in NAMES], d_out))
    first = both()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, both()))
    with torch.no_grad():
        assert all(torch.equal(x, y) for x, y in zip(first, ops.gated_delta(**a)))


def test_captured():
    """Forwards and backwards in a graph, replayed on other inputs, between eager calls; and a single step."""
    a, d_out, _ = made(2, 130, 1, 2, 32, 40, torch.bfloat16)
    a = {k: t.detach().requires_grad_() if k in NAMES else t for k, t in a.items()}
    one = {k: t.detach()[:, :1] if k != "state" else t.detach() for k, t in a.items() if t is not None}

    def both():
        out, last = ops.gated_delta(**a)
        grads = torch.autograd.grad(out, [a[k] for k in NAMES], d_out)
        return (out.detach(), last.detach(), *grads, *ops.gated_delta(**one))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for k in range(3):
        with torch.no_grad():
            a["value"].copy_(torch.randn_like(a["value"]))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, both()):
            assert torch.equal(x, y)


def test_other_stream():
    a, _, _ = made(2, 300, 2, 2, 64, 64, torch.bfloat16)
    want = ops.gated_delta(**a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.gated_delta(**a)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_past_32_bit_offsets():
    """Values of over 2^31 elements: the last window of them, behind a reset, is what it is by itself."""
    T, G, K, V = (1 << 17) + 100, 128, 8, 128
    value = torch.randn(1, 1 << 12, G, V, device="cuda").bfloat16().repeat(1, (T >> 12) + 1, 1, 1)[:, :T]
    assert value.numel() > 1 << 31
    a = {k: torch.randn(1, T, 1, K, device="cuda").bfloat16() for k in ("query", "key")} | {"value": value}
    a |= {k: torch.randn(1, T, G, device="cuda").bfloat16() for k in ("gate", "write")}
    reset = torch.zeros(1, T, dtype=torch.bool, device="cuda")
    reset[:, T - 164] = True                    # the first step of a chunk
    assert (T - 164) % 64 == 0
    # The window has its reset by itself too. Without one its sums of log(keep) begin with log(keep[0]), not with 0; the differences of
    # two sums are those numbers again but rounded otherwise, 2^-24 of them, so that now and then an output is rounded the other way.
    with torch.no_grad():
        out, last = ops.gated_delta(**a, reset=reset)
        o, s = ops.gated_delta(**{k: t[:, T - 164:] for k, t in a.items()}, reset=reset[:, T - 164:])
    assert torch.equal(out[:, T - 164:], o) and torch.equal(last, s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, H, G, K, V, reset", [(2048, 1, 1, 12, 10, None), (2113, 1, 2, 9, 40, 0.002), (3000, 1, 1, 33, 8, None), (1600, 35, 70, 12, 10, 0.001)])
def test_in_pieces(dtype, T, H, G, K, V, reset):
    """Long sequences of few heads, which are walked in pieces: their starts, ends and gradients"""
    a, d_out, d_last = made(1, T, H, G, K, V, dtype, seed=T, reset=reset, keep=-6.0)
    compare(a, d_out, d_last)


@pytest.mark.parametrize("at", [0, 1000, 2047])
def test_reset_in_a_piece(at):
    """A state that is not finite, dropped somewhere in a long sequence, reaches nothing from there on."""
    a, _, _ = made(1, 2100, 1, 1, 16, 24, torch.bfloat16)
    a["reset"] = torch.zeros(1, 2100, dtype=torch.bool, device="cuda")
    a["reset"][:, at] = True
    want = ops.gated_delta(**(a | {"state": None}))
    got = ops.gated_delta(**(a | {"state": torch.full_like(a["state"], float("nan"))}))
    assert torch.equal(got[0][:, at:], want[0][:, at:]) and torch.equal(got[1], want[1])
    if at > 64:
        assert torch.isnan(got[0][:, :at]).all()


def test_pieces_captured():
    a, d_out, _ = made(1, 2200, 1, 2, 16, 24, torch.bfloat16)
    a = {k: t.detach().requires_grad_() if k in NAMES else t for k, t in a.items()}

    def both():
        out, last = ops.gated_delta(**a)
        return (out.detach(), last.detach(), *torch.autograd.grad(out, [a[k] for k in NAMES], d_out))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for k in range(3):
        with torch.no_grad():
            a["value"].copy_(torch.randn_like(a["value"]))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, both()))


@pytest.mark.parametrize("T, H, G, K, V", [(1, 2, 2, 24, 40), (200, 1, 2, 24, 40), (2113, 1, 1, 17, 9)])
def test_memory_that_held_something(T, H, G, K, V):
    """Workspaces and records that lie where NaN lay: nothing is read before it is written."""
    a, d_out, d_last = made(2, T, H, G, K, V, torch.bfloat16)
    leaves = [a[k].requires_grad_() for k in NAMES]

    def run():
        got = ops.gated_delta(**a)
        with torch.no_grad():
            alone = ops.gated_delta(**a)
        return [*(t.clone() for t in (*got, *alone)), *torch.autograd.grad(got, leaves, (d_out, d_last))]

    first = run()
    held = [torch.full((size,), float("nan"), device="cuda") for size in [1 << 22] * 8 + [1 << 16] * 64 + [1 << 10] * 64]
    del held
    for x, y in zip(first, run()):
        assert torch.isfinite(x).all() and torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T, K, V", [(2, 38, 109), (300, 16, 25), (1300, 24, 64)])
def test_only_outputs_are_rounded(dtype, T, K, V):
    """Outputs and gradients in 16 bits are off by little more than what rounding them alone would be. That is spread evenly over
    half a step to both sides, a root mean square of eps / sqrt(12) of the value where mantissas are all 1, the worst that they can
    be. On top of it 5 % for the count of elements, and 0.3 of it, in squares, in bfloat16: one of narrow operands' 11 bits is off by
    1 / 8 of bfloat16's step at most, and an output is made from four."""
    a, d_out, d_last = made(2, T, 2, 4, K, V, dtype, seed=7)
    ref = wide(a)
    leaves = {k: ref[k].requires_grad_() for k in NAMES}
    want = [*delta(**ref)]
    want += torch.autograd.grad(want, list(leaves.values()), [d_out.double().cpu(), d_last.double().cpu()])
    b = a | {k: a[k].detach().requires_grad_() for k in NAMES}
    have = [*ops.gated_delta(**b)]
    have += torch.autograd.grad(have, [b[k] for k in NAMES], [d_out, d_last])
    with torch.no_grad():
        have.append(ops.gated_delta(**a)[0])
        want.append(want[0])
    most = 1.05 * torch.finfo(dtype).eps / 12 ** 0.5 * (1.3 ** 0.5 if dtype == torch.bfloat16 else 1.0)
    for name, h, w in zip(("out", "last", *(f"d_{k}" for k in NAMES), "alone"), have, want):
        if h.dtype == dtype and h.numel() > 1000:
            off = float((h.double().cpu() - w).norm() / w.norm())
            assert off <= most, (name, off, most)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K, V", [(20, 700), (128, 517)])
def test_wide_values(dtype, K, V):
    """More columns of values than the gradients' lanes look at in one turn"""
    a, d_out, d_last = made(1, 70, 1, 2, K, V, dtype, reset=0.02)
    compare(a, d_out, d_last)

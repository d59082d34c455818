"""The head and loss of the next base against the definition in 64 bits (tests/ops_plain.py), and the gradients against the
formula's and against differences. Run with -m gpu."""
import pytest
import torch

from tests import ops_plain as P

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(B, T, D, V, dtype, seed, wtype=None, ignored=0.1):
    gen = torch.Generator().manual_seed(seed)
    hidden = torch.randn(B, T, D, generator=gen).to(dtype).cuda()
    weight = (torch.randn(V, D, generator=gen) * D ** -0.5 * 2).to(wtype or dtype).cuda()
    tokens = torch.randint(V, (B, T), generator=gen, dtype=torch.uint8)
    tokens[torch.rand(B, T, generator=gen) < ignored] = 4
    return hidden, weight, tokens.cuda()


def check(hidden, weight, tokens, ignore=4):
    from panvram_amd import ops
    plain = P.loss(hidden.detach().cpu(), weight.detach().cpu(), tokens.cpu(), ignore)

    def near(name, got, dtype, plain=plain):
        want, bound = plain[name]
        P.inside(got, want, bound + P.rounded(want, dtype))

    loss, dh, dw = ops.next_base_loss_grad(hidden, weight, tokens, ignore=ignore)
    assert dh.dtype == hidden.dtype and dw.dtype == weight.dtype and dh.shape == hidden.shape and loss.shape == ()
    near("loss", loss, torch.float32)
    near("d_hidden", dh, hidden.dtype)
    near("d_weight", dw, weight.dtype)
    near("each", ops.next_base_loss(hidden, weight, tokens, ignore=ignore, reduction="none"), torch.float32)
    near("loss", ops.next_base_loss(hidden, weight, tokens, ignore=ignore), torch.float32)
    h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    d = torch.autograd.grad(ops.next_base_loss(h, w, tokens, ignore=ignore), (h, w))
    near("d_hidden", d[0], hidden.dtype)
    near("d_weight", d[1], weight.dtype)
    gen = torch.Generator().manual_seed(1)
    factor = torch.randn(tokens.shape, generator=gen)
    d = torch.autograd.grad(ops.next_base_loss(h, w, tokens, ignore=ignore, reduction="none"), (h, w), factor.cuda())
    plain = P.loss(hidden.detach().cpu(), weight.detach().cpu(), tokens.cpu(), ignore, factor=factor)
    near("d_hidden", d[0], hidden.dtype, plain)
    near("d_weight", d[1], weight.dtype, plain)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D,V", [(1, 2, 1, 1), (1, 1, 5, 4), (2, 3, 7, 2), (1, 17, 64, 4), (3, 16, 32, 5), (2, 65, 100, 5), (2, 129, 128, 16), (1, 300, 500, 12),
                                     (5, 33, 512, 5), (1, 70, 1000, 16), (2, 100, 1024, 5), (1, 40, 2048, 9), (1, 19, 4100, 7), (1, 33, 8192, 16), (1, 5000, 24, 6)])
def test_sizes(B, T, D, V, dtype):
    check(*make(B, T, D, V, dtype, seed=B * 1000 + T + D + V))


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("D,V", [(60, 5), (512, 5), (1024, 16), (3000, 3)])
def test_weight_in_32_bits(D, V, dtype):
    check(*make(2, 77, D, V, dtype, seed=D, wtype=torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens(dtype):
    """No place counts; one does; int64 ids, some outside the alphabet; nothing ignored; a row of the ignored id."""
    hidden, weight, tokens = make(2, 40, 96, 5, dtype, seed=2)
    check(hidden, weight, torch.full_like(tokens, 4))
    one = torch.full_like(tokens, 4)
    one[1, 17] = 2
    check(hidden, weight, one)
    first = torch.full_like(tokens, 4)
    first[:, 0] = 1                                  # nothing predicts the first token of a row
    check(hidden, weight, first)
    ids = tokens.long()
    ids[0, 5], ids[0, 6], ids[1, 7], ids[1, 8] = -1, 5, 1 << 40, -(1 << 40)
    check(hidden, weight, ids, ignore=None)
    check(hidden, weight, tokens, ignore=None)
    check(hidden, weight, tokens, ignore=2)
    tokens[0] = 4
    check(hidden, weight, tokens)
    check(*make(3, 1, 64, 4, dtype, seed=3))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 65, 520])
def test_strided(D, dtype):
    hidden, weight, tokens = make(3, 70, 2 * D, 5, dtype, seed=D)
    check(hidden[:, :, :D], weight[:, :D], tokens)
    check(hidden[:, 5:45, 1:D + 1], weight[:, 1:D + 1], tokens[:, 5:45])
    check(hidden[..., ::2], weight[:, ::2], tokens)
    check(hidden[..., :D].transpose(0, 1).contiguous().transpose(0, 1), weight[:, :D], tokens.t().contiguous().t())
    shifted = torch.randn(3 * 70 * D + 1, device="cuda").to(dtype)[1:].view(3, 70, D)
    check(shifted, weight[:, :D], tokens)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,V", [(60, 5), (512, 16), (2100, 4)])
def test_factors_of_all_sizes(D, V, dtype):
    """Gradients of the places' losses from 2^-40 to 2^12, rising and falling: none is lost beside a larger one, and sums that
    began small go on as large ones."""
    from panvram_amd import ops
    hidden, weight, tokens = make(2, 900, D, V, dtype, seed=D)
    tokens %= V
    rising = torch.exp2(torch.linspace(-40, 12, 1800)).view(2, 900)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    for factor in (rising, rising.flip(0, 1), torch.where(torch.arange(1800).view(2, 900) % 3 == 0, rising, 0)):
        d = torch.autograd.grad(ops.next_base_loss(h, w, tokens, ignore=None, reduction="none"), (h, w), factor.cuda())
        plain = P.loss(hidden.detach().cpu(), weight.detach().cpu(), tokens.cpu(), None, factor=factor)
        for got, name in zip(d, ("d_hidden", "d_weight")):
            P.inside(got, plain[name][0], plain[name][1] + P.rounded(plain[name][0], dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [60, 512])
def test_nothing_from_places_that_do_not_count(D, dtype):
    """NaN and infinities in hidden where no next token counts leave the loss and both gradients as they are."""
    from panvram_amd import ops
    hidden, weight, tokens = make(2, 90, D, 5, dtype, seed=D)
    idle = torch.ones(2, 90, dtype=torch.bool, device="cuda")
    idle[:, :-1] = tokens[:, 1:] == 4
    assert idle.sum() > 4
    want = ops.next_base_loss_grad(hidden, weight, tokens)
    each = ops.next_base_loss(hidden, weight, tokens, reduction="none")
    for bad in (float("nan"), float("inf"), float("-inf")):
        h = hidden.clone()
        h[idle] = bad
        got = ops.next_base_loss_grad(h, weight, tokens)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert not got[1][idle].any()
        assert torch.equal(ops.next_base_loss(h, weight, tokens, reduction="none"), each)
    h = hidden.clone()
    h[0, 3] = float("nan")
    tokens[0, 4] = 1
    assert torch.isnan(ops.next_base_loss(h, weight, tokens))


def test_large_logits():
    """Logits of +-1000: the largest is taken off before the exponentials."""
    hidden, weight, tokens = make(2, 60, 128, 5, torch.float32, seed=6)
    check(hidden * 300, weight, tokens)


def test_scale():
    from panvram_amd import ops
    hidden, weight, tokens = make(2, 50, 64, 5, torch.float32, seed=7)
    s = torch.tensor([1024.0], device="cuda")
    a, b = ops.next_base_loss_grad(hidden, weight, tokens), ops.next_base_loss_grad(hidden, weight, tokens, scale=s)
    assert torch.equal(a[0], b[0])
    assert torch.allclose(a[1] * 1024, b[1], rtol=1e-6, atol=0) and torch.allclose(a[2] * 1024, b[2], rtol=1e-5, atol=1e-6)
    h = hidden.clone().requires_grad_()
    (ops.next_base_loss(h, weight, tokens) * 1024).backward()
    assert torch.equal(h.grad, b[1])


def test_gradients_against_differences():
    from panvram_amd import ops
    hidden, weight, tokens = make(2, 30, 20, 5, torch.float32, seed=8)
    _, dh, dw = ops.next_base_loss_grad(hidden, weight, tokens)
    x = [hidden.double().cpu(), weight.double().cpu()]
    gen = torch.Generator().manual_seed(9)
    for k, got in enumerate((dh, dw)):
        way = torch.randn(x[k].shape, generator=gen, dtype=torch.float64)
        up, down = ([t + h * way if j == k else t for j, t in enumerate(x)] for h in (1e-5, -1e-5))
        want = (float(P.loss(*up, tokens.cpu(), 4)["loss"][0]) - float(P.loss(*down, tokens.cpu(), 4)["loss"][0])) / 2e-5
        got = got.double().cpu()
        assert abs(float((got * way).sum()) - want) <= 1e-5 * float((got * way).abs().sum()) + 1e-7


def test_same_from_run_to_run_and_captured():
    """The sums have a fixed order: equal bits each time, and from a replayed graph."""
    from panvram_amd import ops
    hidden, weight, tokens = make(3, 2000, 256, 5, torch.bfloat16, seed=10)
    want = ops.next_base_loss_grad(hidden, weight, tokens)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, ops.next_base_loss_grad(hidden, weight, tokens)))
    h = hidden.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = ops.next_base_loss_grad(h, weight, tokens)
    for k in range(4):
        h.copy_(make(3, 2000, 256, 5, torch.bfloat16, seed=40 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, ops.next_base_loss_grad(h, weight, tokens)))

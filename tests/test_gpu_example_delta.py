"""The model with matrices as its states, as a program strings the operators together: its gradients, packed windows, bases one by
one, and what dropout does and does not do."""
import pytest
import torch
import torch.nn.functional as F

from examples import train_delta as E
from panvram_amd import Cohort, ops
from tests.ops_plain import UNIT
from tests.ops_plain_more import delta, kept

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cohort(mini):
    return Cohort.open(mini["dir"], device="cuda", dataset="q4k", reference=mini["ref"])


def small():
    torch.manual_seed(0)
    return E.Model(width=64, depth=2, heads=2, size=32).cuda()


def test_runs(cohort):
    model = small()
    losses = E.train(cohort, model, 3, rows=4, window=300)
    assert len(losses) == 3 and all(0 < x < 20 for x in losses)
    assert all(torch.isfinite(p.grad).all() and bool((p.grad != 0).any()) for p in model.parameters())
    made = E.generate(model, cohort.sample(2, 300, tokens=True), 5, torch.Generator(device="cuda").manual_seed(1))
    assert made.shape == (2, 5) and int(made.max()) < 4


def plain(model, tokens, reset, seed):
    """The loss of the example's step in float64 on the CPU, weights as the model's"""
    w = {k: p.detach().double().cpu().requires_grad_() for k, p in model.named_parameters()}
    B, T = tokens.shape
    drop = lambda x, site: (lambda m, up: torch.where(m.view(x.shape), x * up, 0.0))(*kept(x.numel(), model.drop, seed, site))  # noqa: E731
    stream = drop(w["embed"][tokens.long()], 0)
    step = None
    width = stream.shape[-1]
    for k in range(3):
        if step is not None:
            stream = stream + drop(step, k)
        y = F.layer_norm(stream, (width,), w[f"norms.{k}"], w[f"shifts.{k}"], 1e-5)
        if k == 2:
            break
        parts = (y @ w[f"inward.{k}"].T).view(B, T, model.heads, -1)
        q, key, v, gates = parts.split([model.size] * 3 + [2], -1)
        h, _ = delta(q, key, v, gates[..., 0] + w[f"keep.{k}"], gates[..., 1], reset=reset)
        step = h.flatten(2) @ w[f"outward.{k}"].T
    logits = y @ w["head"].T
    half = T // 2
    logits, targets = logits.view(2 * B, half, 4)[:, :-1], tokens.view(2 * B, half)[:, 1:].long()
    counts = targets < 4
    return F.cross_entropy(logits[counts], targets[counts]), w


def test_gradients():
    """All of the model's gradients against the same model in float64. Activations are bfloat16: some 12 of them between the loss and
    the first weight each way, each off by half a step, 2^-8, at most, and as large as what is added to them."""
    model = small()
    gen = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randint(4, (3, 200), generator=gen, device="cuda", dtype=torch.uint8)
    tokens[0, 17] = 4
    reset = torch.zeros(3, 200, dtype=torch.bool, device="cuda")
    reset[:, 100] = True
    seed = torch.tensor([77], device="cuda")
    hidden, _ = model(tokens, reset=reset, seed=seed)
    loss = ops.next_base_loss(hidden.view(6, 100, -1), model.head, tokens.view(6, 100))
    loss.backward()
    want, w = plain(model, tokens.cpu(), reset.cpu(), 77)
    want.backward()
    assert abs(float(loss.detach()) - float(want)) <= 24 * UNIT[torch.bfloat16] * float(want)
    for k, p in model.named_parameters():
        off = float((p.grad.double().cpu() - w[k].grad).norm() / w[k].grad.norm())
        assert off <= 24 * UNIT[torch.bfloat16], (k, off)


def test_windows_of_a_row_do_not_meet():
    """The second window of a row is what it is alone, in hidden states, but for the roundings of the library's products, which go by
    their number of rows: 12 activations, each off by half a step."""
    model = small()
    tokens = torch.randint(4, (2, 256), device="cuda", dtype=torch.uint8)
    reset = torch.zeros(2, 256, dtype=torch.bool, device="cuda")
    reset[:, 128] = True
    with torch.no_grad():
        both, states = model(tokens, reset=reset)
        alone, last = model(tokens[:, 128:])
    assert float((both[:, 128:].float() - alone.float()).norm() / alone.float().norm()) <= 12 * UNIT[torch.bfloat16]
    for a, b in zip(states, last):
        assert float((a - b).norm() / b.norm()) <= 12 * UNIT[torch.bfloat16]


def test_one_by_one():
    """Bases one by one, with the states carried along, are the sequence at once."""
    model = small()
    tokens = torch.randint(4, (3, 80), device="cuda", dtype=torch.uint8)
    with torch.no_grad():
        want, last = model(tokens)
        states, got = None, []
        for t in range(80):
            h, states = model(tokens[:, t:t + 1], states=states)
            got.append(h)
    got = torch.cat(got, 1)
    assert float((got.float() - want.float()).norm() / want.float().norm()) <= 12 * UNIT[torch.bfloat16]
    for a, b in zip(states, last):
        assert float((a - b).norm() / b.norm()) <= 12 * UNIT[torch.bfloat16]


def test_seeds():
    """The same seed drops the same, another one something else, and none nothing."""
    model = small()
    tokens = torch.randint(4, (2, 100), device="cuda", dtype=torch.uint8)
    with torch.no_grad():
        a, b, c, d = (model(tokens, seed=s)[0] for s in (5, 5, 6, None))
    assert torch.equal(a, b) and not torch.equal(a, c) and not torch.equal(a, d)

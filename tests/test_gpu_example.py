"""examples/train_recurrent.py: the operators together on a cohort's windows. Run with -m gpu."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cohort(mini):
    import panvram_amd
    return panvram_amd.Cohort.open(mini["dir"], device="cuda", dataset=None, reference=mini["ref"])


def test_training_learns(cohort):
    """The loss falls below what the bases' frequencies alone give (2 bits), with finite gradients throughout."""
    import train_recurrent as E
    torch.manual_seed(0)
    model = E.Model(width=128, depth=2).cuda()
    losses = E.train(cohort, model, 60, rows=8, window=1000)
    assert all(math.isfinite(x) for x in losses)
    assert sum(losses[-10:]) / 10 < 2.0 < losses[0]


def test_pieces_and_single_bases(cohort):
    """A window in one call, in pieces with the states carried on, and its bases one by one give the same hidden values to
    bfloat16's rounding of the activations; a packed window's second half is not changed by its first."""
    import train_recurrent as E
    torch.manual_seed(1)
    model = E.Model(width=64, depth=2).cuda()
    tokens, reset = E.batch(cohort, 2, 150, torch.Generator(device="cuda").manual_seed(2))
    with torch.no_grad():
        whole, end = model(tokens)
        first, states = model(tokens[:, :100])
        second, states = model(tokens[:, 100:299], states=states)
        third, states = model(tokens[:, 299:], states=states)
        parts = torch.cat([first, second, third], 1)
        # (two blocks of bfloat16 activations: a difference of one rounding, 2^-8, may pass through a handful of them)
        assert float((parts.float() - whole.float()).norm() / whole.float().norm()) <= 2.0 ** -7
        assert all(float((a - b).norm() / b.norm()) <= 2.0 ** -7 for a, b in zip(states, end))
        packed, _ = model(tokens, reset=reset)
        alone, _ = model(tokens[:, 150:])
        assert float((packed[:, 150:].float() - alone.float()).norm() / alone.float().norm()) <= 2.0 ** -7
        one = E.generate(model, tokens, 20, torch.Generator(device="cuda").manual_seed(3))
        again = E.generate(model, tokens, 20, torch.Generator(device="cuda").manual_seed(3))
        assert one.shape == (2, 20) and torch.equal(one, again) and int(one.max()) < 4
        bits = E.score(model, tokens)
        assert bits.shape == tokens.shape and torch.isfinite(bits).all() and not bits[:, -1].any()

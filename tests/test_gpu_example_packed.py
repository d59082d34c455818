"""examples/train_recurrent.py on packed windows: no window's last place is trained on another window's first base. Run with
-m gpu."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


def test_loss_of_packed_windows(mini):
    """Windows of six bases: a step's loss is the mean over both windows' own places, as of the windows one to a row."""
    import math

    import panvram_amd
    import train_recurrent as E
    cohort = panvram_amd.Cohort.open(mini["dir"], device="cuda", dataset=None, reference=mini["ref"])
    torch.manual_seed(0)
    model = E.Model(width=64, depth=1).cuda()
    tokens, _ = E.batch(cohort, 16, 6, torch.Generator(device=cohort.device).manual_seed(0))
    with torch.no_grad():
        hidden, _ = model(tokens.view(32, 6))
        logits = torch.nn.functional.linear(hidden[:, :-1].double(), model.head.double())
        target = tokens.view(32, 6)[:, 1:].long()
        want = torch.nn.functional.cross_entropy(logits[target < 4], target[target < 4]) / math.log(2)
    (got,) = E.train(cohort, model, 1, rows=16, window=6)
    # one bfloat16 rounding of a few activations between the two shapes of the same products; the places of the windows'
    # ends, 16 of 176, would move the mean by some hundredths
    assert abs(got - float(want)) <= 2e-3 * float(want)

"""The gated scan's sigmoid in 32 bits: as good far from zero as near it. Run with -m gpu."""
import pytest
import torch

from tests import ops_plain as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40, 300])
def test_gates_far_from_zero(T):
    """One step's z value and (1 - z) state, each by itself: a reset at every step (out = z value), and values of zero (out =
    the product of 1 - z, of one step here: the others have gates that keep the state whole, 1 - z = 1). z and 1 - z to nine
    last places: two for 2^t and one for its correction, one for 1 + e, two for the reciprocal, one for their product, two
    for what r leaves out; and one for the product with value or state."""
    from panvram_amd import ops
    gen = torch.Generator().manual_seed(T)
    gate = (torch.rand(3, T, 70, generator=gen) * 160 - 80).cuda()
    value = torch.randn(3, T, 70, generator=gen).cuda()
    every = torch.ones(3, T, dtype=torch.bool, device="cuda")
    out, _ = ops.gated_scan(gate, value, reset=every)
    want = torch.sigmoid(gate.double()) * value.double()
    assert float(((out.double() - want).abs() / want.abs()).max()) <= 10 * P.U
    keeping = torch.full_like(gate, -200.0)
    at = T // 2
    keeping[:, at] = gate[:, at]
    state = torch.randn(3, 70, generator=gen).cuda()
    _, last = ops.gated_scan(keeping, torch.zeros_like(value), state=state)
    want = torch.sigmoid(-gate[:, at].double()) * state.double()
    assert float(((last.double() - want).abs() / want.abs()).max()) <= 10 * P.U

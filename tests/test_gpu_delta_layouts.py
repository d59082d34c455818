"""ops.gated_delta on layouts whose strides say little: of one step, of one sequence, of one head."""
import pytest
import torch

from panvram_amd import ops
from tests.test_gpu_delta import NAMES, made

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("train", [False, True])
def test_one_step_of_many_sequences(train):
    """Time-first tensors of one step, whose step is over 2^22 elements long: no stride of it is used."""
    B, H, K, V = 8200, 4, 128, 130
    a, d_out, _ = made(B, 1, H, H, K, V, torch.bfloat16, state=False)
    first = {k: t.transpose(0, 1).contiguous().transpose(0, 1) for k, t in a.items() if t is not None}
    # (as a slice of a longer sequence has it; torch takes any stride of one step for contiguous)
    for k in ("query", "key", "value"):
        longer = torch.zeros(2, *first[k].transpose(0, 1).shape[1:], dtype=torch.bfloat16, device="cuda")
        longer[:1] = first[k].transpose(0, 1)
        first[k] = longer[:1].transpose(0, 1)
        assert first[k].stride(1) > 1 << 22 and first[k].contiguous().stride(1) > 1 << 22
    if not train:
        assert all(torch.equal(x, y) for x, y in zip(ops.gated_delta(**first), ops.gated_delta(**a)))
        return
    d_first = torch.zeros(2, *d_out.transpose(0, 1).shape[1:], dtype=torch.bfloat16, device="cuda")
    d_first[:1] = d_out.transpose(0, 1)
    d_first = d_first[:1].transpose(0, 1)
    assert d_first.contiguous().stride(1) > 1 << 22
    got = []
    for tensors, d in ((first, d_first), (a, d_out)):
        leaves = [tensors[k].detach().requires_grad_() for k in NAMES[:5]]
        out, last = ops.gated_delta(*leaves)
        got.append((out.detach(), last.detach(), *torch.autograd.grad(out, leaves, d)))
    assert all(torch.equal(x, y) for x, y in zip(*got))


def test_one_of_everything():
    """Strides of dimensions of size 1 that mean nothing"""
    a, _, _ = made(1, 70, 1, 1, 24, 40, torch.bfloat16, state=False)
    odd = {k: t.as_strided(t.shape, (7, t.stride(1), 11, 1)[:t.dim()]) for k, t in a.items() if t is not None}
    assert all(torch.equal(x, y) for x, y in zip(ops.gated_delta(**odd), ops.gated_delta(**a)))
    one = {k: t[:, :1].as_strided(t[:, :1].shape, (7, 1 << 40, 11, 1)[:t.dim()]) for k, t in a.items() if t is not None}
    assert all(torch.equal(x, y) for x, y in zip(ops.gated_delta(**one), ops.gated_delta(**{k: t[:, :1] for k, t in a.items() if t is not None})))

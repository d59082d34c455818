"""The definition of dropout's bits that the GPU tests compare with, against the generator's published known answers (Salmon,
Moraes, Dror, Shaw 2011, ten rounds of four words), and its statistics. Runs without a GPU."""
import pytest

from tests.ops_plain_more import kept, words

PI = (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)


@pytest.mark.parametrize("counter, key, want", [
    ((0,) * 4, (0,) * 2, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    (*PI, (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))])
def test_known_answers(counter, key, want):
    assert tuple(int(w) for w in words(counter, key)) == want


@pytest.mark.parametrize("p", [0.02, 0.5, 0.9])
def test_share(p):
    """Within six standard deviations, for two seeds and two sites; different ones drop differently."""
    n = 1 << 16
    masks = [kept(n, p, seed, site)[0] for seed in (1, 1 << 63) for site in (0, 7)]
    for m in masks:
        assert abs(int(m.sum()) - n * (1 - p)) < 6 * (n * p * (1 - p)) ** 0.5
    assert all((a != b).any() for i, a in enumerate(masks) for b in masks[:i])


def test_all_and_none():
    assert not kept(100, 1.0, 3)[0].any() and kept(100, 0.0, 3)[0].all()
    assert kept(40, 0.5, 3, first=100)[0].tolist() == kept(140, 0.5, 3)[0][100:].tolist()

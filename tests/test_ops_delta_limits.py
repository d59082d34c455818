"""Where the C entries' limits lie: the last size that is taken, by its next check, and the first that is refused. Runs without a GPU."""
import pytest

from tests.test_ops_refusals_more import delta


@pytest.mark.parametrize("more", [dict(T=1), dict(T=64), dict(T=1, V=32)])
def test_delta_sequences(more):
    """B G ceil(T / 64) and B G ceil(V / 32) below 2^23, for calls that go step by step too"""
    of = lambda B: delta(B=B, H=1, G=1, out=None, **({"V": 8} | more))  # noqa: E731
    assert "null" in of((1 << 23) - 1) and "too many" in of(1 << 23)


def test_delta_chunks():
    of = lambda T: delta(B=1, H=1, G=1, T=T, V=8, out=None)  # noqa: E731
    assert "null" in of(((1 << 23) - 1) * 64) and "too many" in of(((1 << 23) - 1) * 64 + 1)


def test_delta_columns():
    of = lambda B, V: delta(B=B, H=1, G=1, T=1, V=V, out=None)  # noqa: E731
    assert "null" in of((1 << 22) - 1, 64) and "too many" in of((1 << 22) - 1, 65) and "too many" in of(1 << 22, 64)

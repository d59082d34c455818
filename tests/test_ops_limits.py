"""Sizes past what one launch takes (below 2^32 work items in a grid): refused by the C entries before any launch, or worked on
in several."""
from panvram_amd import _native as N
from tests.test_ops_refusals import FAKE, refused


def test_scan_workgroups():
    """512 work items for a chunk of a sequence's channels: 2^23 of them are too many."""
    def scan(B, T, D, dtype=N.F32):
        return refused("pv_gated_scan_hip", FAKE, FAKE, None, None, B, T, D, D * T, D, D * T, D, dtype, FAKE, FAKE, None, FAKE, 1 << 50)

    def back(B, T, D, dtype=N.F32):
        return refused("pv_gated_scan_backward_hip", FAKE, FAKE, FAKE, None, B, T, D, D * T, D, D * T, D, FAKE, D * T, D, None, dtype, FAKE, FAKE, None, FAKE, 1 << 50)
    for fn in (scan, back):
        assert "too many chunks" in fn(1 << 23, 33, 1)
        assert "too many chunks" in fn(1 << 23, 33, 128, N.BF16)
        assert "too many chunks" in fn(1, (1 << 31) - 1, 1)
        assert "too many chunks" in fn(1 << 26, 1, 1)

"""The operators' scratch memory: aligned as the header asks for, or refused before any launch."""
import ctypes

from panvram_amd import _native as N
from tests.test_ops_refusals import FAKE, refused


def test_work_alignment():
    vp, i64, i32 = ctypes.c_void_p * 1, ctypes.c_int64 * 1, ctypes.c_int32 * 1
    off = FAKE + 8
    assert "16-byte" in refused("pv_add_rms_norm_backward_hip", FAKE, FAKE, FAKE, 4000, 8, 8, FAKE, None, N.F32, FAKE, FAKE, off, 1 << 20)
    assert "16-byte" in refused("pv_next_base_loss_hip", FAKE, FAKE, FAKE, 2, 5, 8, 5, 40, 8, 5, 4, N.BF16, N.BF16, 1, None, None, None, FAKE, None, None, off, 1 << 20)
    assert "16-byte" in refused("pv_gradient_norm_hip", vp(FAKE), i64(100), i32(N.F32), 1, FAKE, off, 1 << 20)
    assert "16-byte" in refused("pv_gated_scan_hip", FAKE, FAKE, None, None, 1, 5000, 4, 20000, 4, 20000, 4, N.F32, FAKE, FAKE, None, off, 1 << 20)

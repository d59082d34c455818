"""The norm's gradients where a workgroup goes over several groups of rows, the last of them a part of one: more than 1,024
workgroups' rows in every plan that holds a row in registers, and in the one that does not. Run with -m gpu."""
import ctypes

import pytest
import torch

from panvram_amd import _native as N
from tests.test_gpu_norm import check, make

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


# elements of a row that 8, 16, 32 and 64 lanes hold as one pack of 16 bytes each, then as two (rows a workgroup: 32, 16, 8, 4, 4),
# and rows by a workgroup of their own, or too long to be held
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("packs,rows", [(8, 32), (16, 16), (31, 8), (64, 4), (128, 4)])
def test_several_rows_a_workgroup(packs, rows, dtype):
    D = packs * 16 // torch.empty(0, dtype=dtype).element_size() - 3
    check(*make(1024 * rows + rows + 1, D, dtype, seed=packs))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N_,D", [(2 * 1024 + 1, 2056), (1024 + 3, 4100), (1030, 16_500)])
def test_a_row_a_workgroup(N_, D, dtype):
    check(*make(N_, D, dtype, seed=D))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,D", [(1, 64), (31, 60), (33, 60), (5, 512), (17, 1000), (2, 1024), (3, 1025), (40, 2048), (3, 2049), (2, 5000), (1100, 8192),
                                 (2, 16_384), (3, 16_385), (33_000, 64), (2, 40_000)])
def test_workspace(n, D, dtype):
    """The bytes that the library asks for hold what the backward pass writes, and it does not write behind them."""
    x, _, weight, d_y, _ = make(n, D, dtype, seed=n + D, residual=False)
    rstd = (x.float().square().mean(-1) + 1e-6).rsqrt()
    size = N.lib().pv_add_rms_norm_work_bytes(n, D)
    assert size % 4 == 0
    room = torch.full((size // 4 + (1 << 20),), 7.0, device="cuda")
    d, d_weight, err = torch.empty_like(x), torch.empty(D, device="cuda"), N.errbuf()
    kind = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}[dtype]
    code = N.lib().pv_add_rms_norm_backward_hip(x.data_ptr(), rstd.data_ptr(), weight.data_ptr(), n, D, D, d_y.data_ptr(), None, kind, d.data_ptr(),
                                                d_weight.data_ptr(), room.data_ptr(), size, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), err, len(err))
    assert code == N.PV_OK, err.value
    assert bool((room[size // 4:] == 7.0).all())
    want = (d_y.double() * x.double() * rstd.double()[:, None])
    assert bool(((d_weight - want.sum(0)).abs() <= (n + 64) * 2.0 ** -23 * want.abs().sum(0) + 1e-30).all())

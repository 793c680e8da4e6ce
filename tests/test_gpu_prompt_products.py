"""e4m3 products in tiles of 128 x 128 with fetching waves and of 256 x 256, which large 16-bit outputs take: rows that are stored in whole 16 bytes through LDS, more
groups of K than a wave holds the scales of at once (64, and 128), edges in both directions.  Bounds as in test_gpu_prompt.
"""
import ctypes

import pytest
import torch

from conftest import pkg
from test_gpu_prompt import DEV, _operands, _product, name
from test_gpu_states import _check

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


def _run(M, N, K, dtype, seed=80):
    """With a bias and without, twice, and at an address that is no multiple of 16: all of the outputs."""
    ql = pkg("qlinear")
    a, w, xs, ws, bias = _operands(M, N, K, dtype, seed)
    for b in (bias, None):
        got = ql.fp8_gemm(a, w, xs, ws, b, dtype)
        want, bound = _product(a, w, xs, ws, b, dtype)
        _check(got, want, bound, "no bias" if b is None else "bias")
        room = torch.full((M * N + 16,), 7.0, dtype=dtype, device=DEV)
        for at in (8, 1):
            ql.fp8_gemm(a, w, xs, ws, b, dtype, room[at:M * N + at].view(M, N))
            assert torch.equal(room[at:M * N + at].view(M, N), got) and (room[:at] == 7).all() and (room[M * N + at:] == 7).all()
            room.fill_(7.0)


@pytest.mark.parametrize("dtype", HALVES, ids=name)
@pytest.mark.parametrize("form,slices", [(1, 1), (2, 1), (2, 3), (3, 1), (5, 1)])
@pytest.mark.parametrize("M,N,K", [(300, 520, 8400), (300, 520, 16656), (257, 264, 16384), (256, 256, 128), (513, 776, 1040), (129, 248, 8320), (1, 8, 24704)])
def test_forms_at_whole_16_bytes_and_long_k(M, N, K, form, slices, dtype):
    ffi, out = pkg("ffi"), (ctypes.c_int32 * 2)()
    ffi.k("gpu_internal_fp8_gemm_force", 100 * form + slices)
    try:
        ffi.k("gpu_internal_fp8_gemm_plan", M, N, K, ffi.DT_BF16, ctypes.cast(out, ctypes.c_void_p))
        assert out[0] == form
        _run(M, N, K, dtype)
    finally:
        ffi.k("gpu_internal_fp8_gemm_force", -1)


@pytest.mark.parametrize("dtype", HALVES, ids=name)
@pytest.mark.parametrize("M,N,K,plan", [(1500, 6144, 256, (1, 1)), (3000, 3000, 272, (1, 1)), (700, 4096, 256, (2, 1)), (300, 8192, 400, (2, 1)), (300, 4096, 8400, (2, 2)), (200, 3000, 8400, (2, 5)), (64, 256, 8400, (3, 6))])
def test_sizes_that_take_them(M, N, K, plan, dtype):
    ffi, out = pkg("ffi"), (ctypes.c_int32 * 2)()
    ffi.k("gpu_internal_fp8_gemm_plan", M, N, K, ffi.DT_BF16 if dtype == torch.bfloat16 else ffi.DT_F16, ctypes.cast(out, ctypes.c_void_p))
    assert tuple(out) == plan
    _run(M, N, K, dtype)

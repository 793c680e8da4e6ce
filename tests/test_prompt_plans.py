"""How the e4m3 products run their sizes, without a GPU: what the plan promises its kernels and its callers."""
import ctypes
import random

import pytest

from conftest import pkg

ffi = pkg("ffi")
BF16, F16, F32 = ffi.DT_BF16, ffi.DT_F16, ffi.DT_F32


def _plan(M, N, K, dt):
    out = (ctypes.c_int32 * 2)()
    ffi.k("gpu_internal_fp8_gemm_plan", M, N, K, dt, ctypes.cast(out, ctypes.c_void_p))
    return tuple(out)


def _none_empty(M, N, K, dt, what):
    """A slice begins at a group that there is: the kernels read that group's scales before anything else."""
    slices, groups = _plan(M, N, K, dt)[1], -(-K // 128)
    assert slices >= 1 and (slices - 1) * -(-groups // slices) < groups, (what, M, N, K, slices)


@pytest.mark.parametrize("form,M", [(2, 200), (3, 50), (4, 16)])
def test_forced_slices_of_k_all_have_groups(form, M):
    try:
        for slices in range(1, 33):
            ffi.k("gpu_internal_fp8_gemm_force", 100 * form + slices)
            for groups in range(1, 80):
                for dt in (BF16, F32):
                    _none_empty(M, 200, 128 * groups, dt, "form %d in %d" % (form, slices))
                _none_empty(M, 200, 128 * groups + 16, BF16, "form %d in %d" % (form, slices))
            assert _plan(M, 200, 128 * 32 * slices, BF16) == (form, slices)      # where they divide, as many as were asked for
    finally:
        ffi.k("gpu_internal_fp8_gemm_force", -1)


def test_planned_slices_of_k_all_have_groups():
    rng = random.Random(1)
    for _ in range(20000):
        M, N, K = (int(2 ** rng.uniform(0, top)) for top in (13, 15, 17))
        _none_empty(M, N, max(16, K // 16 * 16), rng.choice((BF16, F16, F32)), "planned")

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


# rows and columns of a workgroup by form (few rows: all of them, 32 columns where those are many), and the threads that a launch of it has for each
TILES = {0: (128, 128, 256), 1: (256, 256, 512), 2: (128, 128, 512), 3: (64, 128, 512), 4: (32, 32, 512), 5: (128, 128, 512)}


def _launches(M, N, K, dt):
    form, slices = _plan(M, N, K, dt)
    bm, bn, threads = TILES[form]
    return -(-M // bm) * -(-N // bn) * slices <= 0xffffffff // threads


@pytest.mark.parametrize("M,N,K,dt", [(150, 400000000, 128, F32), (200, 10 ** 9 // 2, 256, F32), (300, 300000000, 128, F32), (1000, 10 ** 8, 128, BF16), (33, 10 ** 9, 256, F32), (5, 3 * 10 ** 8, 128, BF16),
                                      (32, 10 ** 9, 4096, F32), (10 ** 9, 1, 128, F32), (10 ** 9, 100, 4096, F16), (9, 10 ** 9, 64, F32)])
def test_sizes_whose_tiles_of_128_a_launch_holds_are_not_refused(M, N, K, dt):
    assert -(-M // 128) * -(-N // 128) <= 8388607 and _launches(M, N, K, dt), _plan(M, N, K, dt)


def test_large_sizes_take_forms_that_a_launch_holds():
    rng = random.Random(2)
    for _ in range(20000):
        M = int(2 ** rng.uniform(0, 31 - 1e-6))
        N = int(min(2 ** rng.uniform(0, 31), 128 * (8388607 // -(-M // 128))) * 0.999)
        if N >= 1:
            K, dt = rng.choice((16, 128, 400, 4096, 12288)), rng.choice((BF16, F16, F32))
            assert _launches(M, N, K, dt), (M, N, K, dt, _plan(M, N, K, dt))

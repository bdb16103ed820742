"""Which kernel an MXFP4 product takes: the host's choice, asked without a launch (CPU)."""
import ctypes

import pytest

from hopper_megamoe_basedondeepgemm_amd import _lib


def form(m, n, k, swiglu=False, workspace=1 << 40):
    """(tokens, channels, stages, ranges of K, parts of K, blocks of a step, threads along the grid's first axis)"""
    out = (ctypes.c_int64 * 7)()
    _lib.check(_lib.load().dgm_mxfp4_gemm_form(m, n, k, swiglu, workspace, out))
    return tuple(out)


def test_refusals():
    lib, out = _lib.load(), (ctypes.c_int64 * 7)()
    for args in ((0, 8, 32, 0), (8, 0, 32, 0), (8, 8, 0, 0), (8, 8, 48, 0), (1 << 24, 8, 32, 0), (8, 7, 32, 1), (1 << 21, 1 << 21, 32, 0)):
        assert lib.dgm_mxfp4_gemm_form(*args, 0, out) == -1, args
    assert lib.dgm_mxfp4_gemm_form(8, 8, 32, 0, 0, None) == -1


@pytest.mark.parametrize("swiglu", [False, True])
def test_a_launch_has_fewer_than_2_32_threads(swiglu):
    """The largest products that are taken, narrow to wide, short and long sums."""
    most, tall = (1 << 23) - 1, (1 << 24) - 2
    for tiles_n in (1, 2, 3, 4, 7, 31, 32, 33, 47, 255, 2895, 2896, 131071, 262144):
        n = min(64 * tiles_n, tall)
        m = min(64 * (most // tiles_n), tall)
        for rows, channels in ((m, n), (m - 63, n - 62), (m // 2, n)):
            for k in (32, 256, 288, 4096, (1 << 24) - 32):
                for workspace in (0, 1 << 40):
                    f = form(rows, channels, k, swiglu, workspace)
                    assert f[6] < 1 << 32, (rows, channels, k, f)


def test_ranges_of_k_need_their_workspace():
    """What the workspace's size is asked for is what the form takes, and without one K is whole."""
    lib = _lib.load()
    for swiglu in (False, True):
        for m, n, k in ((1, 64, 256), (17, 2, 8864), (64, 4096, 7168), (100, 384, 13056), (777, 640, 1312), (4128, 2, 8032), (8192, 8192, 4096)):
            need = lib.dgm_mxfp4_gemm_workspace_bytes(m, n, k, swiglu)
            f = form(m, n, k, swiglu, need)
            assert f == form(m, n, k, swiglu)
            assert need >= 4 * m * n * f[3] if f[3] > 1 else need == 0, (m, n, k, f)
            assert form(m, n, k, swiglu, 0)[3] == 1

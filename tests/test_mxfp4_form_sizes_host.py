"""The sizes of tests/mxfp4_forms.py reach the kernels that they stand for, and together every one there is (CPU): a new
choice of kernels that leaves one without a size fails here, not in silence."""
import pytest

from tests.mxfp4_forms import PLAIN, SWIGLU
from tests.test_mxfp4_forms_host import form

TILES = [(64, 64, 4), (64, 128, 3), (128, 128, 2), (128, 128, 4), (256, 128, 3), (192, 128, 3), (192, 256, 2), (256, 256, 2)]


def kernels(swiglu):
    rows = [(8, 4), (16, 8), (16, 16), (32, 8), (32, 16), (64, 8), (64, 16)] if swiglu else [(8, 8), (16, 16), (32, 16), (64, 16)]
    some = {(t, c, 0, 1 if t > 8 else 2, blocks, False) for t, c in rows for blocks in (2, 4)}
    some -= {(64, 16, 0, 1, 4, False)} if swiglu else set()                              # (not built)
    tiles = {t + (1, 1, ranges) for t in (TILES[1:] if swiglu else TILES) for ranges in (False, True)}
    return some | (tiles - {(128, 128, 2, 1, 1, True)})                                  # (short sums alone)


@pytest.mark.parametrize("swiglu", [False, True])
def test_every_kernel_has_its_sizes(swiglu):
    sizes = SWIGLU if swiglu else PLAIN
    assert set(sizes) == kernels(swiglu)
    wrong = [(s, want, f) for want, some in sizes.items() for s in some
             if (f := form(*s, swiglu))[:3] + f[4:6] + (f[3] > 1,) != want]
    assert not wrong, wrong
    assert all(sizes.values())

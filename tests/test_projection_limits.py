"""Sizes at which the norm, projection and rotary calls would leave their index arithmetic or their grids, on the CPU: refused
before a launch."""
import pytest

from arcagi2_flashnext_dots3_amd import _lib
from tests.test_linear_choice import choose  # noqa: F401 (a fixture)

ELIMIT = -5


@pytest.mark.parametrize("H,W,n,out", [((1 << 30) + 1, 2, 1, 256), ((1 << 31) - 1, 2, 1, 256), (1, (1 << 31) - 1, 1, 512),
                                       (1, (1 << 30) + 1, 0, 512)])
def test_rope_of_more_heads_or_columns_than_the_loops_count(H, W, n, out):
    """A loop's variable passes the size by up to its stride: beyond 2^31 it would wrap to a negative index."""
    assert _lib.status("spmla_rope", 256, H * W, W, 256, 0, 256, 1, H, W, 0, n, 1, 1.0, 0, 2, out, H * W, W, None) == ELIMIT


@pytest.mark.parametrize("K", [(1 << 22) + 16, (1 << 31) - 16])
def test_linear_of_more_k_than_its_blocks_count(K):
    """One token and one output whose rows' strides say nothing of k: k + 127 passed 2^31."""
    assert _lib.status("spmla_linear_fp8", 256, 16, 256, 1, 256, 16, 256, 1, 1, 1, K, 2, 256, 1, None) == ELIMIT


@pytest.mark.parametrize("T,D", [(1 << 23, 8192), (1 << 22, 16384), (1 << 22, 15361), (1 << 22, 65536), (1 << 23, 32769)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_norm_of_more_threads_than_a_grid_takes(T, D, dtype):
    """Wide rows take 512 or 1024 threads each: 2^32 in all."""
    for odd in (0, 1):
        d = D - odd if D != 15361 and D != 32769 else D + odd
        assert _lib.status("spmla_rms_norm", 256, d, None, 0, None, 0, None, 0, 1e-6, T, d, dtype, 256, d, None, 0, None, 0, 0,
                           None) == ELIMIT


def test_projection_of_more_threads_than_a_grid_takes(choose):  # noqa: F811
    """24892 x 337 tiles of 256 x 256 lie below 2^23, but a grid has whole eights of workgroups: 2^23, of 512 threads."""
    assert choose(24892 * 256, 337 * 256, 16) == -1
    assert choose(24892 * 256, 336 * 256, 16) >= 0
    assert _lib.status("spmla_linear_fp8", 256, 16, 256, 1, 256, 16, 256, 1, 24892 * 256, 337 * 256, 16, 2, 256, 337 * 256,
                       None) == ELIMIT

"""The projection's rule (csrc/spmla_rules.h), compiled for the host: measured points on both sides, shapes that reach every
kernel, sizes beyond every grid."""
import ctypes
import shutil
import subprocess

import pytest

from arcagi2_flashnext_dots3_amd import build

# shapes that the rule gives to each kernel in turn, with ends inside the tiles and inside a block of k; the last kernel once
# with a number of blocks that is a multiple of four (the scales of four blocks at once) and once without
REACHES = [(0, 130, 300, 528), (1, 3, 4100, 144), (2, 65, 1000, 1040), (3, 800, 1000, 272), (4, 400, 1030, 2064),
           (5, 33, 8200, 2064), (6, 300, 4100, 400), (7, 1030, 2050, 528), (8, 700, 16300, 272), (8, 1030, 8200, 2000)]


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("rules")
    (d / "r.cpp").write_text('#include "spmla_rules.h"\n'
                             'extern "C" int choose(int T, int N, int K) { return spmla::rules::linear_kernel(T, N, K); }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", build.CSRC, str(d / "r.cpp"), "-o",
                    str(d / "r.so")], check=True, capture_output=True)
    return ctypes.CDLL(str(d / "r.so")).choose


@pytest.mark.parametrize("kernel,T,N,K", REACHES)
def test_every_kernel_is_reached(choose, kernel, T, N, K):
    assert choose(T, N, K) == kernel


@pytest.mark.parametrize("T,N,K,us", [                     # us of the kernels that were measured there
    (1, 2112, 4096, {0: 3.8, 1: 4.6, 2: 4.4, 3: 5.5, 4: 7.2}),
    (16, 24576, 1536, {0: 14.1, 1: 8.8, 2: 15.4, 3: 9.4, 4: 13.1, 5: 13.2, 6: 9.2, 7: 11.3}),
    (32, 4096, 16384, {0: 18.2, 1: 13.8, 2: 14.2, 3: 16.2, 4: 20.4}),
    (48, 2112, 4096, {0: 7.4, 1: 5.2, 2: 8.6, 3: 5.7, 4: 7.6, 5: 10.7}),
    (64, 24576, 1536, {3: 12.6, 4: 14.4, 5: 14.6, 6: 10.4, 7: 11.0}),
    (64, 2112, 4096, {0: 11.3, 1: 7.8, 2: 9.2, 3: 6.3, 4: 8.3, 5: 11.1}),
    (128, 4096, 16384, {3: 30.2, 4: 23.7, 5: 29.3}),
    (384, 576, 7168, {1: 13.8, 2: 14.7, 3: 9.8, 4: 12.9, 5: 16.8}),
    (1455, 2112, 4096, {4: 51.1, 5: 33.6, 6: 30.7, 7: 22.7}),
    (4096, 4096, 4096, {6: 128.8, 7: 93.5, 8: 70.7}),
    (949, 79, 5200, {0: 12.1, 1: 8.7, 2: 9.3, 3: 10.3, 4: 13.7}),
    (3295, 67, 11472, {1: 40.2, 2: 48.2, 3: 34.4, 4: 29.3, 5: 34.9}),
    (96, 1536, 1536, {0: 6.0, 1: 4.1, 2: 5.1, 3: 3.8, 4: 4.7, 5: 6.0, 6: 7.7}),
    (548, 2497, 736, {3: 9.8, 4: 11.2, 5: 11.0, 6: 8.6, 7: 11.3}),
    (512, 24576, 1536, {6: 46.5, 7: 36.7, 8: 33.6}),
    (768, 24576, 1536, {5: 89.9, 6: 65.3, 7: 55.9, 8: 59.7}),
    (24, 24576, 1536, {1: 10.4, 2: 15.6, 3: 9.3, 4: 13.1, 5: 13.2, 6: 9.5, 7: 10.1}),
    (262, 543, 4896, {0: 14.3, 1: 11.0, 2: 12.1, 3: 9.2, 4: 12.2, 5: 16.4}),
    (64, 4096, 4096, {1: 8.5, 2: 10.1, 3: 6.9, 4: 8.8, 5: 11.3}),
    (6, 1947, 528, {0: 2.9, 1: 3.0, 2: 3.0, 3: 3.3, 4: 4.0, 5: 5.4, 6: 5.1})])
def test_choice_is_within_a_tenth_of_the_fastest(choose, T, N, K, us):
    assert us[choose(T, N, K)] <= 1.1 * min(us.values())


def test_grids_of_too_many_workgroups(choose):
    assert choose(1 << 23, 1 << 23, 16) == -1
    assert choose(1 << 23, 64, 16) >= 0 and choose(1, 1 << 23, 16384) >= 0

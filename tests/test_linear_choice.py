"""The projection's rule (csrc/spmla_rules.h), compiled for the host: measured points on both sides, shapes that reach every
kernel, sizes beyond every grid."""
import ctypes
import shutil
import subprocess

import pytest

from arcagi2_flashnext_dots3_amd import build

# shapes that the rule gives to each kernel in turn, with ends inside the tiles and inside a block of k; the last kernel with
# one tile a workgroup, and with several (k a multiple of 128) of 2, 3, 5 and 8 blocks
REACHES = [(0, 130, 300, 528), (1, 3, 4100, 144), (2, 17, 4100, 528), (3, 400, 1030, 2064), (4, 33, 8200, 2064),
           (5, 300, 4100, 400), (6, 1030, 2050, 528), (7, 700, 16300, 272), (7, 1030, 8200, 2000), (7, 2049, 8200, 128), (7, 2050, 16640, 256),
           (7, 2049, 8200, 384), (7, 1800, 16640, 640), (7, 1300, 16400, 1024)]


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
    (1, 2112, 4096, {0: 3.8, 1: 4.7, 2: 5.3}),
    (16, 24576, 1536, {1: 8.7, 2: 9.3, 3: 13.1, 4: 13.4, 5: 8.9, 6: 9.8}),
    (32, 4096, 16384, {0: 18.4, 1: 14.1, 2: 15.9, 3: 21.0}),
    (48, 2112, 4096, {0: 7.4, 1: 5.2, 2: 5.7, 3: 7.6}),
    (64, 24576, 1536, {2: 12.4, 3: 14.4, 4: 14.4, 5: 9.8, 6: 10.6}),
    (64, 2112, 4096, {0: 11.2, 1: 7.8, 2: 6.2, 3: 8.3, 4: 11.0}),
    (128, 4096, 16384, {2: 28.8, 3: 23.8, 4: 29.2}),
    (384, 576, 7168, {1: 14.0, 2: 9.8, 3: 12.9, 4: 16.8}),
    (1455, 2112, 4096, {3: 51.1, 4: 33.1, 5: 27.3, 6: 20.6}),
    (4096, 4096, 4096, {5: 114.6, 6: 86.1, 7: 62.1}),
    (4096, 24576, 1536, {5: 345.8, 6: 296.4, 7: 160.2}),
    (2255, 145, 13200, {1: 47.4, 2: 40.0, 3: 34.2, 4: 39.8}),
    (2048, 24576, 1536, {5: 203.7, 6: 148.4, 7: 79.6}),
    (11, 9187, 14128, {0: 40.3, 1: 43.7, 2: 44.3, 3: 46.0, 4: 43.7}),
    (365, 1502, 928, {1: 7.7, 2: 6.5, 3: 8.0, 4: 6.1, 5: 6.2, 6: 8.0}),
    (9, 95, 928, {0: 2.7, 1: 3.0, 2: 3.3, 3: 4.2, 4: 5.4}),
    (40, 5882, 3760, {1: 11.4, 2: 10.0, 3: 9.9, 4: 13.2, 5: 16.3}),
    (23, 1158, 3712, {0: 4.0, 1: 4.8, 2: 5.4, 3: 7.5}),
    (9, 4871, 5824, {0: 10.3, 1: 7.6, 2: 8.4, 3: 10.7})])
def test_choice_is_within_a_tenth_of_the_fastest(choose, T, N, K, us):
    assert us[choose(T, N, K)] <= 1.1 * min(us.values())


def test_grids_of_too_many_workgroups(choose):
    assert choose(1 << 23, 1 << 23, 16) == -1
    assert choose(1 << 23, 64, 16) >= 0 and choose(1, 1 << 23, 16384) >= 0

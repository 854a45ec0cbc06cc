"""Places and limits of the attention over all cached rows that are fixed by rules alone (csrc/spmla_rules.h), compiled for the
host."""
import ctypes
import shutil
import subprocess

import pytest

from arcagi2_flashnext_dots3_amd import build


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("rules")
    (d / "r.cpp").write_text('#include "spmla_rules.h"\n'
                             'extern "C" int join_at(int wr, int half, int wp) { return spmla::rules::chunk_join_at(wr, half, wp); }\n'
                             'extern "C" int join_bytes() { return spmla::rules::CHUNK_JOIN; }\n'
                             'extern "C" int rows_at(int wr) { return spmla::rules::chunk_rows_at(wr); }\n'
                             'extern "C" int splits() { return spmla::rules::CHUNK_SPLITS; }\n'
                             'extern "C" int extra(int beyond, int slack, int B) { return spmla::rules::chunk_extra(beyond, slack, B); }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", build.CSRC, str(d / "r.cpp"), "-o",
                    str(d / "r.so")], check=True, capture_output=True)
    return ctypes.CDLL(str(d / "r.so"))


@pytest.mark.parametrize("shares", [2, 4])
def test_rows_are_written_where_no_other_wave_reads(lib, shares):
    """Nothing waits between a wave's last reads of its partner's sums and another wave's bf16 rows (16 of 1024 bytes)."""
    for wr in range(8 // shares):
        at = lib.rows_at(wr)
        for other in range(8 // shares):
            if other != wr:
                lo = lib.join_at(other, 1, 0)
                assert at + 16 * 1024 <= lo or lo + lib.join_bytes() <= at, (wr, other)
                assert abs(at - lib.rows_at(other)) >= 16 * 1024


@pytest.mark.parametrize("shares", [2, 4])
def test_partial_sums_of_a_round_do_not_overlap(lib, shares):
    half = shares // 2
    while half:
        places = [lib.join_at(wr, half, wp) for wr in range(8 // shares) for wp in range(half)]
        places.sort()
        assert all(b - a >= lib.join_bytes() for a, b in zip(places, places[1:])) and places[-1] + lib.join_bytes() <= 4 * 32768
        half //= 2


@pytest.mark.parametrize("beyond", [1, 255, 300, 510, 511])
@pytest.mark.parametrize("slack,requests", [(0, 1), (1, 1), (1, 2), (1, 200), (1, 256)])
def test_no_row_has_more_parts_than_the_join_takes(lib, beyond, slack, requests):
    """One tile may take all of the workgroups beyond one a tile."""
    extra = lib.extra(beyond, slack, requests)
    assert extra + 1 <= lib.splits()
    assert extra >= beyond

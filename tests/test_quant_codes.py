"""The quantizer's rule for codes that two products decide (csrc/spmla_quant.h), compiled for the host."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from arcagi2_flashnext_dots3_amd import build


@pytest.fixture(scope="module")
def decide(tmp_path_factory):
    """(t, c) fp32 arrays -> (codes, decided): the kernel's two products of each t with about c."""
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc")
    d = tmp_path_factory.mktemp("codes")
    (d / "c.hip").write_text('''#include "spmla_quant.h"
using namespace spmla;
extern "C" void decide(const float* t, const float* c, int n, unsigned char* code, unsigned char* decided) {
  for (int i = 0; i < n; ++i) {
    const Around a = around(c[i]);
    code[i] = e4m3_rne(t[i] * a.up);
    decided[i] = e4m3_rne(t[i] * a.dn) == code[i];
  }
}
''')
    subprocess.run([build.HIPCC, *build.FLAGS, "-shared", str(d / "c.hip"), "-o", str(d / "c.so")], check=True, capture_output=True)
    f = ctypes.CDLL(str(d / "c.so")).decide

    def call(t, c):
        t, c = (np.ascontiguousarray(np.broadcast_to(v, np.broadcast_shapes(np.shape(t), np.shape(c))), dtype=np.float32) for v in (t, c))
        out = [np.empty(t.shape, np.uint8) for _ in range(2)]
        f(*(v.ctypes.data_as(ctypes.c_void_p) for v in (t, c)), t.size, *(v.ctypes.data_as(ctypes.c_void_p) for v in out))
        return out[0], out[1].astype(bool)
    return call


def _bf16(v):
    return torch.from_numpy(v.astype(np.float32)).to(torch.bfloat16).float().numpy()


def _code(q):
    """e4m3 codes of q (float64, |q| <= 448), to nearest, ties to even, and whether q is halfway between two."""
    _, e = np.frexp(q)
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    v = np.round(q / step) * step
    return torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), np.abs(q / step % 1) == 0.5


def test_groups_maxima_zeros_and_whole_codes_are_decided(decide):
    """The largest value of a group is 448 within the product's rounding, a code and not a middle; so are zeros and whole codes."""
    rng = np.random.default_rng(1)
    am = np.abs(rng.standard_normal(200000) * np.exp(4 * rng.standard_normal(200000))).astype(np.float32)
    for top in (am, _bf16(am)):
        code, ok = decide(np.concatenate((top, -top)), np.tile(np.float32(448) / top, 2))
        assert ok.all() and (code == np.repeat([0x7E, 0xFE], top.size)).all()
    code, ok = decide(np.array([0.0, -0.0], np.float32), np.float32(3))
    assert ok.all() and code.tolist() == [0, 0x80]
    whole = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    whole = whole[np.isfinite(whole)]
    for c in (1.0, 2.0 ** -7, 2.0 ** 9):
        code, ok = decide(whole / np.float32(c), np.float32(c))
        assert ok.all() and (code == _code(whole.astype(np.float64))[0]).all()


def test_middles_are_not_decided_and_decided_codes_are_exact(decide):
    rng = np.random.default_rng(2)
    for few in (False, True):                                       # 16-bit values: many exact middles
        t = rng.standard_normal((4000, 128)) * np.exp(3 * rng.standard_normal((4000, 1)))
        t[:, 5:40] *= np.exp2(-rng.integers(0, 18, (4000, 35)))     # codes down to the smallest steps
        t = _bf16(t) if few else t.astype(np.float32)
        am = np.abs(t).max(1, keepdims=True)
        q = t.astype(np.float64) * 448.0 / am                       # within 2^-52; an exact middle is one here
        want, half = _code(q)
        code, ok = decide(t, np.float32(448) / am)
        assert not ok[half].any() and (code[ok] == want[ok]).all()
        assert half.sum() > 100 or not few
        # the products differ by 2^-20 of a value, a middle lies within 2^-20 * 16 steps of it at most: 2^-16 of the others
        assert (~ok & ~half).mean() <= 2 * 2.0 ** -16


def test_most_groups_of_products_are_decided(decide):
    """Groups of 512 products of two bf16 values (a wave's): a division for one in some six."""
    rng = np.random.default_rng(3)
    t = _bf16(rng.standard_normal((2000, 4, 128))) * _bf16(1 + 0.2 * rng.standard_normal((2000, 4, 128)))
    _, ok = decide(t, np.float32(448) / np.abs(t).max(2, keepdims=True))
    assert (~ok).any((1, 2)).mean() < 0.4

"""Rotary frequencies, on the CPU."""
import math

import pytest
import torch

from arcagi2_flashnext_dots3_amd import rotary


def test_plain_linear_and_ntk():
    f, c = rotary.frequencies(64)
    assert c == 1.0 and f.dtype == torch.float64 and f.shape == (32,)
    for i in (0, 7, 31):
        assert float(f[i]) == pytest.approx(10000.0 ** (-2 * i / 64), rel=2.0 ** -50)
    g, c = rotary.frequencies(64, scaling={"type": "linear", "factor": 8.0})
    assert c == 1.0 and torch.equal(g, f / 8.0)
    g, c = rotary.frequencies(64, scaling={"type": "ntk", "factor": 8.0})
    assert c == 1.0 and float(g[0]) == 1.0 and float(g[31]) == pytest.approx(float(f[31]) / 8.0, rel=1e-12)


def test_yarn_keeps_fast_and_stretches_slow_frequencies():
    f, _ = rotary.frequencies(64)
    g, c = rotary.frequencies(64, scaling={"type": "yarn", "factor": 40.0, "original": 4096})
    assert c == pytest.approx(0.1 * math.log(40.0) + 1.0, rel=1e-15)
    turns = 4096 * f / (2 * math.pi)
    i = torch.arange(32)
    lo, hi = int(i[turns >= 32].max()), int(i[turns <= 1].min())
    assert torch.equal(g[:lo + 1], f[:lo + 1]) and torch.allclose(g[hi:], f[hi:] / 40.0, rtol=1e-15, atol=0)
    ratio = g / f
    assert bool((ratio[1:] <= ratio[:-1] + 1e-15).all()) and bool((g[1:] < g[:-1]).all())
    assert rotary.frequencies(64, scaling={"type": "yarn", "factor": 4.0, "original": 4096, "attention_factor": 1.0})[1] == 1.0
    assert rotary.frequencies(64, scaling={"type": "yarn", "factor": 1.0, "original": 4096})[1] == 1.0


@pytest.mark.parametrize("dim,scaling", [(0, None), (63, None), (64, {"type": "linear", "factor": 0.0}), (2, {"type": "ntk"}),
                                         (64, {"type": "yarn", "factor": 4.0}), (64, {"type": "other", "factor": 2.0})])
def test_refusals(dim, scaling):
    with pytest.raises(ValueError):
        rotary.frequencies(dim, scaling=scaling)

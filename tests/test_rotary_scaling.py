"""The keys of a rotary scaling, on the CPU: those that weigh cosine and sine are taken, unknown ones refused."""
import math

import pytest
import torch

from arcagi2_flashnext_dots3_amd import rotary

YARN = {"type": "yarn", "factor": 40.0, "original": 4096}


def _m(a, s=40.0):
    return 0.1 * a * math.log(s) + 1.0


@pytest.mark.parametrize("keys,factor", [
    ({}, _m(1)), ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0), ({"mscale": 0.707, "mscale_all_dim": 0.707}, 1.0),
    ({"mscale": 0.707, "mscale_all_dim": 1.0}, _m(0.707) / _m(1)), ({"mscale": 0.5}, _m(0.5)), ({"mscale_all_dim": 1.0}, 1.0),
    ({"mscale": 1.0, "mscale_all_dim": 0.0}, _m(1)), ({"attention_factor": 0.25}, 0.25), ({"mscale": None, "beta_slow": None}, _m(1))])
def test_yarn_weighs_cosine_and_sine_as_the_model_states(keys, factor):
    f, c = rotary.frequencies(64, scaling={**YARN, **keys})
    assert c == pytest.approx(factor, rel=1e-15)
    assert torch.equal(f, rotary.frequencies(64, scaling=YARN)[0])
    r = rotary.Rotary(64, scaling={**YARN, **keys}, device="cpu")
    assert r.factor == c and torch.equal(r.freqs, f)


def test_no_stretch_no_factor():
    assert rotary.frequencies(64, scaling={**YARN, "factor": 1.0, "mscale": 2.0, "mscale_all_dim": 0.5})[1] == 1.0


@pytest.mark.parametrize("scaling,name", [
    ({**YARN, "mscales": 1.0}, "mscales"), ({**YARN, "attention_factor": 1.0, "mscale": 1.0}, "attention_factor"),
    ({"type": "linear", "factor": 2.0, "mscale": 1.0}, "mscale"), ({"type": "ntk", "factor": 2.0, "beta_fast": 32}, "beta_fast"),
    ({"type": "ntk", "factor": 2.0, "attention_factor": 1.5}, "attention_factor"), ({**YARN, "original_length": 1}, "original_length")])
def test_what_is_not_known_is_refused(scaling, name):
    with pytest.raises(ValueError, match=name):
        rotary.frequencies(64, scaling=scaling)


def test_the_original_length_is_a_fact_of_the_model():
    for kind in ("linear", "ntk"):
        a, b = (rotary.frequencies(64, scaling={"type": kind, "factor": 8.0, **k}) for k in ({}, {"original": 4096}))
        assert a[1] == b[1] == 1.0 and torch.equal(a[0], b[0])

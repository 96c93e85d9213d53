"""Rotary tables of model configurations' rope_scaling: every parameter counts, is known to change nothing, or is refused.  No GPU."""
import math

import numpy as np
import pytest
import torch

from turboquant.kernels.rotary import make_rotary_table


def _angles_and_size(table):
    half = table.shape[1] // 2
    cos, sin = table[1, :half].double(), table[1, half:].double()
    return torch.atan2(sin, cos).numpy(), torch.hypot(cos, sin).numpy()


def _yarn(dim, base, factor, trained, truncate, fast=32.0, slow=1.0):
    """Frequencies of YaRN: pairs that turn more than `fast` times over the trained length stay, fewer than `slow` are stretched, a ramp between."""
    f = base ** (-np.arange(0, dim, 2) / dim)
    pair_of = lambda turns: dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = pair_of(fast), pair_of(slow)
    if truncate:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    ramp = np.clip((np.arange(dim // 2) - low) / max(high - low, 0.001), 0, 1)
    return f * (1 - ramp) + f / factor * ramp


@pytest.mark.parametrize("truncate", [None, True, False])
@pytest.mark.parametrize("dim,base,factor,trained", [(64, 150000.0, 32.0, 4096), (128, 10000.0, 4.0, 32768), (64, 10000.0, 40.0, 4096)])
def test_yarn_with_and_without_whole_borders(dim, base, factor, trained, truncate):
    spec = {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": trained}
    if truncate is not None:
        spec["truncate"] = truncate
    angles, _ = _angles_and_size(make_rotary_table(dim, 2, base, spec))
    # angles at position 1 lie below pi and come from two fp32 numbers, rounded to 2^-25 of at most 1.4 (the factor): 1e-7 each
    np.testing.assert_allclose(angles, _yarn(dim, base, factor, trained, truncate is not False), rtol=0, atol=3e-7)


def test_yarn_pair_that_truncation_moves():
    """The pair whose frequency depends most on it, by hand: dim 64, base 150000, factor 32, trained length 4096."""
    spec = {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096}
    cut, _ = _angles_and_size(make_rotary_table(64, 2, 150000.0, spec))
    exact, _ = _angles_and_size(make_rotary_table(64, 2, 150000.0, {**spec, "truncate": False}))
    assert (np.abs(cut / exact - 1)).max() > 0.1


def _mscale(factor, m=1.0):
    return 1.0 if factor <= 1 else 0.1 * m * math.log(factor) + 1.0


@pytest.mark.parametrize("more,want", [
    ({}, _mscale(40.0)), ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0), ({"mscale": 0.707, "mscale_all_dim": 0.707}, 1.0),
    ({"mscale": 1.0, "mscale_all_dim": 0.707}, _mscale(40.0) / _mscale(40.0, 0.707)), ({"mscale": 0.707}, _mscale(40.0)),
    ({"mscale": 1.0, "mscale_all_dim": 0.0}, _mscale(40.0)), ({"attention_factor": 0.9}, 0.9), ({"attention_factor": 0.9, "mscale": 1.0, "mscale_all_dim": 1.0}, 0.9),
    ({"attention_factor": None, "mscale": None}, _mscale(40.0))])
def test_yarn_factor_on_cosines_and_sines(more, want):
    spec = {"type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "beta_fast": 32, "beta_slow": 1, **more}
    _, size = _angles_and_size(make_rotary_table(64, 2, 10000.0, spec))
    np.testing.assert_allclose(size, want, rtol=3e-7)


def test_yarn_of_factor_one_changes_nothing():
    spec = {"rope_type": "yarn", "factor": 1.0, "original_max_position_embeddings": 4096, "mscale": 1.0, "mscale_all_dim": 0.5}
    assert torch.equal(make_rotary_table(64, 100, 10000.0, spec), make_rotary_table(64, 100, 10000.0))


LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
DYNAMIC = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 512}


@pytest.mark.parametrize("spec,key", [
    ({**YARN, "extrapolation_factor": 1.0}, "extrapolation_factor"), ({**LLAMA3, "mscale": 1.0}, "mscale"), ({**DYNAMIC, "alpha": 1000.0}, "alpha"),
    ({"rope_type": "linear", "factor": 2.0, "truncate": False}, "truncate"), ({"rope_type": "default", "mrope_section": [16, 24, 24]}, "mrope_section"),
    ({"mrope_section": [16, 24, 24]}, "mrope_section")])
def test_parameters_that_are_not_known_are_refused(spec, key):
    with pytest.raises(ValueError, match=key):
        make_rotary_table(64, 16, scaling=spec)


@pytest.mark.parametrize("spec,key", [({k: v for k, v in spec.items() if k != key}, key) for spec in (LLAMA3, YARN, DYNAMIC, {"rope_type": "linear", "factor": 2.0})
                                      for key in spec if key != "rope_type"] + [({**DYNAMIC, "original_max_position_embeddings": None}, "original_max_position_embeddings")])
def test_parameters_that_are_missing_are_named(spec, key):
    with pytest.raises(ValueError, match=key):
        make_rotary_table(64, 16, scaling=spec)


def test_parameters_that_go_with_every_type():
    """A configuration may name its base and the rotated part of a head beside the scaling: the base has to be the call's, the part is rotary_dim."""
    for spec in ({"rope_type": "default"}, {"rope_type": "linear", "factor": 2.0}, LLAMA3, YARN, DYNAMIC):
        want = make_rotary_table(64, 600, 500000.0, spec)
        assert torch.equal(make_rotary_table(64, 600, 500000.0, {**spec, "rope_theta": 500000.0, "partial_rotary_factor": 0.5}), want)
        with pytest.raises(ValueError, match="rope_theta"):
            make_rotary_table(64, 600, 10000.0, {**spec, "rope_theta": 500000.0})


def test_both_names_of_the_type_agree_or_are_refused():
    assert torch.equal(make_rotary_table(64, 16, scaling={"rope_type": "linear", "type": "linear", "factor": 2.0}),
                       make_rotary_table(64, 16, scaling={"type": "linear", "factor": 2.0}))
    assert torch.equal(make_rotary_table(64, 16, scaling={}), make_rotary_table(64, 16))


def test_values_that_make_no_table_are_refused():
    for spec in ({**LLAMA3, "high_freq_factor": 1.0}, {**YARN, "beta_fast": 0.0}, {**YARN, "factor": math.inf}, {**YARN, "original_max_position_embeddings": 0}):
        with pytest.raises(ValueError):
            make_rotary_table(64, 16, scaling=spec)
    with pytest.raises(ValueError, match="rotary_dim"):
        make_rotary_table(2, 1024, scaling=DYNAMIC)                         # the base's exponent is R / (R - 2)
    with pytest.raises(ValueError, match="base"):
        make_rotary_table(64, 16, base=1.0, scaling=YARN)

"""CPU tests of paged.rope_frequencies on the keys that a model's rope_scaling may hold.  The numbers are the definitions',
worked out with 40 decimal digits."""
import pytest
import torch

from exl3rocm import paged

YARN = {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096}


def frequencies(scaling, rot_dim=64, base=150000):
    return paged.rope_frequencies(rot_dim, base, scaling, device="cpu")


@pytest.mark.parametrize("truncate,want", [
    (False, {0: 1.0, 8: 0.050813274815461475, 9: 0.03170569618466377, 12: 0.006794959489732218, 17: 0.00012931870124506273, 18: 3.8308812373753384e-05}),
    (True, {0: 1.0, 8: 0.050813274815461475, 9: 0.03162075227534649, 12: 0.007015713910504388, 17: 0.00022794779579512526, 18: 3.8308812373753384e-05}),
])
def test_yarn_ends_of_the_ramp(truncate, want):
    """The ramp runs from pair 8.0928 to 17.398, or, whole pairs, from 8 to 18."""
    f, _ = frequencies({**YARN, "truncate": truncate, "beta_fast": 32, "beta_slow": 1})
    assert all(abs(f[i].item() / w - 1) < 1e-12 for i, w in want.items())
    if truncate:
        assert torch.equal(f, frequencies(YARN)[0])


@pytest.mark.parametrize("keys,want", [({}, 1.368887945411393630), ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0), ({"mscale": 0.707, "mscale_all_dim": 0.707}, 1.0),
                                       ({"mscale": 1.0, "mscale_all_dim": 0.707}, 1.085726399256135652), ({"mscale": 1.0, "mscale_all_dim": 0}, 1.368887945411393630),
                                       ({"attention_factor": 1.25, "mscale": 1.0, "mscale_all_dim": 1.0}, 1.25), ({"attention_factor": None}, 1.368887945411393630)])
def test_yarn_factor_on_cosine_and_sine(keys, want):
    _, m = frequencies({**YARN, "factor": 40, **keys})
    assert abs(m / want - 1) < 1e-14


def test_factor_of_one():
    f, m = frequencies({**YARN, "factor": 1.0, "mscale": 2.0, "mscale_all_dim": 0.5})
    assert m == 1.0 and torch.allclose(f, frequencies(None)[0], rtol=1e-14)


@pytest.mark.parametrize("scaling", [{**YARN, "mscale": 1.0}, {**YARN, "mscale_all_dim": 1.0}, {**YARN, "scaling_beta": 0.1}, {**YARN, "short_factor": [1.0]},
                                     {"rope_type": "default", "factor": 2.0}, {"rope_type": "linear", "factor": 2.0, "attention_factor": 1.5},
                                     {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                      "original_max_position_embeddings": 8192, "beta_fast": 16}, {"rope_type": "default", "rope_theta": 1e6},
                                     {"rope_type": "longrope", "factor": 2.0}])
def test_keys_that_would_change_the_result_are_refused(scaling):
    with pytest.raises(RuntimeError, match="rope_frequencies"):
        frequencies(scaling)


def test_keys_beside_it():
    f, m = frequencies(None)
    same = {"rope_type": "default", "rope_theta": 150000.0, "partial_rotary_factor": 0.25, "mrope_section": [11, 11, 10], "mrope_interleaved": True, "factor": None}
    g, n = frequencies(same)
    assert torch.equal(f, g) and m == n == 1.0
    f, _ = frequencies({"type": "linear", "factor": 4.0, "original_max_position_embeddings": 4096, "finetuned": True})
    assert torch.equal(f, frequencies(None)[0] / 4)

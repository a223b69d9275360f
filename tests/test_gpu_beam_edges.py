"""Beam search at the edges of its arguments' ranges, against the definition in 64 bits (np_beam.py)."""
import math

import numpy as np
import pytest

from tests import np_beam as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def s(lib):
    from born_b200 import Sampler
    with Sampler(device=0, max_batch=512, max_vocab=262144) as h:
        yield h


def test_beams_that_go_on_are_normalised_as_the_pool(s):
    """score / length^length_penalty in 64 bits, rounded once: equal scores are equal wherever they come from."""
    import torch
    from born_b200 import BeamConfig, BeamSearch
    N, K, V = 32, 16, 300
    z = torch.randn((N * K, V), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for penalty in (1.0, 0.7):
        search = BeamSearch(s, N, K, 3, V, BeamConfig(length_penalty=penalty))
        search.begin()
        for _ in range(3):
            search.step(z)
        got = search.result()["scores"].cpu().numpy()
        norm = np.float64(3) ** np.float64(np.float32(penalty))
        want = (search.scores.cpu().numpy().astype(np.float64) / norm).astype(np.float32).reshape(N, K)
        assert np.array_equal(got, -np.sort(-want, axis=1))


def test_length_penalties_beyond_all_numbers(s):
    """length^length_penalty is infinite: every score is (negative) zero, the beams keep their order."""
    import torch
    from born_b200 import BeamConfig, BeamSearch
    N, K, V = 2, 4, 100
    search = BeamSearch(s, N, K, 4, V, BeamConfig(length_penalty=600.0))
    search.begin()
    for t in range(4):
        search.step(torch.randn((N * K, V), device="cuda"))
    found = search.result()
    assert (found["scores"] == 0).all() and (found["lens"] == 4).all()
    assert torch.equal(found["tokens"][:, :, 3], search.tokens.view(N, K))

"""The example that takes a search's passages through 4-bit projections, cache and attention."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


def test_answer_step(gpu):
    import answer_step

    similarity = answer_step.main(num_docs=64, batch=3, k=2, steps=4)
    # Three quantisations to 4 bits, each of about 10 % of a Gaussian row's norm,
    # and the output projection's: less than a quarter of the norm in all.
    assert float(similarity.mean()) > 1 - 0.25**2 / 2

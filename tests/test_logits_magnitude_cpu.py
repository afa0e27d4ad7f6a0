"""Rows of large magnitude and small temperatures in the CPU mode (tests/logits_magnitude_cases.py)."""

import numpy as np
import pytest

from numba_cuda_amd import simulator
from tests import logits_magnitude_cases as cases


@pytest.mark.parametrize("name", ["float32", "bfloat16"])
@pytest.mark.parametrize("picked", ["ORDINARY", "STEEP", "BORDER"])
def test_cpu_mode(name, picked):
    rng = np.random.default_rng(6)
    for kind, magnitude, temperature in getattr(cases, picked):
        if name == "bfloat16" and kind == "about":           # steps of float32
            continue
        cases.check(simulator, name, [cases.rows_of(kind, magnitude, temperature, 301, rng)], temperature)

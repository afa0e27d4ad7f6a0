"""Rows of large magnitude and small temperatures on the device (tests/logits_magnitude_cases.py)."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import numba_cuda_amd as cuda
from tests import logits_magnitude_cases as cases


def _lines(picked, vocab, seed):
    rng = np.random.default_rng(seed)
    by = {}
    for kind, magnitude, temperature in picked:
        by.setdefault(temperature, []).append(cases.rows_of(kind, magnitude, temperature, vocab, rng))
    return by


# rows of a wavefront, of a workgroup, and spread over several
@pytest.mark.parametrize("vocab", [1009, 9001, 60011, 100003])
@pytest.mark.parametrize("name", ["float32", "bfloat16"])
def test_large_magnitudes(name, vocab):
    for temperature, lines in _lines(cases.ORDINARY, vocab, 1).items():
        cases.check(cuda, name, lines, temperature)


@pytest.mark.parametrize("vocab", [1009, 9001, 60011, 100003])
def test_small_temperatures(vocab):
    for temperature, lines in _lines(cases.STEEP, vocab, 2).items():
        cases.check(cuda, "float32", lines, temperature)


@pytest.mark.parametrize("vocab", [700, 20011])
def test_small_temperatures_of_float16(vocab):
    for temperature, lines in _lines([("small temperature", 1.0, 1e-9), ("small temperature", 1.0, 1e-6),
                                      ("peaks", 6e4, 1e-3), ("masked", 6e4, 1e-3), ("falling", 8000.0, 1e-3),
                                      ("begins masked", 6e4, 1e-4)], vocab, 3).items():
        cases.check(cuda, "float16", lines, temperature)


@pytest.mark.parametrize("vocab", [1009, 9001, 60011, 100003])
def test_about_the_border(vocab):
    for temperature, lines in _lines(cases.BORDER, vocab, 4).items():
        cases.check(cuda, "float32", lines, temperature)


# many rows: small workgroups in the order of memory (loss, gradient), 256 and 512 lanes a row (both)
@pytest.mark.parametrize("picked", ["ORDINARY", "STEEP", "BORDER"])
def test_many_rows(picked):
    for temperature, lines in _lines(getattr(cases, picked), 27001, 5).items():
        cases.check(cuda, "float32", lines, temperature, copies=-(-1300 // len(lines)))

"""An empty history or no biases, as an empty list: NumPy makes float64 of it, which stands for no integers."""

import numpy as np
import pytest

from numba_cuda_amd import simulator
from numba_cuda_amd.kernels import logits as gpu_logits

X = np.arange(80, dtype=np.float32).reshape(2, 40)
NONE = dict(tokens=[], offsets=[0, 0, 0], repetition=2.0, presence=1.0, bias_tokens=(), bias_values=[],
            bias_offsets=[0, 0, 0])


def test_cpu_mode():
    assert np.array_equal(simulator.logits.adjust(X, **NONE).copy_to_host(), X)
    loss, lse = simulator.logits.distill_loss(X, np.zeros((2, 0), np.float32), [[], []])
    assert not loss.copy_to_host().any() and np.isfinite(lse.copy_to_host()).all()


def test_gpu_mode_on_a_stand_in(fake_gpu, monkeypatch):
    launched = []
    monkeypatch.setattr(fake_gpu, "nbh_logits_adjust", lambda *a: launched.append(a) or 0, raising=False)
    gpu_logits.adjust(X, **NONE)
    assert len(launched) == 1
    with pytest.raises(TypeError, match="unsupported dtype float64"):       # an array says what it is
        gpu_logits.adjust(X, **{**NONE, "tokens": np.zeros(0)})
    with pytest.raises(TypeError, match="unsupported dtype float64"):
        simulator.logits.adjust(X, **{**NONE, "tokens": np.zeros(0)})


@pytest.mark.gpu
def test_on_the_device():
    assert np.array_equal(gpu_logits.adjust(X, **NONE).copy_to_host(), X)
    loss, lse = gpu_logits.distill_loss(X, np.zeros((2, 0), np.float32), [[], []])
    assert not loss.copy_to_host().any()
    # 40 terms a few roundings each, 6 of the result
    want = np.log(np.exp(X.astype(np.float64) - 79).sum(1)) + 79
    assert (np.abs(lse.copy_to_host() - want) <= 2.0 ** -24 * (60 + 6 * np.abs(want))).all()

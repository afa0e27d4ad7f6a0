"""The imaginary part of a conjugated tensor lies negated in memory."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from numba_cuda_amd import logits


def test_weights_that_are_an_imaginary_part():
    torch = pytest.importorskip("torch")
    x, v = torch.randn(3, 50, device="cuda"), torch.randn(3, 2, device="cuda")
    i = torch.tensor([[1, 2], [3, 4], [0, 49]], device="cuda")
    pairs = torch.randn(3, dtype=torch.complex64, device="cuda")
    torch.cuda.synchronize()
    want = logits.distill_loss_and_grad(pairs.imag.contiguous(), x, v, i)[2].copy_to_host()
    assert np.array_equal(logits.distill_loss_and_grad(pairs.imag, x, v, i)[2].copy_to_host(), want)
    for _ in range(2):
        with pytest.raises(TypeError, match="resolve_neg"):
            logits.distill_loss_and_grad(pairs.conj().imag, x, v, i)
        with pytest.raises(TypeError, match="resolve_neg"):
            logits.distill_loss_and_grad(pairs.conj().imag[:1], x[:1], v[:1], i[:1])
    got = logits.distill_loss_and_grad(torch.resolve_neg(pairs.conj().imag), x, v, i)[2].copy_to_host()
    assert np.array_equal(got, -want)

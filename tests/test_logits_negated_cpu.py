"""Tensors whose memory holds the negated values (the imaginary part of a conjugated tensor, say) are refused: the
operators read memory."""

import ctypes

import pytest

from numba_cuda_amd.kernels import logits


class Tensor:
    """What the operators ask a tensor for; its class is known by its name."""

    is_cuda = True

    def __init__(self, shape, strides, negated, dtype="torch.float32"):
        self.shape, self._strides, self.negated, self.dtype = shape, strides, negated, dtype
        self._memory = (ctypes.c_double * 512)()

    def stride(self):
        return self._strides

    def data_ptr(self):
        return (ctypes.addressof(self._memory) + 15) // 16 * 16

    def is_neg(self):
        return self.negated


@pytest.fixture(autouse=True)
def tables(fake_gpu, monkeypatch):
    for table in logits._TABLES:                 # the stand-in's class and dtype go again
        for key in (Tensor, "torch.float32", "torch.int32"):
            monkeypatch.setitem(table, key, None)
            monkeypatch.delitem(table, key)
    monkeypatch.setattr(logits, "_foreign_dtypes", {})
    monkeypatch.setattr(logits, "_several_devices", False)
    for name in ("nbh_logits_adjust", "nbh_rows_distill"):
        monkeypatch.setattr(fake_gpu, name, lambda *a: 0, raising=False)
    monkeypatch.setattr(fake_gpu, "nbh_rows_distill_workspace", lambda *a: 0, raising=False)


def test_weights_of_every_other_item():
    x, v = Tensor((3, 8), (8, 1), False), Tensor((3, 2), (2, 1), False)
    i = Tensor((3, 2), (2, 1), False, "torch.int32")
    for _ in range(2):                           # the second time the native path knows the class
        logits.distill_loss_and_grad(Tensor((3,), (2,), False), x, v, i)
        with pytest.raises(TypeError, match="resolve_neg"):
            logits.distill_loss_and_grad(Tensor((3,), (2,), True), x, v, i)


@pytest.mark.parametrize("strides", [(2,), (7,)])
def test_one_item(strides):
    x, t, o = Tensor((1, 8), (8, 1), False), Tensor((4,), (1,), False, "torch.int32"), Tensor((2,), (1,), False, "torch.int32")
    for _ in range(2):
        logits.adjust(x, tokens=t, offsets=o, presence=Tensor((1,), strides, False))
        with pytest.raises(TypeError, match="resolve_neg"):
            logits.adjust(x, tokens=t, offsets=o, presence=Tensor((1,), strides, True))


def test_one_column():
    for _ in range(2):
        logits.adjust(Tensor((4, 1), (2, 2), False))
        with pytest.raises(TypeError, match="resolve_neg"):
            logits.adjust(Tensor((4, 1), (2, 2), True))

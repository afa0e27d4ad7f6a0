"""Rows upside down, repeated and overlapping one another, for every operator: the results are those of the same rows
laid out in the ordinary way, bit for bit (the order of every sum goes by sizes and alignment, and these are alike)."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import numba_cuda_amd as cuda
from numba_cuda_amd import logits
from numba_cuda_amd.cudadrv import devicearray


def upside_down(a):
    """The device's rows of `a` from the last to the first."""
    d = cuda.to_device(np.ascontiguousarray(a[::-1]))
    step = a.shape[1] * a.itemsize
    return devicearray.DeviceNDArray(a.shape, (-step, a.itemsize), a.dtype, gpu_data=d.gpu_data.view((len(a) - 1) * step))


def repeated(row, rows):
    d = cuda.to_device(row)
    return devicearray.DeviceNDArray((rows, len(row)), (0, row.itemsize), row.dtype, gpu_data=d.gpu_data)


def windows(line, rows, columns, step):
    """Row r begins r * step items into `line`."""
    d = cuda.to_device(line)
    return devicearray.DeviceNDArray((rows, columns), (step * line.itemsize, line.itemsize), line.dtype, gpu_data=d.gpu_data)


def host(d):
    """The rows of a result upside down, read from the memory they lie in."""
    base = devicearray.DeviceNDArray(d.shape, (-d.strides[0], d.strides[1]), d.dtype,
                                     gpu_data=_beginning(d))
    return base.copy_to_host()[::-1]


def _beginning(d):
    address = d.device_ctypes_pointer.value + (d.shape[0] - 1) * d.strides[0]
    from numba_cuda_amd.cudadrv.driver import MemoryPointer
    return MemoryPointer(cuda.current_context(), address, size=d.shape[0] * -d.strides[0], owner=d)


# rows of a multiple of 16 bytes, so that alignment is alike
SHAPES = [(5, 1200), (3, 9008), (4, 70016), (130, 20000), (520, 24576)]


@pytest.mark.parametrize("rows, vocab", SHAPES)
def test_adjust(rows, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    mask = rng.integers(0, 2 ** 32, (rows, (vocab + 31) // 32), dtype=np.uint64).astype(np.uint32)
    tokens = cuda.to_device(rng.integers(0, vocab, rows * 50).astype(np.int32))
    kw = dict(tokens=tokens, offsets=cuda.to_device(np.arange(rows + 1) * 50), repetition=1.5, frequency=0.25)
    want = logits.adjust(cuda.to_device(x), mask=cuda.to_device(mask), **kw).copy_to_host()
    out = upside_down(np.full_like(x, 7))
    logits.adjust(upside_down(x), out, mask=upside_down(mask), **kw)
    assert np.array_equal(host(out), want)
    own = upside_down(x)
    logits.adjust(own, own, mask=upside_down(mask), **kw)
    assert np.array_equal(host(own), want)
    got = logits.adjust(repeated(x[1], rows), mask=repeated(mask[2], rows), **kw).copy_to_host()
    same = cuda.to_device(np.repeat(x[1:2], rows, 0))
    assert np.array_equal(got, logits.adjust(same, mask=cuda.to_device(np.repeat(mask[2:3], rows, 0)), **kw).copy_to_host())


@pytest.mark.parametrize("rows, vocab", SHAPES)
def test_top(rows, vocab):
    rng = np.random.default_rng(vocab + 1)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    want = [a.copy_to_host() for a in logits.top(cuda.to_device(x), 20, lse=True)]
    v, i = upside_down(np.zeros((rows, 20), np.float32)), upside_down(np.zeros((rows, 20), np.int32))
    lse = logits.top(upside_down(x), 20, values=v, indices=i, lse=True)[2]
    assert np.array_equal(host(v), want[0]) and np.array_equal(host(i), want[1])
    assert np.array_equal(lse.copy_to_host(), want[2])
    line = rng.standard_normal(vocab + 4 * rows).astype(np.float32)
    there = logits.top(windows(line, rows, vocab, 4), 20, lse=True)
    apart = np.lib.stride_tricks.as_strided(line, (rows, vocab), (16, 4))
    for got, expected in zip(there, logits.top(cuda.to_device(np.ascontiguousarray(apart)), 20, lse=True)):
        assert np.array_equal(got.copy_to_host(), expected.copy_to_host())


@pytest.mark.parametrize("rows, vocab", SHAPES)
def test_distill(rows, vocab):
    rng = np.random.default_rng(vocab + 2)
    x, t = rng.standard_normal((rows, vocab)).astype(np.float32), rng.standard_normal((rows, 8)).astype(np.float32)
    i = rng.integers(-1, vocab, (rows, 8))
    g = rng.random(rows).astype(np.float32)
    dg, backwards = cuda.to_device(g), cuda.to_device(g[::-1].copy())
    dg_up = devicearray.DeviceNDArray((rows,), (-4,), np.float32, gpu_data=backwards.gpu_data.view((rows - 1) * 4))
    dx, dt, di = (cuda.to_device(a) for a in (x, t, i))
    want = [a.copy_to_host() for a in logits.distill_loss_and_grad(dg, dx, dt, di)]
    up = [upside_down(a) for a in (x, t, i)]
    out = upside_down(np.full_like(x, 7))
    loss, lse, _ = logits.distill_loss_and_grad(dg_up, *up, out=out)
    assert np.array_equal(loss.copy_to_host(), want[0]) and np.array_equal(lse.copy_to_host(), want[1])
    assert np.array_equal(host(out), want[2])
    alone = logits.distill_loss(dx, dt, di)
    for got, expected in zip(logits.distill_loss(*up), alone):
        assert np.array_equal(got.copy_to_host(), expected.copy_to_host())
    gradient = logits.distill_grad(dg, dx, dt, di, lse).copy_to_host()
    logits.distill_grad(dg_up, *up, lse, out=up[0])
    assert np.array_equal(host(up[0]), gradient)
    # one student and one teacher for all rows, and rows that overlap
    one = [repeated(a[1], rows) for a in (x, t, i)]
    each = [cuda.to_device(np.repeat(a[1:2], rows, 0)) for a in (x, t, i)]
    for got, expected in zip(logits.distill_loss_and_grad(dg, *one), logits.distill_loss_and_grad(dg, *each)):
        assert np.array_equal(got.copy_to_host(), expected.copy_to_host())
    line = rng.standard_normal(vocab + 4 * rows).astype(np.float32)
    apart = np.ascontiguousarray(np.lib.stride_tricks.as_strided(line, (rows, vocab), (16, 4)))
    for got, expected in zip(logits.distill_loss_and_grad(dg, windows(line, rows, vocab, 4), dt, di),
                             logits.distill_loss_and_grad(dg, cuda.to_device(apart), dt, di)):
        assert np.array_equal(got.copy_to_host(), expected.copy_to_host())

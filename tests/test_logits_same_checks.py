"""The CPU mode of the row operators refuses and takes what the GPU mode does: both are given the same calls (the
GPU mode on a stand-in library that launches nothing)."""

import numpy as np
import pytest

import numba_cuda_amd as cuda
from numba_cuda_amd import simulator
from numba_cuda_amd.kernels import logits as gpu_logits

LAUNCHES = ("nbh_logits_adjust", "nbh_rows_top", "nbh_rows_distill")


class Device:
    logits = gpu_logits
    to_device = staticmethod(cuda.to_device)


@pytest.fixture(params=["device", "host"])
def api(request, fake_gpu, monkeypatch):
    for name in LAUNCHES:
        monkeypatch.setattr(fake_gpu, name, lambda *a: 0, raising=False)
    for name in ("nbh_rows_top_workspace", "nbh_rows_distill_workspace"):
        monkeypatch.setattr(fake_gpu, name, lambda *a: 0, raising=False)
    return Device if request.param == "device" else simulator


def buffer(api, n=4096):
    return api.to_device(np.zeros(n, np.float32))


def part(block, first, shape, dtype=np.float32):
    """`shape` items of `dtype` of the block, from its float `first` on."""
    dtype = np.dtype(dtype)
    n = int(np.prod(shape)) * dtype.itemsize // 4
    return block[first:first + n].view(dtype).reshape(shape)


def f32(api, *shape):
    return api.to_device(np.zeros(shape, np.float32))


def i32(api, *shape):
    return api.to_device(np.zeros(shape, np.int32))


def test_adjust_refuses_results_that_touch_other_arguments(api):
    block = buffer(api)
    x, out = f32(api, 2, 40), part(block, 100, (2, 40))
    history = dict(tokens=i32(api, 10), offsets=i32(api, 3))
    pairs = dict(bias_tokens=i32(api, 10), bias_values=f32(api, 10), bias_offsets=i32(api, 3))
    refused = [
        ("the history or the penalties", dict(history, tokens=part(block, 95, (10,), np.int32))),
        ("the history or the penalties", dict(history, offsets=part(block, 179, (3,), np.int32))),
        ("the history or the penalties", dict(history, prompt_lengths=part(block, 120, (2,), np.int32))),
        ("the history or the penalties", dict(history, repetition=part(block, 99, (2,)))),
        ("the history or the penalties", dict(history, presence=part(block, 140, (2,)))),
        ("the history or the penalties", dict(history, frequency=part(block, 178, (2,)))),
        ("the biases", dict(pairs, bias_tokens=part(block, 91, (10,), np.int32))),
        ("the biases", dict(pairs, bias_values=part(block, 170, (10,)))),
        ("the biases", dict(pairs, bias_offsets=part(block, 98, (3,), np.int32))),
        ("mask", dict(mask=part(block, 97, (2, 2), np.int32))),
        ("mask", dict(mask=part(block, 99, (2,), np.int32))),
        ("mask", dict(mask=part(block, 179, (2, 2), np.uint32)))]
    for name, kw in refused:
        with pytest.raises(ValueError, match="out overlaps " + name):
            api.logits.adjust(x, out, **kw)
    with pytest.raises(ValueError, match="out overlaps logits"):
        api.logits.adjust(part(block, 60, (2, 40)), out)
    wide = f32(api, 2, 60)
    with pytest.raises(ValueError, match="out overlaps logits"):
        api.logits.adjust(wide[:, :40], wide[:, 10:50])
    with pytest.raises(ValueError, match="out overlaps logits"):             # the same place, another type
        api.logits.adjust(part(block, 100, (2, 40), np.float16), out)
    # on either side, beside, and in place
    api.logits.adjust(x, out, mask=part(block, 96, (2, 2), np.int32), tokens=part(block, 90, (6,), np.int32),
                      offsets=part(block, 180, (3,), np.int32))
    api.logits.adjust(wide[:, :20], wide[:, 20:40])
    api.logits.adjust(wide[:, :20], wide[:, :20])


def test_results_whose_rows_touch_each_other(api):
    block = buffer(api)
    once = block[:40].reshape(1, 40)
    rows = _repeated(api, once, 3)
    x = f32(api, 3, 40)
    with pytest.raises(ValueError, match="rows of out overlap"):
        api.logits.adjust(x, rows)
    with pytest.raises(ValueError, match="rows of values overlap"):
        api.logits.top(x, 40, values=rows)
    v, i = f32(api, 3, 2), i32(api, 3, 2)
    with pytest.raises(ValueError, match="rows of out overlap"):
        api.logits.distill_loss_and_grad(1.0, x, v, i, out=rows)
    api.logits.adjust(rows, x)                   # as an input they may


def _repeated(api, row, times):
    if api is simulator:
        return type(row)(np.lib.stride_tricks.as_strided(row._ary, (times, row.shape[1]), (0, 4)))
    from numba_cuda_amd.cudadrv import devicearray
    return devicearray.DeviceNDArray((times, row.shape[1]), (0, 4), row.dtype, gpu_data=row.gpu_data)


def test_top_and_distill_refuse_results_that_touch_other_arguments(api):
    block = buffer(api)
    x, v, i, g = part(block, 0, (2, 40)), part(block, 100, (2, 3)), part(block, 200, (2, 3), np.int32), f32(api, 2)
    for name, kw in (("values overlaps logits", dict(values=part(block, 70, (2, 5)))),
                     ("indices overlaps logits", dict(indices=part(block, 79, (2, 5), np.int32))),
                     ("lse overlaps logits", dict(lse=part(block, 3, (2,)))),
                     ("values overlaps indices", dict(values=part(block, 300, (2, 5)),
                                                      indices=part(block, 309, (2, 5), np.int32)))):
        with pytest.raises(ValueError, match=name):
            api.logits.top(x, 5, **kw)
    op = api.logits
    for name, call, kw in (("loss overlaps student", op.distill_loss, dict(loss=part(block, 79, (2,)))),
                           ("lse overlaps values", op.distill_loss, dict(lse=part(block, 105, (2,)))),
                           ("loss overlaps lse", op.distill_loss, dict(loss=g, lse=g)),
                           ("loss overlaps indices", op.distill_loss, dict(loss=part(block, 200, (2,)))),
                           ("lse overlaps teacher_lse", op.distill_loss, dict(lse=g, teacher_lse=g))):
        with pytest.raises(ValueError, match=name):
            call(x, v, i, **kw)
    for name, kw in (("out overlaps values", dict(out=part(block, 90, (2, 40)))),
                     ("out overlaps student", dict(out=part(block, 1, (2, 40)))),
                     ("out overlaps indices", dict(out=part(block, 190, (2, 40))))):
        with pytest.raises(ValueError, match=name):
            op.distill_loss_and_grad(g, x, v, i, **kw)
    weights = part(block, 500, (2,))
    with pytest.raises(ValueError, match="out overlaps grad_loss"):
        op.distill_loss_and_grad(weights, x, v, i, out=part(block, 450, (2, 40)))
    with pytest.raises(ValueError, match="out overlaps lse"):
        op.distill_grad(1.0, x, v, i, weights, out=part(block, 450, (2, 40)))
    op.distill_loss_and_grad(g, x, v, i, out=x)


def test_device_arrays_of_other_types_and_strides(api):
    x, t, o = f32(api, 2, 40), i32(api, 5), i32(api, 3)
    double = api.to_device(np.ones(2))
    v, i = f32(api, 2, 3), i32(api, 2, 3)
    op = api.logits
    for call, args, kw in ((op.adjust, (x,), dict(tokens=t, offsets=o, presence=double)),
                           (op.distill_loss, (x, v, i), dict(teacher_lse=double)),
                           (op.distill_loss_and_grad, (double, x, v, i), {}),
                           (op.distill_grad, (1.0, x, v, i, double), {})):
        with pytest.raises(TypeError, match="unsupported dtype float64"):
            call(*args, **kw)
    for kw in (dict(tokens=i32(api, 10)[::2], offsets=o), dict(tokens=t, offsets=i32(api, 6)[::2]),
               dict(tokens=t, offsets=o, presence=f32(api, 4)[::2])):
        with pytest.raises(ValueError, match="unit stride"):
            op.adjust(x, **kw)
    with pytest.raises(ValueError, match="next to each other"):
        op.adjust(x, mask=i32(api, 2, 4)[:, ::2])
    with pytest.raises(TypeError, match="32-bit"):
        op.adjust(x, mask=api.to_device(np.ones((2, 2), np.int64)))
    with pytest.raises(TypeError, match="values has dtype"):
        op.top(x, 1, values=api.to_device(np.zeros((2, 1), np.float16)))
    with pytest.raises(TypeError, match="out has dtype"):
        op.distill_loss_and_grad(1.0, x, v, i, out=api.to_device(np.zeros((2, 40), np.float16)))
    op.distill_loss_and_grad(f32(api, 4)[::2], x, v, i)      # of any stride


def test_arrays_off_their_alignment(api):
    raw = api.to_device(np.zeros(401, np.uint8))
    off = raw[1:401].view(np.float32)
    with pytest.raises(ValueError, match="logits is not aligned"):
        api.logits.top(off.reshape(2, 50), 1)
    with pytest.raises(ValueError, match="presence is not aligned"):
        api.logits.adjust(f32(api, 2, 40), tokens=i32(api, 3), offsets=i32(api, 3), presence=off[:2])


def test_host_inputs_of_any_strides_and_lists(api):
    x = np.zeros((40, 2), np.float32).T
    api.logits.adjust(x, tokens=np.zeros(10, np.int64)[::2], offsets=[0, 1, 2], presence=[1.0, 2.0])
    v, i = f32(api, 2, 3), i32(api, 2, 3)
    api.logits.distill_grad([1.0, 2.0], x, v, i, [0.5, 0.25], teacher_lse=(1, 2))


def test_workspaces(api):
    x = f32(api, 2, 40)
    api.logits.top(x, 1, workspace=f32(api, 64))
    with pytest.raises(TypeError, match="workspace must be a device array"):
        api.logits.top(x, 1, workspace=np.zeros(64, np.float32))
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        api.logits.top(x, 1, workspace=f32(api, 64)[::2])
    with pytest.raises(ValueError, match="aligned to 16"):
        api.logits.distill_loss(x, f32(api, 2, 3), i32(api, 2, 3), workspace=f32(api, 64)[1:])

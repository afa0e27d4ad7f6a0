"""A call that is recorded into a graph takes nothing from host memory: every replay would copy from what
the call no longer holds."""

import numpy as np
import pytest

import numba_cuda_amd as cuda
from numba_cuda_amd.kernels import logits


def _f32(*shape):
    return cuda.to_device(np.zeros(shape, np.float32))


def _i32(*shape):
    return cuda.to_device(np.zeros(shape, np.int32))


ADJUST = [("logits", {}), ("tokens", dict(tokens=[1, 2, 3])), ("offsets", dict(offsets=np.array([0, 1, 2]))),
          ("prompt_lengths", dict(prompt_lengths=[0, 1])), ("repetition", dict(repetition=[1.0, 1.5])),
          ("presence", dict(presence=np.ones(2, np.float32))), ("frequency", dict(frequency=(0.5, 0.25))),
          ("bias_tokens", dict(bias_tokens=[1, 2, 3, 4, 5])), ("bias_values", dict(bias_values=[1.0] * 5)),
          ("bias_offsets", dict(bias_offsets=[0, 1, 2])), ("mask", dict(mask=np.zeros((2, 2), np.int32)))]


@pytest.fixture
def recording(fake_gpu, monkeypatch):
    """The fake library with a stream that is being captured: (library, stream)."""
    monkeypatch.setattr(fake_gpu, "nbh_logits_adjust", lambda *a: fake_gpu._log("nbh_logits_adjust") or 0, raising=False)
    monkeypatch.setattr(fake_gpu, "nbh_rows_top_workspace", lambda *a: 0, raising=False)
    monkeypatch.setattr(fake_gpu, "nbh_rows_distill_workspace", lambda *a: 0, raising=False)
    for name in ("nbh_rows_top", "nbh_rows_distill"):
        monkeypatch.setattr(fake_gpu, name, lambda *a, n=name: fake_gpu._log(n) or 0, raising=False)
    stream = cuda.stream()

    def capturing(handle, out):
        out._obj.value = 1 if handle else 0
        return 0
    monkeypatch.setattr(fake_gpu, "nbh_stream_is_capturing", capturing, raising=False)
    yield fake_gpu, stream


def _refused(lib, name, call, *args, **kw):
    before = len(lib.calls)
    with pytest.raises(ValueError, match="captured into a graph needs %s in device memory" % name):
        call(*args, **kw)
    assert not [c for c in lib.calls[before:] if "alloc" in c[0] or "memcpy" in c[0] or "rows" in c[0] or "adjust" in c[0]]


@pytest.mark.parametrize("name, given", ADJUST, ids=[a[0] for a in ADJUST])
def test_adjust(recording, name, given):
    lib, stream = recording
    x, out = _f32(2, 40), _f32(2, 40)
    kw = dict(tokens=_i32(3), offsets=_i32(3), prompt_lengths=_i32(2), repetition=1.5, presence=_f32(2),
              frequency=0.25, bias_tokens=_i32(5), bias_values=_f32(5), bias_offsets=_i32(3), mask=_i32(2, 2))
    logits.adjust(x, out, stream=stream, **kw)       # from the device: taken
    assert lib.calls[-1][0] == "nbh_logits_adjust"
    kw.update(given)
    _refused(lib, name, logits.adjust, np.zeros((2, 40), np.float32) if name == "logits" else x, out, stream=stream, **kw)
    if name != "logits":                             # not captured: copied over, as ever
        logits.adjust(x, out, **kw)


def test_top(recording):
    lib, stream = recording
    v, i = _f32(2, 3), _i32(2, 3)
    logits.top(_f32(2, 40), 3, values=v, indices=i, stream=stream)
    _refused(lib, "logits", logits.top, np.zeros((2, 40), np.float32), 3, values=v, indices=i, stream=stream)


@pytest.mark.parametrize("name", ["student", "values", "indices", "teacher_lse", "grad_loss", "lse"])
def test_distill(recording, name):
    lib, stream = recording
    host = dict(student=np.zeros((2, 40), np.float32), values=np.zeros((2, 3), np.float32),
                indices=np.zeros((2, 3), np.int64), teacher_lse=[1.0, 2.0], grad_loss=[0.5, 0.5], lse=[1.0, 1.0])
    a = dict(student=_f32(2, 40), values=_f32(2, 3), indices=_i32(2, 3), teacher_lse=_f32(2), grad_loss=_f32(2),
             lse=_f32(2))
    out, loss = _f32(2, 40), _f32(2)

    def gradient(a):
        logits.distill_grad(a["grad_loss"], a["student"], a["values"], a["indices"], a["lse"],
                            teacher_lse=a["teacher_lse"], out=out, stream=stream)

    def both(a):
        logits.distill_loss_and_grad(a["grad_loss"], a["student"], a["values"], a["indices"],
                                     teacher_lse=a["teacher_lse"], loss=loss, lse=a["lse"], out=out, stream=stream)

    gradient(a)
    both(a)
    a[name] = host[name]
    _refused(lib, name, gradient, a)
    if name != "lse":                                # a result there
        _refused(lib, name, both, a)

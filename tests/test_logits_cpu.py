"""The operators over rows of logits without a GPU: the CPU mode against the float64 oracle, the
oracle's gradient against differences, host conversions, and every refusal of the GPU mode (its
checks come before any kernel; the driver is a stand-in that has none)."""

import numpy as np
import pytest

import numba_cuda_amd as cuda
from numba_cuda_amd import simulator
from numba_cuda_amd._logits_host import bfloat16, from_bfloat16, to_bfloat16
from numba_cuda_amd.cudadrv import devicearray
from numba_cuda_amd.kernels import logits
from oracle import logits64
from tests import logits_cases as cases


# ---- the CPU mode --------------------------------------------------------------------------

@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("rows, vocab, longest, pairs, mask", [
    (1, 1, 1, 0, None), (3, 7, 20, 3, "rows"), (5, 100, 300, 40, "shared"), (6, 33, 0, 0, "rows")])
def test_adjust(name, rows, vocab, longest, pairs, mask):
    cases.check_adjust(simulator, rows, vocab, name, name, longest, pairs, mask)
    cases.check_adjust(simulator, rows, vocab, name, "float32", longest, pairs, mask, index="int64", per_row=False)


@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("rows, vocab, k", [(1, 1, 1), (9, 30, 30), (3, 300, 5)])
def test_top(name, rows, vocab, k):
    cases.check_top(simulator, rows, vocab, name, k)
    cases.check_top(simulator, rows, vocab, name, k, kind="edge", temperature=0.7)


@pytest.mark.parametrize("name", cases.DTYPES)
@pytest.mark.parametrize("what", ["loss", "both", "apart"])
def test_distill(name, what):
    cases.check_distill(simulator, 6, 50, name, 7, what=what)
    cases.check_distill(simulator, 6, 50, name, 7, what=what, temperature=2.0, full=True, teacher=name, index="int64")
    cases.check_distill(simulator, 6, 20, name, 30, what=what, repeated=True)
    cases.check_distill(simulator, 9, 41, name, 5, what=what, kind="edge")


def test_cpu_mode_refuses_what_the_gpu_mode_refuses():
    x = simulator.to_device(np.zeros((2, 8), np.float32))
    with pytest.raises(ValueError, match="tokens and offsets come together"):
        simulator.logits.adjust(x, tokens=np.zeros(3, np.int32))
    with pytest.raises(ValueError, match="k must be between"):
        simulator.logits.top(x, 9)
    with pytest.raises(TypeError, match="device array"):
        simulator.logits.top(x, 2, values=np.zeros((2, 2), np.float32))
    with pytest.raises(ValueError, match="temperature"):
        simulator.logits.top(x, 2, temperature=0)


# ---- the oracle ----------------------------------------------------------------------------

@pytest.mark.parametrize("full", [False, True])
def test_oracle_gradient_against_differences(full):
    rng = np.random.default_rng(5)
    x, values = rng.standard_normal((3, 11)), rng.standard_normal((3, 4))
    indices = np.array([[0, 3, 3, 10], [5, -1, 2, 1], [-1, -1, 11, -1]])
    norm = np.log(np.exp(values / 1.5).sum(1) + 1) if full else None
    weights = np.array([1.0, -0.5, 2.0])
    _, _, grad = logits64.distill(x, values, indices, 1.5, norm, weights)
    step = 1e-6
    for r in range(3):
        for v in range(11):
            ends = []
            for sign in (1, -1):
                moved = x.copy()
                moved[r, v] += sign * step
                ends.append((logits64.distill(moved, values, indices, 1.5, norm)[0] * weights).sum())
            # central differences: third derivatives below 1, rounding 1e-16 / step
            assert abs((ends[0] - ends[1]) / (2 * step) - grad[r, v]) < 1e-8


def test_bfloat16_conversions():
    x = np.float32([1, 1.00390625, 1.01171875, 3.4e38, np.inf, -np.inf, -0.0, 1e-40])
    got = from_bfloat16(to_bfloat16(x))
    want = np.float32([1, 1, 1.015625, np.inf, np.inf, -np.inf, -0.0, 1e-40])
    assert np.array_equal(got[:7], want[:7]) and np.signbit(got[6]) and abs(got[7] - 1e-40) <= 2.0 ** -134
    assert np.isnan(from_bfloat16(to_bfloat16(np.float32([np.nan])))[0])
    assert to_bfloat16(x.reshape(2, 4)).shape == (2, 4) and to_bfloat16(x).dtype == bfloat16


# ---- refusals of the GPU mode ----------------------------------------------------------------

def _f32(*shape):
    return cuda.to_device(np.zeros(shape, np.float32))


def _i32(*shape):
    return cuda.to_device(np.zeros(shape, np.int32))


def test_adjust_refusals(fake_gpu):
    x = _f32(2, 40)
    t, o = _i32(5), _i32(3)
    refused = [
        (ValueError, "2-d", (_f32(40),), {}),
        (TypeError, "unsupported dtype float64", (cuda.to_device(np.zeros((2, 4))),), {}),
        (ValueError, "next to each other", (_f32(40, 2)[:, ::2].reshape(40, 1) if False else _f32(4, 8)[:, ::2],), {}),
        (ValueError, "come together", (x,), dict(tokens=t)),
        (ValueError, "come together", (x,), dict(offsets=o)),
        (ValueError, "need tokens", (x,), dict(repetition=1.2)),
        (ValueError, "need tokens", (x,), dict(prompt_lengths=_i32(2))),
        (ValueError, "expected 3", (x,), dict(tokens=t, offsets=_i32(2))),
        (TypeError, "unsupported dtype", (x,), dict(tokens=_f32(5), offsets=o)),
        (ValueError, "1-d", (x,), dict(tokens=_i32(5, 1), offsets=o)),
        (ValueError, "unit stride", (x,), dict(tokens=_i32(10)[::2], offsets=o)),
        (ValueError, "expected 2", (x,), dict(tokens=t, offsets=o, prompt_lengths=_i32(3))),
        (ValueError, "positive", (x,), dict(tokens=t, offsets=o, repetition=0)),
        (ValueError, "finite", (x,), dict(tokens=t, offsets=o, presence=float("nan"))),
        (ValueError, "expected 2", (x,), dict(tokens=t, offsets=o, frequency=_f32(5))),
        (ValueError, "come together", (x,), dict(bias_tokens=t, bias_values=_f32(5))),
        (ValueError, "expected 5", (x,), dict(bias_tokens=t, bias_values=_f32(4), bias_offsets=o)),
        (TypeError, "32-bit", (x,), dict(mask=cuda.to_device(np.ones((2, 40), bool)))),
        (ValueError, "40 entries need 2", (x,), dict(mask=_i32(2, 1))),
        (ValueError, "mask has shape", (x,), dict(mask=_i32(3, 2))),
        (ValueError, "next to each other", (x,), dict(mask=_i32(2, 4)[:, ::2])),
        (TypeError, "device array", (x, np.zeros((2, 40), np.float32)), {}),
        (ValueError, "expected", (x, _f32(2, 41)), {}),
        (TypeError, "out has dtype", (x, cuda.to_device(np.zeros((2, 40), np.float16))), {}),
        (TypeError, "Expected a Stream", (x,), dict(stream="s")),
    ]
    for error, text, args, kw in refused:
        with pytest.raises(error, match=text):
            logits.adjust(*args, **kw)
    # results that touch their input without being it, and rows that touch each other
    wide = _f32(2, 60)
    with pytest.raises(ValueError, match="out overlaps logits"):
        logits.adjust(wide[:, :40], wide[:, 10:50])
    once = devicearray.DeviceNDArray((2, 40), (0, 4), np.float32, gpu_data=x.gpu_data)
    with pytest.raises(ValueError, match="rows of out overlap"):
        logits.adjust(_f32(2, 40), once)
    half = cuda.to_device(np.zeros((2, 40), np.float16))
    assert not [c for c in fake_gpu.calls if c[0].startswith("nbh_logits")], half


def test_columns_beside_each_other_do_not_overlap():
    def block(start, n, pitch=100, rows=3, name="logits"):
        return 4096 + 4 * start, rows, 4 * n, 4 * pitch, name

    def check(one, other, same=None):
        logits._refuse_overlaps([(*one[:4], "out")], [other], same=same)
    check(block(0, 40), block(40, 60))
    check(block(40, 60), block(0, 40))
    for start, n in ((39, 10), (0, 40), (30, 5), (90, 20)):
        with pytest.raises(ValueError, match="out overlaps logits"):
            check(block(0, 40), block(start, n, rows=4))
    x = block(0, 40)
    check(block(0, 40), x, same=x)
    for other in (block(0, 40, pitch=99), block(0, 80), block(1, 40)):      # another pitch, type or start
        with pytest.raises(ValueError):
            check(other, x, same=x)


def test_top_refusals(fake_gpu):
    x = _f32(2, 40)
    refused = [
        (ValueError, "between 1 and 40", (x, 0), {}),
        (ValueError, "between 1 and 40", (x, 41), {}),
        (ValueError, "between 1 and 1024", (_f32(1, 2000), 1025), {}),
        (ValueError, "between 1 and 0", (_f32(2, 0), 1), {}),
        (TypeError, "integer", (x, 1.0), {}),
        (TypeError, "integer", (x, True), {}),
        (ValueError, "temperature", (x, 1), dict(temperature=0)),
        (ValueError, "temperature", (x, 1), dict(temperature=-1.0)),
        (ValueError, "temperature", (x, 1), dict(temperature=float("inf"))),
        (TypeError, "unsupported dtype", (_i32(2, 40), 1), {}),
        (TypeError, "device array", (x, 1), dict(indices=np.zeros((2, 1), np.int32))),
        (TypeError, "unsupported dtype", (x, 1), dict(indices=cuda.to_device(np.zeros((2, 1), np.int64)))),
        (TypeError, "values has dtype", (x, 1), dict(values=cuda.to_device(np.zeros((2, 1), np.float16)))),
        (ValueError, "expected", (x, 2), dict(values=_f32(2, 3))),
        (ValueError, "expected 2", (x, 2), dict(lse=_f32(3))),
        (ValueError, "values overlaps logits", (x, 2), dict(values=x[:, :2])),
    ]
    for error, text, args, kw in refused:
        with pytest.raises(error, match=text):
            logits.top(*args, **kw)


def test_distill_refusals(fake_gpu):
    x, v, i, g = _f32(2, 40), _f32(2, 3), _i32(2, 3), _f32(2)
    both, loss, grad = logits.distill_loss_and_grad, logits.distill_loss, logits.distill_grad
    refused = [
        (ValueError, "2-d", loss, (_f32(40), v, i), {}),
        (ValueError, "2-d", loss, (x, _f32(3), i), {}),
        (ValueError, "indices has shape", loss, (x, v, _i32(2, 4)), {}),
        (ValueError, "values has 3 rows", loss, (x, _f32(3, 3), _i32(3, 3)), {}),
        (TypeError, "unsupported dtype", loss, (x, v, v), {}),
        (TypeError, "unsupported dtype", loss, (x, i, i), {}),
        (ValueError, "1024", loss, (x, _f32(2, 1025), _i32(2, 1025)), {}),
        (ValueError, "temperature", loss, (x, v, i), dict(temperature=0)),
        (ValueError, "expected 2", loss, (x, v, i), dict(teacher_lse=_f32(3))),
        (ValueError, "expected 2", loss, (x, v, i), dict(loss=_f32(1))),
        (ValueError, "loss overlaps values", loss, (x, v, i), dict(loss=v[0, :2])),
        (ValueError, "loss overlaps lse", loss, (x, v, i), dict(loss=g, lse=g)),
        (ValueError, "grad_loss has shape", both, (_f32(3), x, v, i), {}),
        (ValueError, "grad_loss", both, (float("nan"), x, v, i), {}),
        (TypeError, "grad_loss", both, (i[:, 0], x, v, i), {}),
        (TypeError, "out has dtype", both, (g, x, v, i), dict(out=cuda.to_device(np.zeros((2, 40), np.float16)))),
        (ValueError, "out overlaps values", both, (g, x, _f32(2, 40)[:, :3], i), dict(out=None)),
        (ValueError, "expected 2", grad, (g, x, v, i, _f32(3)), {}),
    ]
    for error, text, call, args, kw in refused:
        if "out overlaps values" in text:
            home = _f32(2, 40)
            args, kw = (g, x, home[:, :3], i), dict(out=home)
        with pytest.raises(error, match=text):
            call(*args, **kw)


def test_memory_of_another_device_is_refused(fake_gpu, monkeypatch):
    def pointer_device(address, out):
        out._obj.value = 1
        return 0
    monkeypatch.setattr(logits, "_several_devices", True)
    monkeypatch.setattr(fake_gpu, "nbh_pointer_device", pointer_device, raising=False)
    with pytest.raises(ValueError, match="logits is on device 1, the current device is 0"):
        logits.top(_f32(2, 40), 1)


def test_a_captured_call_needs_its_own_arrays(fake_gpu, monkeypatch):
    def capturing(stream, out):
        out._obj.value = 1
        return 0
    monkeypatch.setattr(fake_gpu, "nbh_stream_is_capturing", capturing, raising=False)
    monkeypatch.setattr(fake_gpu, "nbh_rows_top_workspace", lambda *a: 4096, raising=False)
    stream = cuda.stream()
    x, v, i = _f32(2, 40), _f32(2, 1), _i32(2, 1)
    with pytest.raises(ValueError, match="needs its values array"):
        logits.top(x, 1, stream=stream)
    with pytest.raises(ValueError, match="needs a workspace of 4096 bytes"):
        logits.top(x, 1, values=v, indices=i, stream=stream)
    with pytest.raises(ValueError, match="must hold 4096 bytes"):
        logits.top(x, 1, values=v, indices=i, stream=stream, workspace=_f32(10))


def test_the_entry_points_check_their_arguments():
    from numba_cuda_amd import _lib
    lib = _lib.load()
    assert lib.nbh_logits_adjust(None, None) != 0
    assert lib.nbh_logits_adjust(logits._ADJUST.pack(8, *([0] * 29)), None) != 0            # another structure
    empty = [logits._ADJUST.size] + [0] * 29
    assert lib.nbh_logits_adjust(logits._ADJUST.pack(*empty), None) == 0                    # no rows
    assert lib.nbh_rows_top(None, 1, 10, 40, 0, 1, None, 4, None, 4, None, 1.0, None, 0, None) != 0
    assert lib.nbh_rows_top(None, 0, 10, 40, 0, 1, None, 4, None, 4, None, 1.0, None, 0, None) == 0
    assert lib.nbh_rows_top(None, 0, 10, 40, 0, 11, None, 4, None, 4, None, 1.0, None, 0, None) != 0
    assert lib.nbh_rows_top(None, 0, 10, 40, 0, 1, None, 4, None, 4, None, 0.0, None, 0, None) != 0
    assert lib.nbh_rows_distill(logits._DISTILL.pack(8, *([0] * 24)), None) != 0
    # long rows are spread over workgroups, short ones are not
    assert lib.nbh_rows_top_workspace(1, 131072, 50, 0) > 0 == lib.nbh_rows_top_workspace(4096, 1000, 50, 0)
    assert lib.nbh_rows_distill_workspace(1, 1310720, 8, 2, 1) > 0 == lib.nbh_rows_distill_workspace(1, 131072, 8, 2, 2)


def test_results_may_not_touch_any_other_argument(fake_gpu, monkeypatch):
    launched = []
    monkeypatch.setattr(fake_gpu, "nbh_logits_adjust", lambda *a: launched.append(a) or 0, raising=False)
    block = cuda.to_device(np.zeros(4096, np.float32))

    def part(first, shape, dtype):
        strides = tuple(np.zeros(shape, dtype).strides)
        return devicearray.DeviceNDArray(shape, strides, np.dtype(dtype), gpu_data=block[first:].gpu_data)

    x, out = _f32(2, 40), part(100, (2, 40), np.float32)                 # floats 100 .. 179 of the block
    tokens, offsets, values = _i32(10), _i32(3), _f32(10)
    for kw in (dict(tokens=part(95, (10,), np.int32), offsets=offsets), dict(tokens=tokens, offsets=part(179, (3,), np.int32)),
               dict(tokens=tokens, offsets=offsets, prompt_lengths=part(120, (2,), np.int32)),
               dict(tokens=tokens, offsets=offsets, repetition=part(99, (2,), np.float32)),
               dict(tokens=tokens, offsets=offsets, presence=part(140, (2,), np.float32)),
               dict(tokens=tokens, offsets=offsets, frequency=part(178, (2,), np.float32))):
        with pytest.raises(ValueError, match="out overlaps the history or the penalties"):
            logits.adjust(x, out, **kw)
    for kw in (dict(bias_tokens=part(91, (10,), np.int32), bias_values=values, bias_offsets=offsets),
               dict(bias_tokens=tokens, bias_values=part(170, (10,), np.float32), bias_offsets=offsets),
               dict(bias_tokens=tokens, bias_values=values, bias_offsets=part(98, (3,), np.int32))):
        with pytest.raises(ValueError, match="out overlaps the biases"):
            logits.adjust(x, out, **kw)
    for mask in (part(97, (2, 2), np.int32), part(99, (2,), np.int32), part(179, (2, 2), np.int32)):
        with pytest.raises(ValueError, match="out overlaps mask"):
            logits.adjust(x, out, mask=mask)
    assert not launched
    # on either side of it
    logits.adjust(x, out, tokens=part(90, (10,), np.int32), offsets=part(180, (3,), np.int32), mask=part(96, (2, 2), np.int32))
    assert len(launched) == 1


def test_a_workspace_may_not_touch_the_other_arguments(fake_gpu, monkeypatch):
    monkeypatch.setattr(fake_gpu, "nbh_rows_top_workspace", lambda *a: 64, raising=False)
    monkeypatch.setattr(fake_gpu, "nbh_rows_distill_workspace", lambda *a: 64, raising=False)
    x, v, i = _f32(2, 40), _f32(2, 3), _i32(2, 3)
    with pytest.raises(ValueError, match="workspace overlaps logits"):
        logits.top(x, 3, workspace=x)
    with pytest.raises(ValueError, match="workspace overlaps student"):
        logits.distill_loss(x, v, i, workspace=x)

"""The operators over the rows of logits (numba_cuda_amd/kernels/logits.py) in the CPU mode:
float32 arithmetic row by row over NumPy arrays, the same names, arguments and checks."""

import math

import numpy as np

from numba_cuda_amd._logits_host import bfloat16, from_bfloat16, to_bfloat16
from numba_cuda_amd.simulator.hostarray import device_array

MOST = 1024
_f32 = np.float32
_ROW_DTYPES = (np.dtype(np.float32), np.dtype(np.float16), bfloat16)


def _host(obj, dtype=None):
    return np.asarray(getattr(obj, "_ary", obj), dtype=dtype)


def _rows(obj, name, shape=None, dtypes=_ROW_DTYPES):
    a = _host(obj)
    if a.ndim != 2:
        raise ValueError("%s must be a 2-d array, got %d-d" % (name, a.ndim))
    if a.dtype not in dtypes:
        raise TypeError("%s has unsupported dtype %s" % (name, a.dtype))
    if shape is not None and a.shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, a.shape, shape))
    if a.shape[1] > 1 and a.strides[1] != a.dtype.itemsize:
        raise ValueError("the items of a row of %s must lie next to each other (strides %s)" % (name, a.strides))
    return a


def _vector(obj, name, length, dtypes, dtype=None):
    a = _host(obj, dtype)
    if a.ndim != 1:
        raise ValueError("%s must be a 1-d array, got %d-d" % (name, a.ndim))
    if a.dtype not in [np.dtype(d) for d in dtypes]:
        raise TypeError("%s has unsupported dtype %s" % (name, a.dtype))
    if length is not None and a.shape[0] != length:
        raise ValueError("%s has %d items, expected %d" % (name, a.shape[0], length))
    return a


_INTEGERS = (np.int32, np.int64)


def _values(a):
    return from_bfloat16(a) if a.dtype == bfloat16 else a.astype(_f32)


def _store(a, row, x):
    a[row] = to_bfloat16(x) if a.dtype == bfloat16 else x.astype(a.dtype)


def _result(obj, name, shape, dtype, stream):
    if obj is None or obj is True:
        obj = device_array(shape, dtype=dtype, stream=stream)
    elif not getattr(obj, "__cuda_ndarray__", False):
        raise TypeError("%s must be a device array" % name)
    return obj


def _number(value, name, low=None, high=None):
    value = float(value)
    if not math.isfinite(value) or (low is not None and not low <= value <= high):
        raise ValueError("%s must be %s, got %r" % (
            name, "a finite number" if low is None else "between %g and %g" % (low, high), value))
    return value


def _is_number(value):
    return isinstance(value, (int, float, np.number))


def _per_row(value, name, rows, number):
    if value is None:
        return np.full(rows, number, _f32)
    if _is_number(value):
        value = _number(value, name)
        if name == "repetition" and value <= 0:
            raise ValueError("repetition must be positive, got %r" % value)
        return np.full(rows, value, _f32)
    return _vector(value, name, rows, (np.float32,), np.float32)


def _cut(values, offsets, row):
    begin = min(max(int(offsets[row]), 0), len(values))
    return begin, min(max(int(offsets[row + 1]), begin), len(values))


@np.errstate(all="ignore")
def adjust(logits, out=None, *, tokens=None, offsets=None, prompt_lengths=None, repetition=None, presence=None,
           frequency=None, bias_tokens=None, bias_values=None, bias_offsets=None, mask=None, stream=0):
    x = _rows(logits, "logits")
    rows, vocab = x.shape
    if (tokens is None) != (offsets is None):
        raise ValueError("tokens and offsets come together")
    if tokens is None and any(v is not None for v in (prompt_lengths, repetition, presence, frequency)):
        raise ValueError("penalties and prompt lengths need tokens and offsets")
    if len({bias_tokens is None, bias_values is None, bias_offsets is None}) != 1:
        raise ValueError("bias_tokens, bias_values and bias_offsets come together")
    out = _result(out, "out", x.shape, x.dtype, stream)
    y = _rows(out, "out", x.shape)
    if y.dtype != x.dtype and y.dtype != np.dtype(np.float32):
        raise TypeError("out has dtype %s, expected %s or float32" % (y.dtype, x.dtype))
    prompts = None
    if tokens is not None:
        tokens = _vector(tokens, "tokens", None, _INTEGERS)
        offsets = _vector(offsets, "offsets", rows + 1, _INTEGERS)
        if prompt_lengths is not None:
            prompts = _vector(prompt_lengths, "prompt_lengths", rows, _INTEGERS)
    repetition = _per_row(repetition, "repetition", rows, 1.0)
    presence = _per_row(presence, "presence", rows, 0.0)
    frequency = _per_row(frequency, "frequency", rows, 0.0)
    if bias_tokens is not None:
        bias_tokens = _vector(bias_tokens, "bias_tokens", None, _INTEGERS)
        bias_values = _vector(bias_values, "bias_values", len(bias_tokens), (np.float32,), np.float32)
        bias_offsets = _vector(bias_offsets, "bias_offsets", rows + 1, _INTEGERS)
    if mask is not None:
        mask = _host(mask)
        if mask.dtype.kind not in "iu" or mask.dtype.itemsize != 4:
            raise TypeError("mask has dtype %s, expected 32-bit integers" % mask.dtype)
        if mask.ndim not in (1, 2) or (mask.ndim == 2 and mask.shape[0] not in (1, rows)):
            raise ValueError("mask has shape %s, expected one row of words or %d" % (mask.shape, rows))
        if mask.shape[-1] * 32 < vocab:
            raise ValueError("mask has %d words, %d entries need %d" % (mask.shape[-1], vocab, -(-vocab // 32)))
        mask = np.broadcast_to(mask, (rows, mask.shape[-1]))
    for r in range(rows):
        line = _values(x[r])
        if tokens is not None:
            begin, end = _cut(tokens, offsets, r)
            made = begin + (min(max(int(prompts[r]), 0), end - begin) if prompts is not None else 0)
            history = tokens[begin:end]
            seen = np.zeros(vocab, bool)
            seen[history[(history >= 0) & (history < vocab)]] = True
            line = np.where(seen, np.where(line > 0, line / repetition[r], line * repetition[r]), line)
            history = tokens[made:end]
            count = np.bincount(history[(history >= 0) & (history < vocab)], minlength=vocab)
            line = np.where(count > 0, line - frequency[r] * count.astype(_f32) - presence[r], line)
        if bias_tokens is not None:
            begin, end = _cut(bias_tokens, bias_offsets, r)
            last = {int(v): b for v, b in zip(bias_tokens[begin:end], bias_values[begin:end]) if 0 <= v < vocab}
            for v, b in last.items():
                line[v] += b
        if mask is not None:
            v = np.arange(vocab)
            line = np.where((mask[r].view(np.uint32)[v >> 5] >> (v & 31).astype(np.uint32)) & 1, line, _f32(-np.inf))
        _store(y, r, line)
    return out


def _softmax(x, temperature):
    """(peak, sum of exp((x - peak) / temperature)) with a finite peak."""
    limit = np.finfo(_f32).max
    peak = _f32(np.clip(np.fmax.reduce(x, initial=_f32(-limit)), -limit, limit))
    return peak, np.exp((x - peak) / temperature).sum(dtype=_f32)


def _temperature(value):
    return _f32(_number(value, "temperature", 1e-30, 1e30))


def top_workspace(rows, vocab, k, dtype):
    return 0


@np.errstate(all="ignore")
def top(logits, k, *, values=None, indices=None, lse=None, temperature=1.0, workspace=None, stream=0):
    x = _rows(logits, "logits")
    rows, vocab = x.shape
    if isinstance(k, bool) or not isinstance(k, (int, np.integer)):
        raise TypeError("k must be an integer, got %s" % type(k).__name__)
    if not 1 <= k <= min(vocab, MOST):
        raise ValueError("k must be between 1 and %d, got %d" % (min(vocab, MOST), k))
    temperature = _temperature(temperature)
    values = _result(values, "values", (rows, k), x.dtype, stream)
    indices = _result(indices, "indices", (rows, k), np.int32, stream)
    v = _rows(values, "values", (rows, k), (x.dtype,))
    i = _rows(indices, "indices", (rows, k), (np.dtype(np.int32),))
    z = None
    if lse is not None and lse is not False:
        lse = _result(lse, "lse", (rows,), np.float32, stream)
        z = _vector(lse, "lse", rows, (np.float32,))
    for r in range(rows):
        line = _values(x[r]) + _f32(0)
        order = np.lexsort((np.arange(vocab), -line, ~np.isnan(line)))[:k]
        v[r], i[r] = x[r][order], order
        if z is not None:
            peak, total = _softmax(line, temperature)
            z[r] = peak / temperature + np.log(total)
    return (values, indices) if z is None else (values, indices, lse)


def distill_workspace(rows, vocab, k, dtype, *, loss=True, grad=False):
    return 0


@np.errstate(all="ignore")
def _distill(with_loss, with_grad, grad_loss, student, values, indices, temperature, teacher_lse, loss, lse, out,
             stream):
    x = _rows(student, "student")
    rows, vocab = x.shape
    v = _rows(values, "values")
    i = _rows(indices, "indices", v.shape, tuple(np.dtype(d) for d in _INTEGERS))
    if v.shape[0] != rows:
        raise ValueError("values has %d rows, student has %d" % (v.shape[0], rows))
    if v.shape[1] > MOST:
        raise ValueError("a row of values may hold %d entries, got %d" % (MOST, v.shape[1]))
    temperature = _temperature(temperature)
    if teacher_lse is not None:
        teacher_lse = _vector(teacher_lse, "teacher_lse", rows, (np.float32,), np.float32)
    if with_grad:
        if _is_number(grad_loss):
            grad_loss = np.full(rows, _number(grad_loss, "grad_loss"), _f32)
        grad_loss = _host(grad_loss, np.float32)
        if grad_loss.shape != (rows,):
            raise ValueError("grad_loss has shape %s, expected (%d,)" % (grad_loss.shape, rows))
        out = _result(out, "out", x.shape, x.dtype, stream)
        y = _rows(out, "out", x.shape, (x.dtype,))
    if with_loss:
        loss = _result(loss, "loss", (rows,), np.float32, stream)
        lse = _result(lse, "lse", (rows,), np.float32, stream)
        losses = _vector(loss, "loss", rows, (np.float32,))
    norms = _vector(lse, "lse", rows, (np.float32,))
    for r in range(rows):
        line = _values(x[r])
        t, at = _values(v[r]), i[r]
        there = (at >= 0) & (at < vocab) & (t != -np.inf)
        t, at = t[there], at[there]
        if teacher_lse is not None:
            log_p = t / temperature - teacher_lse[r]
        else:
            peak, total = _softmax(t, temperature)
            log_p = (t - peak) / temperature - np.log(total)
        p = np.exp(log_p)
        if with_loss:
            peak, total = _softmax(line, temperature)
            norms[r] = peak / temperature + np.log(total)
            q = np.exp((line - peak) / temperature) / (total if total else _f32(1))
            log_q = np.where(line[at] == -np.inf, line[at], (line[at] - peak) / temperature - np.log(total))
            losses[r] = np.where(p != 0, p * (log_p - log_q), _f32(0)).sum(dtype=_f32)
        elif norms[r] == -np.inf:
            q = np.zeros(vocab, _f32)
        else:
            # the difference in float64: in float32 the quotient alone is off by far more than one for large logits
            q = np.exp(line / np.float64(temperature) - np.float64(norms[r])).astype(_f32)
        if with_grad:
            factor = grad_loss[r] / temperature
            if not len(at) or factor == 0:
                grad = np.zeros(vocab, _f32)
            else:
                grad = factor * p.sum(dtype=_f32) * q
                np.add.at(grad, at, -factor * p)
            _store(y, r, grad)
    return loss, lse, out


def distill_loss(student, values, indices, *, temperature=1.0, teacher_lse=None, loss=None, lse=None, workspace=None,
                 stream=0):
    return _distill(True, False, None, student, values, indices, temperature, teacher_lse, loss, lse, None, stream)[:2]


def distill_grad(grad_loss, student, values, indices, lse, *, temperature=1.0, teacher_lse=None, out=None,
                 workspace=None, stream=0):
    return _distill(False, True, grad_loss, student, values, indices, temperature, teacher_lse, None, lse, out,
                    stream)[2]


def distill_loss_and_grad(grad_loss, student, values, indices, *, temperature=1.0, teacher_lse=None, loss=None,
                          lse=None, out=None, workspace=None, stream=0):
    return _distill(True, True, grad_loss, student, values, indices, temperature, teacher_lse, loss, lse, out, stream)

"""The operators over the rows of logits (numba_cuda_amd/kernels/logits.py) in the CPU mode:
float32 arithmetic row by row over NumPy arrays, the same names, arguments and checks (a workspace
may be small: none is needed here)."""

import math

import numpy as np

from numba_cuda_amd._logits_host import bfloat16, from_bfloat16, host_array, refuse_overlaps, to_bfloat16
from numba_cuda_amd.simulator.hostarray import device_array

MOST = 1024
_f32 = np.float32
_ROW_DTYPES = (np.dtype(np.float32), np.dtype(np.float16), bfloat16)
_INTEGERS = (np.dtype(np.int32), np.dtype(np.int64))
_FLOATS = (np.dtype(np.float32),)


def _array(obj, dtype=None):
    """The NumPy array of an argument; of an input on the host a compact one, as a copy over is."""
    if getattr(obj, "__cuda_ndarray__", False):
        return obj._ary
    return host_array(obj, dtype)


def _address(a):
    return a.__array_interface__["data"][0]


def _aligned(a, name):
    if _address(a) % a.dtype.itemsize or (a.shape[0] > 1 and a.strides[0] % a.dtype.itemsize):
        raise ValueError("%s is not aligned to its item size" % name)
    return a


def _rows(obj, name, shape=None, dtypes=_ROW_DTYPES, output=False):
    a = _array(obj)
    if a.ndim != 2:
        raise ValueError("%s must be a 2-d array, got %d-d" % (name, a.ndim))
    if a.dtype not in dtypes:
        raise TypeError("%s has unsupported dtype %s" % (name, a.dtype))
    if a.shape[1] > 1 and a.strides[1] != a.dtype.itemsize:
        raise ValueError("the items of a row of %s must lie next to each other (strides %s)" % (name, a.strides))
    _aligned(a, name)
    if shape is not None and a.shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, a.shape, shape))
    if output and a.shape[0] > 1 and a.shape[1] and abs(a.strides[0]) < a.shape[1] * a.dtype.itemsize:
        raise ValueError("the rows of %s overlap (%d bytes from one to the next)" % (name, a.strides[0]))
    return a


def _vector(obj, name, length, dtypes, dtype=None):
    a = _array(obj, dtype)
    if a.ndim != 1:
        raise ValueError("%s must be a 1-d array, got %d-d" % (name, a.ndim))
    if a.dtype not in dtypes:
        raise TypeError("%s has unsupported dtype %s" % (name, a.dtype))
    if length is not None and a.shape[0] != length:
        raise ValueError("%s has %d items, expected %d" % (name, a.shape[0], length))
    if a.shape[0] > 1 and a.strides[0] != a.dtype.itemsize:
        raise ValueError("%s must have unit stride" % name)
    return _aligned(a, name)


def _block(a, name):
    """What refuse_overlaps takes: of rows, or of a vector as one row."""
    if a.ndim == 2:
        return (_address(a), a.shape[0], a.shape[1] * a.dtype.itemsize, a.strides[0] if a.shape[0] > 1 else 0, name)
    return _address(a), 1, a.shape[0] * a.dtype.itemsize, 0, name


def _workspace(given):
    if given is None:
        return
    if not getattr(given, "__cuda_ndarray__", False):
        raise TypeError("workspace must be a device array")
    a = given._ary
    if a.size and not a.flags.c_contiguous:
        raise ValueError("workspace must be contiguous")
    if _address(a) % 16:
        raise ValueError("workspace must be aligned to 16")


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


def _per_row(value, name, rows, number, arrays):
    if value is None:
        return np.full(rows, number, _f32)
    if _is_number(value):
        value = _number(value, name)
        if name == "repetition" and value <= 0:
            raise ValueError("repetition must be positive, got %r" % value)
        return np.full(rows, value, _f32)
    arrays.append(_vector(value, name, rows, _FLOATS, np.float32))
    return arrays[-1]


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
    y = _rows(out, "out", x.shape, output=True)
    if y.dtype != x.dtype and y.dtype != np.dtype(np.float32):
        raise TypeError("out has dtype %s, expected %s or float32" % (y.dtype, x.dtype))
    block, same = _block(y, "out"), _block(x, "logits")
    refuse_overlaps([block], [same], same=same)
    prompts, history = None, []
    if tokens is not None:
        tokens = _vector(tokens, "tokens", None, _INTEGERS)
        offsets = _vector(offsets, "offsets", rows + 1, _INTEGERS)
        history += [tokens, offsets]
        if prompt_lengths is not None:
            prompts = _vector(prompt_lengths, "prompt_lengths", rows, _INTEGERS)
            history.append(prompts)
    repetition = _per_row(repetition, "repetition", rows, 1.0, history)
    presence = _per_row(presence, "presence", rows, 0.0, history)
    frequency = _per_row(frequency, "frequency", rows, 0.0, history)
    refuse_overlaps([block], [_block(a, "the history or the penalties") for a in history])
    if bias_tokens is not None:
        bias_tokens = _vector(bias_tokens, "bias_tokens", None, _INTEGERS)
        bias_values = _vector(bias_values, "bias_values", len(bias_tokens), _FLOATS, np.float32)
        bias_offsets = _vector(bias_offsets, "bias_offsets", rows + 1, _INTEGERS)
        refuse_overlaps([block], [_block(a, "the biases") for a in (bias_tokens, bias_values, bias_offsets)])
    if mask is not None:
        mask = _array(mask)
        if mask.dtype not in (np.dtype(np.int32), np.dtype(np.uint32)):
            raise TypeError("mask has dtype %s, expected 32-bit integers" % mask.dtype)
        if mask.ndim not in (1, 2) or (mask.ndim == 2 and mask.shape[0] not in (1, rows)):
            raise ValueError("mask has shape %s, expected one row of words or %d" % (mask.shape, rows))
        if mask.shape[-1] > 1 and mask.strides[-1] != 4:
            raise ValueError("the words of a mask must lie next to each other (strides %s)" % (mask.strides,))
        if mask.shape[-1] * 32 < vocab:
            raise ValueError("mask has %d words, %d entries need %d" % (mask.shape[-1], vocab, -(-vocab // 32)))
        mask = np.broadcast_to(mask, (rows, mask.shape[-1]))
        if rows and vocab:
            refuse_overlaps([block], [_block(mask[:, :(vocab + 31) // 32], "mask")])
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
    v = _rows(values, "values", (rows, k), output=True)
    if v.dtype != x.dtype:
        raise TypeError("values has dtype %s, expected %s" % (v.dtype, x.dtype))
    indices = _result(indices, "indices", (rows, k), np.int32, stream)
    i = _rows(indices, "indices", (rows, k), _INTEGERS[:1], output=True)
    results = [_block(v, "values"), _block(i, "indices")]
    z = None
    if lse is not None and lse is not False:
        lse = _result(lse, "lse", (rows,), np.float32, stream)
        z = _vector(lse, "lse", rows, _FLOATS)
        results.append(_block(z, "lse"))
    refuse_overlaps(results, [_block(x, "logits")])
    if rows:
        _workspace(workspace)
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
             workspace, stream):
    x = _rows(student, "student")
    rows, vocab = x.shape
    v = _rows(values, "values")
    i = _rows(indices, "indices", v.shape, _INTEGERS)
    if v.shape[0] != rows:
        raise ValueError("values has %d rows, student has %d" % (v.shape[0], rows))
    if v.shape[1] > MOST:
        raise ValueError("a row of values may hold %d entries, got %d" % (MOST, v.shape[1]))
    temperature = _temperature(temperature)
    same = _block(x, "student")
    inputs, results = [same, _block(v, "values"), _block(i, "indices")], []
    if teacher_lse is not None:
        teacher_lse = _vector(teacher_lse, "teacher_lse", rows, _FLOATS, np.float32)
        inputs.append(_block(teacher_lse, "teacher_lse"))
    if with_grad:
        if _is_number(grad_loss):
            grad_loss = np.full(rows, _number(grad_loss, "grad_loss"), _f32)
        grad_loss = _array(grad_loss, np.float32)
        if grad_loss.shape != (rows,):
            raise ValueError("grad_loss has shape %s, expected (%d,)" % (grad_loss.shape, rows))
        if grad_loss.dtype not in _FLOATS:
            raise TypeError("grad_loss has unsupported dtype %s" % grad_loss.dtype)
        _aligned(grad_loss, "grad_loss")
        inputs.append((_address(grad_loss), rows, 4, grad_loss.strides[0], "grad_loss"))
    if with_loss:
        loss = _result(loss, "loss", (rows,), np.float32, stream)
        lse = _result(lse, "lse", (rows,), np.float32, stream)
        losses = _vector(loss, "loss", rows, _FLOATS)
        norms = _vector(lse, "lse", rows, _FLOATS)
        results += [_block(losses, "loss"), _block(norms, "lse")]
    else:
        norms = _vector(lse, "lse", rows, _FLOATS, np.float32)
        inputs.append(_block(norms, "lse"))
    if with_grad:
        out = _result(out, "out", x.shape, x.dtype, stream)
        y = _rows(out, "out", x.shape, output=True)
        if y.dtype != x.dtype:
            raise TypeError("out has dtype %s, expected %s" % (y.dtype, x.dtype))
        results.append(_block(y, "out"))
    refuse_overlaps(results, inputs, same=same)
    if rows:
        _workspace(workspace)
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
    return _distill(True, False, None, student, values, indices, temperature, teacher_lse, loss, lse, None, workspace,
                    stream)[:2]


def distill_grad(grad_loss, student, values, indices, lse, *, temperature=1.0, teacher_lse=None, out=None,
                 workspace=None, stream=0):
    return _distill(False, True, grad_loss, student, values, indices, temperature, teacher_lse, None, lse, out,
                    workspace, stream)[2]


def distill_loss_and_grad(grad_loss, student, values, indices, *, temperature=1.0, teacher_lse=None, loss=None,
                          lse=None, out=None, workspace=None, stream=0):
    return _distill(True, True, grad_loss, student, values, indices, temperature, teacher_lse, loss, lse, out, workspace,
                    stream)

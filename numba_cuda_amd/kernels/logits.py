"""Operators over the rows of a 2-d array of logits (one row per position, one column per entry
of a vocabulary): `adjust`, `top`, and `distill_loss` / `distill_grad` / `distill_loss_and_grad`.
Not in the reference; they stand beside its reductions (numba_cuda/numba/cuda/kernels/reduction.py).

    from numba_cuda_amd import logits

    logits.adjust(x, out=x, tokens=history, offsets=starts, repetition=1.1, mask=grammar)
    values, indices = logits.top(x, 50)

    t, i, z = logits.top(teacher, 64, lse=True, temperature=2.0)
    loss, lse, grad = logits.distill_loss_and_grad(1.0 / rows, student, t, i, temperature=2.0)

Arrays are device arrays of this package or anything that exports __cuda_array_interface__ (torch
tensors included); inputs on the host are copied over first, as for any kernel here.  Logits are
float32, float16 or bfloat16, which NumPy has no type for: two-byte void items (`logits.bfloat16`,
the type string "<V2") are bfloat16.  Items of a row lie next to each other; rows may be any multiple
of the item size apart.  Arithmetic is float32, results are rounded once.

Everything is asynchronous on `stream`, and results do not depend on how the work was spread.  A call
that needs a workspace keeps one per stream; a call recorded into a graph takes the caller's
(`workspace=`, at least `top_workspace` / `distill_workspace` bytes) and the caller's result arrays,
since a graph may run beside later calls on its stream.
"""

import ctypes
import math
import struct

import numpy as np

from numba_cuda_amd._logits_host import bfloat16, from_bfloat16, to_bfloat16  # noqa: F401
from numba_cuda_amd.cudadrv import devicearray, devices
from numba_cuda_amd.cudadrv import driver as _driver

MOST = 1024                                  # NBH_ROW_TOP_MOST: entries `top` returns and the distillation takes

_F32, _F16, _BF16 = 0, 1, 2                  # enum nbh_row_dtype
_LOSS, _GRAD = 1, 2                          # enum nbh_distill_what
_float32, _int32, _int64 = np.dtype(np.float32), np.dtype(np.int32), np.dtype(np.int64)
_ROW_DTYPE = {_float32: _F32, np.dtype(np.float16): _F16, bfloat16: _BF16}

_ADJUST = struct.Struct("@qPP6q3P4q3P3d3P3qPq")       # struct nbh_logits_adjust_args
_DISTILL = struct.Struct("@qqP4q2P5q2Pqdd3PqPq")      # struct nbh_rows_distill_args


# ---- arguments ---------------------------------------------------------------------------

class _Array:
    """Address, shape, byte strides and dtype of an argument, and what keeps it alive."""

    __slots__ = ("address", "shape", "strides", "dtype", "owner")

    def __init__(self, address, shape, strides, dtype, owner):
        self.address, self.shape, self.strides, self.dtype, self.owner = address, shape, strides, dtype, owner


_foreign_dtypes = {}                         # dtype objects of other libraries -> np.dtype


def _foreign_dtype(dtype):
    name = str(dtype).rpartition(".")[2]
    try:
        found = bfloat16 if name == "bfloat16" else np.dtype(name)
    except TypeError:
        raise TypeError("unsupported dtype: %s" % (dtype,)) from None
    _foreign_dtypes[dtype] = found
    return found


def _device_view(obj):
    """The _Array of something in device memory, None for anything else."""
    if getattr(obj, "__cuda_ndarray__", False):
        return _Array(obj.device_ctypes_pointer.value or 0, obj.shape, obj.strides, obj.dtype, obj)
    if getattr(obj, "is_cuda", None) is True and hasattr(obj, "data_ptr"):
        # a torch tensor: its attributes cost a tenth of what its interface dictionary does
        dtype = _foreign_dtypes.get(obj.dtype) or _foreign_dtype(obj.dtype)
        size = dtype.itemsize
        return _Array(obj.data_ptr(), tuple(obj.shape), tuple([s * size for s in obj.stride()]), dtype, obj)
    if hasattr(obj, "__cuda_array_interface__"):
        array = devicearray.auto_device(obj)[0]
        return _Array(array.device_ctypes_pointer.value or 0, array.shape, array.strides, array.dtype, array)
    return None


_several_devices = None


def _checked_device(array, name):
    """Refuse memory of another device than the calling thread's."""
    global _several_devices
    if _several_devices is None:
        _several_devices = _driver.driver.get_device_count() > 1
    if _several_devices and array.address:
        where, here = ctypes.c_int(), ctypes.c_int()
        _driver.driver.nbh_get_device(ctypes.byref(here))
        _driver.driver.nbh_pointer_device(array.address, ctypes.byref(where))
        if where.value != here.value:
            raise ValueError("%s is on device %d, the current device is %d" % (name, where.value, here.value))
    return array


def _input(obj, name, stream, dtype=None):
    """The _Array of an input; what is on the host is copied over."""
    array = _device_view(obj)
    if array is None:
        host = np.asarray(obj) if dtype is None else np.asarray(obj, dtype=dtype)
        if not host.flags["C_CONTIGUOUS"]:
            host = np.ascontiguousarray(host)
        array = _device_view(devicearray.auto_device(host, stream=stream)[0])
    return _checked_device(array, name)


def _output(obj, name):
    array = _device_view(obj)
    if array is None:
        raise TypeError("%s must be a device array" % name)
    return _checked_device(array, name)


def _as_rows(array, name, shape=None, dtypes=_ROW_DTYPE):
    """Check a 2-d operand; returns the bytes from row to row."""
    if len(array.shape) != 2:
        raise ValueError("%s must be a 2-d array, got %d-d" % (name, len(array.shape)))
    if array.dtype not in dtypes:
        raise TypeError("%s has unsupported dtype %s" % (name, array.dtype))
    if shape is not None and array.shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, array.shape, shape))
    size = array.dtype.itemsize
    if array.shape[1] > 1 and array.strides[1] != size:
        raise ValueError("the items of a row of %s must lie next to each other (strides %s)" % (name, array.strides))
    if array.address % size or (array.shape[0] > 1 and array.strides[0] % size):
        raise ValueError("%s is not aligned to its item size" % name)
    return array.strides[0] if array.shape[0] > 1 else 0


def _as_result_rows(array, name, shape, dtypes=_ROW_DTYPE):
    stride = _as_rows(array, name, shape, dtypes)
    if shape[0] > 1 and shape[1] and abs(stride) < shape[1] * array.dtype.itemsize:
        raise ValueError("the rows of %s overlap (strides %s)" % (name, array.strides))
    return stride


def _as_vector(array, name, length, dtypes):
    if len(array.shape) != 1:
        raise ValueError("%s must be a 1-d array, got %d-d" % (name, len(array.shape)))
    if array.dtype not in dtypes:
        raise TypeError("%s has unsupported dtype %s" % (name, array.dtype))
    if length is not None and array.shape[0] != length:
        raise ValueError("%s has %d items, expected %d" % (name, array.shape[0], length))
    if array.shape[0] > 1 and array.strides[0] != array.dtype.itemsize:
        raise ValueError("%s must have unit stride" % name)
    if array.address % array.dtype.itemsize:
        raise ValueError("%s is not aligned to its item size" % name)
    return array


_INTEGERS = (_int32, _int64)
_FLOATS = (_float32,)


def _extent(array):
    low = high = array.address
    for n, s in zip(array.shape, array.strides):
        if n == 0:
            return low, low
        if s < 0:
            low += (n - 1) * s
        else:
            high += (n - 1) * s
    return low, high + array.dtype.itemsize


def _refuse_overlap(out, name, other, other_name, same=False):
    """ValueError when the result array touches an input; `same` allows the very same items."""
    if same and out.address == other.address and out.dtype == other.dtype and (
            out.shape[0] <= 1 or out.strides[0] == other.strides[0]):
        return
    low, high = _extent(out)
    other_low, other_high = _extent(other)
    if low >= high or other_low >= other_high or high <= other_low or other_high <= low:
        return
    # columns of one wider buffer may lie between each other without touching
    if len(out.shape) == len(other.shape) == 2 and out.strides[0] == other.strides[0] > 0:
        pitch = out.strides[0]
        gap = (other.address - out.address) % pitch
        if gap >= out.shape[1] * out.dtype.itemsize and gap + other.shape[1] * other.dtype.itemsize <= pitch:
            return
    raise ValueError("%s overlaps %s" % (name, other_name))


def _number(value, name, low=None, high=None):
    value = float(value)
    if not math.isfinite(value) or (low is not None and not low <= value <= high):
        raise ValueError("%s must be %s, got %r" % (
            name, "a finite number" if low is None else "between %g and %g" % (low, high), value))
    return value


def _temperature(value):
    return _number(value, "temperature", 1e-30, 1e30)


def _is_number(value):
    return isinstance(value, (int, float, np.number))


def _capturing(handle):
    if not handle:
        return False                         # the default stream cannot be captured
    flag = ctypes.c_int()
    _driver.driver.nbh_stream_is_capturing(handle, ctypes.byref(flag))
    return bool(flag.value)


def _new(shape, dtype, stream, handle, name):
    if _capturing(handle):
        raise ValueError("a call that is captured into a graph needs its %s array" % name)
    strides = (shape[1] * dtype.itemsize, dtype.itemsize) if len(shape) == 2 else (dtype.itemsize,)
    return devicearray.DeviceNDArray(shape, strides, dtype, stream=stream)


def _result(obj, name, shape, dtype, stream, handle):
    """(what the caller gets back, its _Array) for a result that may have been given."""
    if obj is None or obj is True:
        obj = _new(shape, dtype, stream, handle, name)
    return obj, _output(obj, name)


def _workspace(given, nbytes, handle):
    """(address, bytes, what keeps it alive)."""
    if given is not None:
        array = _output(given, "workspace")
        low, high = _extent(array)
        items = 1
        for n in array.shape:
            items *= n
        if items * array.dtype.itemsize != high - low:
            raise ValueError("workspace must be contiguous")
        if high - low < nbytes or low % 16:
            raise ValueError("workspace must hold %d bytes, aligned to 16" % nbytes)
        return low, high - low, array.owner
    if not nbytes:
        return 0, 0, None
    if _capturing(handle):
        raise ValueError("a call that is captured into a graph needs a workspace of %d bytes" % nbytes)
    return devices.get_context().workspace(handle, nbytes)


# ---- penalties, biases, masks --------------------------------------------------------------

def _per_row(value, name, rows, stream, number):
    """(address, value in its place, what keeps it alive) of a number or one number per row."""
    if value is None:
        return 0, number, None
    if _is_number(value):
        value = _number(value, name)
        if name == "repetition" and value <= 0:
            raise ValueError("repetition must be positive, got %r" % value)
        return 0, value, None
    array = _as_vector(_input(value, name, stream, np.float32), name, rows, _FLOATS)
    return array.address, number, array.owner


def adjust(logits, out=None, *, tokens=None, offsets=None, prompt_lengths=None, repetition=None, presence=None,
           frequency=None, bias_tokens=None, bias_values=None, bias_offsets=None, mask=None, stream=0):
    """Penalties for repeated tokens, biases and a mask on every row of `logits`; returns `out`.

    tokens, offsets : row r's history is tokens[offsets[r]:offsets[r + 1]] (int32 or int64, `offsets`
                      one longer than there are rows); tokens outside the vocabulary are skipped
    prompt_lengths  : how many of them, from the front, are the prompt (none if not given)
    repetition      : entries that occur in the history: x / repetition where x > 0, else x * repetition
    presence        : subtracted from entries that occur behind the prompt
    frequency       : times how often they do, subtracted first
    bias_tokens, bias_values, bias_offsets : added to the entries named, laid out like the history; of
                      several pairs for one entry the last counts
    mask            : bit v % 32 of word v // 32 tells whether entry v stays (else it becomes -inf); 32-bit
                      integers, one row of words per row of logits or a single one for all
    The three penalties are numbers or float32 arrays of one number per row.  In that order, each in
    float32.  `out` has the type of the logits or float32, and may be `logits` itself.
    """
    devices.get_context()
    handle = _driver._stream_handle(stream)
    x = _input(logits, "logits", stream)
    in_stride = _as_rows(x, "logits")
    rows, vocab = x.shape
    if (tokens is None) != (offsets is None):
        raise ValueError("tokens and offsets come together")
    if tokens is None and any(v is not None for v in (prompt_lengths, repetition, presence, frequency)):
        raise ValueError("penalties and prompt lengths need tokens and offsets")
    if len({bias_tokens is None, bias_values is None, bias_offsets is None}) != 1:
        raise ValueError("bias_tokens, bias_values and bias_offsets come together")

    out, y = _result(out, "out", x.shape, x.dtype, stream, handle)
    out_stride = _as_result_rows(y, "out", x.shape)
    if y.dtype != x.dtype and y.dtype != _float32:
        raise TypeError("out has dtype %s, expected %s or float32" % (y.dtype, x.dtype))
    _refuse_overlap(y, "out", x, "logits", same=True)

    t = o = p = None
    history = (0, 0, 0, 0, 4, 4, 4)
    if tokens is not None:
        t = _as_vector(_input(tokens, "tokens", stream), "tokens", None, _INTEGERS)
        o = _as_vector(_input(offsets, "offsets", stream), "offsets", rows + 1, _INTEGERS)
        if prompt_lengths is not None:
            p = _as_vector(_input(prompt_lengths, "prompt_lengths", stream), "prompt_lengths", rows, _INTEGERS)
        history = (t.address, o.address, p.address if p else 0, t.shape[0], t.dtype.itemsize, o.dtype.itemsize,
                   p.dtype.itemsize if p else 4)
    rep = _per_row(repetition, "repetition", rows, stream, 1.0)
    pre = _per_row(presence, "presence", rows, stream, 0.0)
    fre = _per_row(frequency, "frequency", rows, stream, 0.0)
    bt = bo = bv = None
    bias = (0, 0, 0, 0, 4, 4)
    if bias_tokens is not None:
        bt = _as_vector(_input(bias_tokens, "bias_tokens", stream), "bias_tokens", None, _INTEGERS)
        bv = _as_vector(_input(bias_values, "bias_values", stream, np.float32), "bias_values", bt.shape[0], _FLOATS)
        bo = _as_vector(_input(bias_offsets, "bias_offsets", stream), "bias_offsets", rows + 1, _INTEGERS)
        bias = (bt.address, bo.address, bv.address, bt.shape[0], bt.dtype.itemsize, bo.dtype.itemsize)
    m, mask_stride = None, 0
    if mask is not None:
        m = _input(mask, "mask", stream)
        if m.dtype.kind not in "iu" or m.dtype.itemsize != 4:
            raise TypeError("mask has dtype %s, expected 32-bit integers" % m.dtype)
        if len(m.shape) not in (1, 2) or (len(m.shape) == 2 and m.shape[0] not in (1, rows)):
            raise ValueError("mask has shape %s, expected one row of words or %d" % (m.shape, rows))
        if m.shape[-1] * 32 < vocab:
            raise ValueError("mask has %d words, %d entries need %d" % (m.shape[-1], vocab, -(-vocab // 32)))
        if m.shape[-1] > 1 and m.strides[-1] != 4:
            raise ValueError("the words of a mask must lie next to each other (strides %s)" % (m.strides,))
        if len(m.shape) == 2 and m.shape[0] > 1:
            mask_stride = m.strides[0]

    if rows and vocab:
        _driver.driver.nbh_logits_adjust(
            _ADJUST.pack(_ADJUST.size, x.address, y.address, rows, vocab, in_stride, out_stride, _ROW_DTYPE[x.dtype],
                         _ROW_DTYPE[y.dtype], *history, rep[0], pre[0], fre[0], rep[1], pre[1], fre[1], *bias,
                         m.address if m else 0, mask_stride), handle or None)
    return out


# ---- the largest entries of a row ----------------------------------------------------------

def _count(k, most):
    if isinstance(k, bool) or not isinstance(k, (int, np.integer)):
        raise TypeError("k must be an integer, got %s" % type(k).__name__)
    if not 1 <= k <= most:
        raise ValueError("k must be between 1 and %d, got %d" % (most, k))
    return int(k)


def _row_code(dtype):
    dtype = _foreign_dtypes.get(dtype) or (np.dtype(dtype) if not str(dtype).startswith("torch.")
                                           else _foreign_dtype(dtype))
    if dtype not in _ROW_DTYPE:
        raise TypeError("unsupported dtype %s" % dtype)
    return _ROW_DTYPE[dtype]


def top_workspace(rows, vocab, k, dtype):
    """Bytes of workspace `top` needs for `rows` rows of `vocab` entries of `dtype` (0: none)."""
    _driver.driver.ensure_initialized()
    return _driver.driver.lib.nbh_rows_top_workspace(rows, vocab, k, _row_code(dtype))


def top(logits, k, *, values=None, indices=None, lse=None, temperature=1.0, workspace=None, stream=0):
    """The `k` largest entries of every row, largest first: (values, indices), and with `lse` the
    rows' log sum exp(logits / temperature) as a third result.

    k       : 1 to 1024, at most the row's length
    values  : rows x k of the logits' type, indices: rows x k int32, lse: float32 of one number per row;
              allocated unless given (lse=True allocates it)
    NaN counts as larger than everything, -0 and +0 as equal; equal entries come in the order of their
    indices.
    """
    devices.get_context()
    handle = _driver._stream_handle(stream)
    x = _input(logits, "logits", stream)
    stride = _as_rows(x, "logits")
    rows, vocab = x.shape
    k = _count(k, min(vocab, MOST))
    temperature = _temperature(temperature)
    shape = (rows, k)
    values, v = _result(values, "values", shape, x.dtype, stream, handle)
    values_stride = _as_result_rows(v, "values", shape, (x.dtype,))
    _refuse_overlap(v, "values", x, "logits")
    indices, i = _result(indices, "indices", shape, _int32, stream, handle)
    indices_stride = _as_result_rows(i, "indices", shape, (_int32,))
    _refuse_overlap(i, "indices", x, "logits")
    z = None
    if lse is not None and lse is not False:
        lse, z = _result(lse, "lse", (rows,), _float32, stream, handle)
        _as_vector(z, "lse", rows, _FLOATS)
        _refuse_overlap(z, "lse", x, "logits")
    code = _ROW_DTYPE[x.dtype]
    if rows:
        space = _workspace(workspace, _driver.driver.lib.nbh_rows_top_workspace(rows, vocab, k, code), handle)
        _driver.driver.nbh_rows_top(x.address, rows, vocab, stride, code, k, v.address, values_stride, i.address,
                                    indices_stride, z.address if z else None, temperature, space[0] or None,
                                    space[1], handle or None)
    return (values, indices) if z is None else (values, indices, lse)


# ---- distillation --------------------------------------------------------------------------

def distill_workspace(rows, vocab, k, dtype, *, loss=True, grad=False):
    """Bytes of workspace the distillation functions need (0: none); `dtype` is the student's."""
    _driver.driver.ensure_initialized()
    return _driver.driver.lib.nbh_rows_distill_workspace(rows, vocab, k, _row_code(dtype),
                                                         (_LOSS if loss else 0) | (_GRAD if grad else 0))


def _distill(what, grad_loss, student, values, indices, temperature, teacher_lse, loss, lse, out, workspace, stream):
    devices.get_context()
    handle = _driver._stream_handle(stream)
    x = _input(student, "student", stream)
    stride = _as_rows(x, "student")
    rows, vocab = x.shape
    v = _input(values, "values", stream)
    values_stride = _as_rows(v, "values")
    i = _input(indices, "indices", stream)
    indices_stride = _as_rows(i, "indices", v.shape, _INTEGERS)
    if v.shape[0] != rows:
        raise ValueError("values has %d rows, student has %d" % (v.shape[0], rows))
    k = v.shape[1]
    if k > MOST:
        raise ValueError("a row of values may hold %d entries, got %d" % (MOST, k))
    temperature = _temperature(temperature)
    t = g = None
    if teacher_lse is not None:
        t = _as_vector(_input(teacher_lse, "teacher_lse", stream, np.float32), "teacher_lse", rows, _FLOATS)
    g_stride, g_value = 0, 0.0
    if what & _GRAD:
        if _is_number(grad_loss):
            g_value = _number(grad_loss, "grad_loss")
        else:
            g = _input(grad_loss, "grad_loss", stream, np.float32)
            if g.shape != (rows,):
                raise ValueError("grad_loss has shape %s, expected (%d,)" % (g.shape, rows))
            if g.dtype != _float32:
                raise TypeError("grad_loss has unsupported dtype %s" % g.dtype)
            g_stride = g.strides[0]
            if g.address % 4 or g_stride % 4:
                raise ValueError("grad_loss is not aligned to its item size")

    small = [(v, "values"), (i, "indices")] + ([(t, "teacher_lse")] if t else []) + ([(g, "grad_loss")] if g else [])
    l = z = y = None
    if what & _LOSS:
        loss, l = _result(loss, "loss", (rows,), _float32, stream, handle)
        _as_vector(l, "loss", rows, _FLOATS)
        lse, z = _result(lse, "lse", (rows,), _float32, stream, handle)
        _as_vector(z, "lse", rows, _FLOATS)
        for other in small + [(x, "student"), (z, "lse")]:
            _refuse_overlap(l, "loss", *other)
        for other in small + [(x, "student")]:
            _refuse_overlap(z, "lse", *other)
    else:
        z = _as_vector(_input(lse, "lse", stream, np.float32), "lse", rows, _FLOATS)
        small.append((z, "lse"))
    out_stride = 0
    if what & _GRAD:
        out, y = _result(out, "out", x.shape, x.dtype, stream, handle)
        out_stride = _as_result_rows(y, "out", x.shape, (x.dtype,))
        _refuse_overlap(y, "out", x, "student", same=True)
        for other in small + ([(l, "loss"), (z, "lse")] if what & _LOSS else []):
            _refuse_overlap(y, "out", *other)

    if rows:
        code = _ROW_DTYPE[x.dtype]
        space = _workspace(workspace, _driver.driver.lib.nbh_rows_distill_workspace(rows, vocab, k, code, what), handle)
        _driver.driver.nbh_rows_distill(
            _DISTILL.pack(_DISTILL.size, what, x.address, rows, vocab, stride, code, v.address, i.address, k,
                          values_stride, _ROW_DTYPE[v.dtype], indices_stride, i.dtype.itemsize,
                          t.address if t else 0, g.address if g else 0, g_stride, g_value, temperature,
                          l.address if l else 0, z.address, y.address if y else 0, out_stride, space[0], space[1]),
            handle or None)
    return loss, lse, out


def distill_loss(student, values, indices, *, temperature=1.0, teacher_lse=None, loss=None, lse=None, workspace=None,
                 stream=0):
    """Divergence of the student's distribution from a teacher's, given by the teacher's largest
    logits, for every row: (loss, lse), float32 of one number per row.

        lse = log sum exp(student / T);  log q(v) = student[v] / T - lse
        loss = sum over the teacher's entries of p (log p - log q(index))

    student : rows x vocabulary
    values  : rows x k (k up to 1024) of the teacher's logits, indices: the entries they belong to (int32
              or int64).  An entry with an index outside the vocabulary (-1, say) or the value -inf is
              absent; a row without entries has loss 0.  An index may occur more than once.
    teacher_lse : the teacher's own log sum exp(logits / T) (as `top` returns it): p = exp(values / T -
              teacher_lse).  Without it p is the softmax of values / T over the entries present.
    """
    loss, lse, _ = _distill(_LOSS, None, student, values, indices, temperature, teacher_lse, loss, lse, None,
                            workspace, stream)
    return loss, lse


def distill_grad(grad_loss, student, values, indices, lse, *, temperature=1.0, teacher_lse=None, out=None, stream=0):
    """The gradient of sum(grad_loss * loss) with respect to `student`, from the `lse` that
    distill_loss returned:

        out[v] = grad_loss / T * (q(v) sum of p - sum of p over the entries of index v)

    grad_loss : a number or a float32 array of one number per row (any stride, 0 too)
    out       : of the student's shape and type; may be `student` itself
    A row without entries, or with grad_loss 0, has gradient 0.  Other arguments as for distill_loss.
    """
    return _distill(_GRAD, grad_loss, student, values, indices, temperature, teacher_lse, None, lse, out, None,
                    stream)[2]


def distill_loss_and_grad(grad_loss, student, values, indices, *, temperature=1.0, teacher_lse=None, loss=None,
                          lse=None, out=None, workspace=None, stream=0):
    """distill_loss and distill_grad in one pass over the student's logits: (loss, lse, out).
    `loss` is not multiplied by grad_loss."""
    return _distill(_LOSS | _GRAD, grad_loss, student, values, indices, temperature, teacher_lse, loss, lse, out,
                    workspace, stream)

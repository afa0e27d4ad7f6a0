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

Everything is asynchronous on `stream`.  Results are the same from call to call.  Sums are formed in an
order that goes by the number of rows, their length and alignment, so the last bits of lse, loss and
gradients of a row depend on the array it is in; `adjust` and the entries of `top` do not.  A call
that needs a workspace keeps one per stream; a call recorded into a graph takes the caller's
(`workspace=`, at least `top_workspace` / `distill_workspace` bytes) and the caller's result arrays,
since a graph may run beside later calls on its stream, and inputs in device memory only.
"""

import ctypes
import math
import struct

import numpy as np

from numba_cuda_amd._logits_host import beside as _beside, refuse_overlaps as _refuse_overlaps
from numba_cuda_amd._logits_host import bfloat16, from_bfloat16, host_array, to_bfloat16  # noqa: F401
from numba_cuda_amd.cudadrv import devicearray, devices
from numba_cuda_amd.cudadrv import driver as _driver

MOST = 1024                                  # NBH_ROW_TOP_MOST: entries `top` returns and the distillation takes

_F32, _F16, _BF16 = 0, 1, 2                  # enum nbh_row_dtype
_LOSS, _GRAD = 1, 2                          # enum nbh_distill_what
_float32, _float16 = np.dtype(np.float32), np.dtype(np.float16)
_int32, _int64, _uint32 = np.dtype(np.int32), np.dtype(np.int64), np.dtype(np.uint32)

_ADJUST = struct.Struct("@qPP6q3P4q3P3d3P3qPq")       # struct nbh_logits_adjust_args
_DISTILL = struct.Struct("@qqP4q2P5q2Pqdd3PqPq")      # struct nbh_rows_distill_args


# ---- arguments ---------------------------------------------------------------------------
#
# A call of a few microseconds on the device should not take many on the host.  An argument becomes a
# row view (address, rows, columns, bytes from row to row, code) or a vector view (address, items, item
# size), for ordinary ones in one native call (row_view / vector_view of _hostbuf, which go by these
# tables); whatever that declines takes the path through _device_view, which also raises what there is
# to raise.  Class -> are its strides counted in items; dtype object -> (item size, code).  The classes
# and dtype objects of torch are added when the first of them is seen.
_ROWS = {devicearray.DeviceNDArray: False, _float32: (4, _F32), _float16: (2, _F16), bfloat16: (2, _BF16)}
_INTEGER_ROWS = {devicearray.DeviceNDArray: False, _int32: (4, 4), _int64: (8, 8)}
_INT32_ROWS = {devicearray.DeviceNDArray: False, _int32: (4, 4)}
_WORDS = {devicearray.DeviceNDArray: False, _int32: (4, 0), _uint32: (4, 0)}
_INTEGERS = {devicearray.DeviceNDArray: False, _int32: (4, 4), _int64: (8, 8)}
_FLOATS = {devicearray.DeviceNDArray: False, _float32: (4, 0)}
_TABLES = (_ROWS, _INTEGER_ROWS, _INT32_ROWS, _WORDS, _INTEGERS, _FLOATS)

_row_view = getattr(_driver._hostbuf, "row_view", lambda *_: None)         # None from an older build: slower
_vector_view = getattr(_driver._hostbuf, "vector_view", lambda *_: None)

_foreign_dtypes = {}                         # dtype objects of other libraries -> np.dtype


def _foreign_dtype(dtype):
    name = str(dtype).rpartition(".")[2]
    try:
        found = bfloat16 if name == "bfloat16" else np.dtype(name)
    except TypeError:
        raise TypeError("unsupported dtype: %s" % (dtype,)) from None
    _foreign_dtypes[dtype] = found
    for table in _TABLES:
        if found in table:
            table[dtype] = table[found]
    return found


def _is_tensor(obj):
    if not (hasattr(obj, "is_cuda") and hasattr(obj, "data_ptr") and hasattr(obj, "stride")):
        return False
    if type(obj).__name__ == "Tensor":       # not its subclasses
        for table in _TABLES:
            table[type(obj)] = True
    return True


def _device_view(obj):
    """(address, shape, byte strides, dtype, what keeps it alive) of something in device memory, None
    for anything else."""
    if getattr(obj, "__cuda_ndarray__", False):
        return obj.device_ctypes_pointer.value or 0, tuple(obj.shape), tuple(obj.strides), obj.dtype, obj
    if _is_tensor(obj):
        if not obj.is_cuda:
            return None
        if getattr(obj, "is_neg", bool)():
            raise TypeError("the tensor is a negated view of its memory: torch.resolve_neg makes an ordinary one")
        dtype = _foreign_dtypes.get(obj.dtype) or _foreign_dtype(obj.dtype)
        return obj.data_ptr(), tuple(obj.shape), tuple([n * dtype.itemsize for n in obj.stride()]), dtype, obj
    if hasattr(obj, "__cuda_array_interface__"):
        return _device_view(devicearray.auto_device(obj)[0])
    return None


_several_devices = None


def _one_device():
    global _several_devices
    if _several_devices is None:
        _several_devices = _driver.driver.get_device_count() > 1
    return not _several_devices


def _checked_view(obj, name, stream, dtype=None, output=False):
    """_device_view of an argument; an input on the host is copied over."""
    view = _device_view(obj)
    if view is None:
        if output:
            raise TypeError("%s must be a device array" % name)
        if _capturing(_driver._stream_handle(stream)):       # each replay would copy from a host array that is gone
            raise ValueError("a call that is captured into a graph needs %s in device memory" % name)
        view = _device_view(devicearray.auto_device(host_array(obj, dtype), stream=stream)[0])
    if not _one_device() and view[0]:        # memory of another device than the calling thread's
        where, here = ctypes.c_int(), ctypes.c_int()
        _driver.driver.nbh_get_device(ctypes.byref(here))
        _driver.driver.nbh_pointer_device(view[0], ctypes.byref(where))
        if where.value != here.value:
            raise ValueError("%s is on device %d, the current device is %d" % (name, where.value, here.value))
    return view


def _rows_of(obj, name, stream, table=_ROWS, output=False, keep=None):
    """The row view of a 2-d argument; what a copy from the host needs alive goes into `keep`."""
    if _several_devices is False:
        view = _row_view(obj, table)
        if view is not None:
            return view
    address, shape, strides, dtype, owner = _checked_view(obj, name, stream, output=output)
    if len(shape) != 2:
        raise ValueError("%s must be a 2-d array, got %d-d" % (name, len(shape)))
    if dtype not in table:
        raise TypeError("%s has unsupported dtype %s" % (name, dtype))
    size, code = table[dtype]
    rows, columns = shape
    if columns > 1 and strides[1] != size:
        raise ValueError("the items of a row of %s must lie next to each other (strides %s)" % (name, strides))
    if address % size or (rows > 1 and strides[0] % size):
        raise ValueError("%s is not aligned to its item size" % name)
    if keep is not None:
        keep.append(owner)
    return address, rows, columns, strides[0] if rows > 1 else 0, code


def _vector_of(obj, name, length, stream, table, dtype=None, output=False, keep=None):
    """The vector view of a 1-d argument of `length` items (None: any number)."""
    if _several_devices is False:
        view = _vector_view(obj, table, -1 if length is None else length)
        if view is not None:
            return view
    address, shape, strides, dtype, owner = _checked_view(obj, name, stream, dtype, output)
    if len(shape) != 1:
        raise ValueError("%s must be a 1-d array, got %d-d" % (name, len(shape)))
    if dtype not in table:
        raise TypeError("%s has unsupported dtype %s" % (name, dtype))
    size, n = dtype.itemsize, shape[0]
    if length is not None and n != length:
        raise ValueError("%s has %d items, expected %d" % (name, n, length))
    if n > 1 and strides[0] != size:
        raise ValueError("%s must have unit stride" % name)
    if address % size:
        raise ValueError("%s is not aligned to its item size" % name)
    if keep is not None:
        keep.append(owner)
    return address, n, size


_SIZE = (4, 2, 2)                            # item size by row code


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


def _result_rows(obj, name, rows, columns, dtype, stream, handle, table=_ROWS):
    """(what the caller gets back, its row view) for a rows x columns result that may have been given."""
    if obj is None:
        obj = _new((rows, columns), dtype, stream, handle, name)
    view = _rows_of(obj, name, stream, table, output=True)
    if view[1] != rows or view[2] != columns:
        raise ValueError("%s has shape %s, expected %s" % (name, view[1:3], (rows, columns)))
    if rows > 1 and columns and abs(view[3]) < columns * (_SIZE[view[4]] if table is _ROWS else view[4]):
        raise ValueError("the rows of %s overlap (%d bytes from one to the next)" % (name, view[3]))
    return obj, view


def _result_numbers(obj, name, rows, stream, handle):
    if obj is None or obj is True:
        obj = _new((rows,), _float32, stream, handle, name)
    return obj, _vector_of(obj, name, rows, stream, _FLOATS, output=True)[0]


def _workspace(given, nbytes, handle, others):
    """(address, bytes, what keeps it alive)."""
    if given is not None:
        address, shape, strides, dtype, owner = _checked_view(given, "workspace", 0, output=True)
        expect = dtype.itemsize
        for n, step in zip(shape[::-1], strides[::-1]):
            if n > 1 and step != expect:
                raise ValueError("workspace must be contiguous")
            expect *= n
        if expect < nbytes or address % 16:
            raise ValueError("workspace must hold %d bytes, aligned to 16" % nbytes)
        if nbytes:
            _refuse_overlaps([(address, 1, nbytes, 0, "workspace")], others)
        return address, expect, owner
    if not nbytes:
        return _NO_WORKSPACE
    if _capturing(handle):
        raise ValueError("a call that is captured into a graph needs a workspace of %d bytes" % nbytes)
    return devices.get_context().workspace(handle, nbytes)


_NO_WORKSPACE = (0, 0, None)


def _launch(space, entry, *args):
    """A call that may be several launches.  Those of two threads that share a stream's workspace must not
    come between each other: the second would write what the first has still to read."""
    if space is _NO_WORKSPACE:
        entry(*args)
    else:
        with devices.get_context().workspace_lock:
            entry(*args)


# ---- penalties, biases, masks --------------------------------------------------------------

def _per_row(value, name, rows, stream, number, keep):
    """(address, value in its place) of a number or one number per row."""
    if value is None:
        return 0, number
    if _is_number(value):
        value = _number(value, name)
        if name == "repetition" and value <= 0:
            raise ValueError("repetition must be positive, got %r" % value)
        return 0, value
    return _vector_of(value, name, rows, stream, _FLOATS, np.float32, keep=keep)[0], number


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
    keep = []                                # copies of host arrays, alive until the launch is made
    address, rows, vocab, in_stride, code = _rows_of(logits, "logits", stream, keep=keep)
    if (tokens is None) != (offsets is None):
        raise ValueError("tokens and offsets come together")
    if tokens is None and not (prompt_lengths is repetition is presence is frequency is None):
        raise ValueError("penalties and prompt lengths need tokens and offsets")
    if (bias_tokens is None) != (bias_values is None) or (bias_tokens is None) != (bias_offsets is None):
        raise ValueError("bias_tokens, bias_values and bias_offsets come together")

    out, y = _result_rows(out, "out", rows, vocab, _DTYPE[code], stream, handle)
    if y[4] != code and y[4] != _F32:
        raise TypeError("out has dtype %s, expected %s or float32" % (_DTYPE[y[4]], _DTYPE[code]))
    x = (address, rows, vocab * _SIZE[code], in_stride, "logits")
    _refuse_overlaps([(y[0], rows, vocab * _SIZE[y[4]], y[3], "out")], [x], same=x)

    low = high = 0                           # the bytes `out` lies in: no other array may touch them
    if rows and vocab:
        low, high = y[0] + min(0, (rows - 1) * y[3]), y[0] + max(0, (rows - 1) * y[3]) + vocab * _SIZE[y[4]]
    history, bias = _NO_HISTORY, _NO_BIAS
    if tokens is not None:
        t = _vector_of(tokens, "tokens", None, stream, _INTEGERS, keep=keep)
        o = _vector_of(offsets, "offsets", rows + 1, stream, _INTEGERS, keep=keep)
        p = _NO_PROMPTS
        if prompt_lengths is not None:
            p = _vector_of(prompt_lengths, "prompt_lengths", rows, stream, _INTEGERS, keep=keep)
        rep = _per_row(repetition, "repetition", rows, stream, 1.0, keep)
        pre = _per_row(presence, "presence", rows, stream, 0.0, keep)
        fre = _per_row(frequency, "frequency", rows, stream, 0.0, keep)
        history = (t[0], o[0], p[0], t[1], t[2], o[2], p[2], rep[0], pre[0], fre[0], rep[1], pre[1], fre[1])
        if (t[0] < high and low < t[0] + t[1] * t[2]) or (o[0] < high and low < o[0] + (rows + 1) * o[2]) or (
                p[0] < high and low < p[0] + rows * p[2]) or (rep[0] < high and low < rep[0] + rows * 4) or (
                pre[0] < high and low < pre[0] + rows * 4) or (fre[0] < high and low < fre[0] + rows * 4):
            raise ValueError("out overlaps the history or the penalties")
    if bias_tokens is not None:
        t = _vector_of(bias_tokens, "bias_tokens", None, stream, _INTEGERS, keep=keep)
        v = _vector_of(bias_values, "bias_values", t[1], stream, _FLOATS, np.float32, keep=keep)
        o = _vector_of(bias_offsets, "bias_offsets", rows + 1, stream, _INTEGERS, keep=keep)
        bias = (t[0], o[0], v[0], t[1], t[2], o[2])
        if (t[0] < high and low < t[0] + t[1] * t[2]) or (v[0] < high and low < v[0] + t[1] * 4) or (
                o[0] < high and low < o[0] + (rows + 1) * o[2]):
            raise ValueError("out overlaps the biases")
    mask_address = mask_stride = 0
    if mask is not None:
        mask_address, mask_stride = _mask_of(mask, rows, vocab, stream, keep)
        words = (vocab + 31) // 32 * 4
        if rows and vocab and mask_address + min(0, mask_stride * (rows - 1)) < high and (
                low < mask_address + max(0, mask_stride * (rows - 1)) + words) and not _beside(
                (y[0], rows, vocab * _SIZE[y[4]], y[3]), (mask_address, rows, words, mask_stride)):
            raise ValueError("out overlaps mask")

    if rows and vocab:
        _driver.driver.nbh_logits_adjust(
            _ADJUST.pack(_ADJUST_SIZE, address, y[0], rows, vocab, in_stride, y[3], code, y[4], *history, *bias,
                         mask_address, mask_stride), handle or None)
    return out


def _mask_of(mask, rows, vocab, stream, keep):
    """(address, bytes from row to row) of the words of a mask."""
    view = _row_view(mask, _WORDS) if _several_devices is False else None
    if view is not None:
        address, masks, words, stride, _ = view
    else:
        address, shape, strides, dtype, owner = _checked_view(mask, "mask", stream)
        keep.append(owner)
        if dtype not in _WORDS:
            raise TypeError("mask has dtype %s, expected 32-bit integers" % dtype)
        if len(shape) not in (1, 2):
            raise ValueError("mask has shape %s, expected one row of words or %d" % (shape, rows))
        words, masks = shape[-1], shape[0] if len(shape) == 2 else 1
        if words > 1 and strides[-1] != 4:
            raise ValueError("the words of a mask must lie next to each other (strides %s)" % (strides,))
        stride = strides[0] if masks > 1 else 0
    if masks != rows and masks != 1:
        raise ValueError("mask has shape %s, expected one row of words or %d" % ((masks, words), rows))
    if words * 32 < vocab:
        raise ValueError("mask has %d words, %d entries need %d" % (words, vocab, -(-vocab // 32)))
    return address, stride if masks > 1 else 0


_DTYPE = (_float32, _float16, bfloat16)      # by code
_ADJUST_SIZE = _ADJUST.size
_NO_PROMPTS = (0, 0, 4)
_NO_HISTORY = (0, 0, 0, 0, 4, 4, 4, 0, 0, 0, 1.0, 0.0, 0.0)
_NO_BIAS = (0, 0, 0, 0, 4, 4)


# ---- the largest entries of a row ----------------------------------------------------------

def _count(k, most):
    if isinstance(k, bool) or not isinstance(k, (int, np.integer)):
        raise TypeError("k must be an integer, got %s" % type(k).__name__)
    if not 1 <= k <= most:
        raise ValueError("k must be between 1 and %d, got %d" % (most, k))
    return int(k)


def _row_code(dtype):
    if str(dtype).startswith("torch."):
        dtype = _foreign_dtype(dtype)
    dtype = np.dtype(dtype)
    if dtype not in _DTYPE:
        raise TypeError("unsupported dtype %s" % dtype)
    return _DTYPE.index(dtype)


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
    keep = []
    address, rows, vocab, stride, code = _rows_of(logits, "logits", stream, keep=keep)
    k = _count(k, min(vocab, MOST))
    temperature = _temperature(temperature)
    values, v = _result_rows(values, "values", rows, k, _DTYPE[code], stream, handle)
    if v[4] != code:
        raise TypeError("values has dtype %s, expected %s" % (_DTYPE[v[4]], _DTYPE[code]))
    indices, i = _result_rows(indices, "indices", rows, k, _int32, stream, handle, _INT32_ROWS)
    results = [(v[0], rows, k * _SIZE[code], v[3], "values"), (i[0], rows, k * 4, i[3], "indices")]
    lse_address, wanted = None, lse is not None and lse is not False
    if wanted:
        lse, lse_address = _result_numbers(lse, "lse", rows, stream, handle)
        results.append((lse_address, 1, rows * 4, 0, "lse"))
    inputs = [(address, rows, vocab * _SIZE[code], stride, "logits")]
    _refuse_overlaps(results, inputs)
    if rows:
        space = _workspace(workspace, _driver.driver.lib.nbh_rows_top_workspace(rows, vocab, k, code), handle,
                           results + inputs)
        _launch(space, _driver.driver.nbh_rows_top, address, rows, vocab, stride, code, k, v[0], v[3], i[0], i[3],
                lse_address, temperature, space[0] or None, space[1], handle or None)
    return (values, indices, lse) if wanted else (values, indices)


# ---- distillation --------------------------------------------------------------------------

def distill_workspace(rows, vocab, k, dtype, *, loss=True, grad=False):
    """Bytes of workspace the distillation functions need (0: none); `dtype` is the student's."""
    _driver.driver.ensure_initialized()
    return _driver.driver.lib.nbh_rows_distill_workspace(rows, vocab, k, _row_code(dtype),
                                                         (_LOSS if loss else 0) | (_GRAD if grad else 0))


def _distill(what, grad_loss, student, values, indices, temperature, teacher_lse, loss, lse, out, workspace, stream):
    devices.get_context()
    handle = _driver._stream_handle(stream)
    keep = []
    address, rows, vocab, stride, code = _rows_of(student, "student", stream, keep=keep)
    v = _rows_of(values, "values", stream, keep=keep)
    i = _rows_of(indices, "indices", stream, _INTEGER_ROWS, keep=keep)
    k = v[2]
    if i[1] != v[1] or i[2] != k:
        raise ValueError("indices has shape %s, expected %s" % (i[1:3], v[1:3]))
    if v[1] != rows:
        raise ValueError("values has %d rows, student has %d" % (v[1], rows))
    if k > MOST:
        raise ValueError("a row of values may hold %d entries, got %d" % (MOST, k))
    temperature = _temperature(temperature)
    x = (address, rows, vocab * _SIZE[code], stride, "student")
    inputs = [x, (v[0], rows, k * _SIZE[v[4]], v[3], "values"), (i[0], rows, k * i[4], i[3], "indices")]
    results = []
    teacher_address = grad_address = grad_stride = loss_address = out_address = out_stride = 0
    grad_value = 0.0
    if teacher_lse is not None:
        teacher_address = _vector_of(teacher_lse, "teacher_lse", rows, stream, _FLOATS, np.float32, keep=keep)[0]
        inputs.append((teacher_address, 1, rows * 4, 0, "teacher_lse"))
    if what & _GRAD:
        if _is_number(grad_loss):
            grad_value = _number(grad_loss, "grad_loss")
        else:
            grad_address, grad_stride = _grad_loss_of(grad_loss, rows, stream, keep)
            inputs.append((grad_address, rows, 4, grad_stride, "grad_loss"))
    if what & _LOSS:
        loss, loss_address = _result_numbers(loss, "loss", rows, stream, handle)
        lse, lse_address = _result_numbers(lse, "lse", rows, stream, handle)
        results += [(loss_address, 1, rows * 4, 0, "loss"), (lse_address, 1, rows * 4, 0, "lse")]
    else:
        lse_address = _vector_of(lse, "lse", rows, stream, _FLOATS, np.float32, keep=keep)[0]
        inputs.append((lse_address, 1, rows * 4, 0, "lse"))
    if what & _GRAD:
        out, y = _result_rows(out, "out", rows, vocab, _DTYPE[code], stream, handle)
        if y[4] != code:
            raise TypeError("out has dtype %s, expected %s" % (_DTYPE[y[4]], _DTYPE[code]))
        out_address, out_stride = y[0], y[3]
        results.append((out_address, rows, vocab * _SIZE[code], out_stride, "out"))
    _refuse_overlaps(results, inputs, same=x)

    if rows:
        space = _workspace(workspace, _driver.driver.lib.nbh_rows_distill_workspace(rows, vocab, k, code, what), handle,
                           results + inputs)
        arguments = _DISTILL.pack(_DISTILL_SIZE, what, address, rows, vocab, stride, code, v[0], i[0], k, v[3], v[4], i[3],
                                  i[4], teacher_address, grad_address, grad_stride, grad_value, temperature,
                                  loss_address, lse_address, out_address, out_stride, space[0], space[1])
        _launch(space, _driver.driver.nbh_rows_distill, arguments, handle or None)
    return loss, lse, out


def _grad_loss_of(grad_loss, rows, stream, keep):
    """(address, stride): of any stride, 0 too."""
    if _several_devices is False:
        view = _vector_view(grad_loss, _FLOATS, rows)
        if view is not None:
            return view[0], 4
    address, shape, strides, dtype, owner = _checked_view(grad_loss, "grad_loss", stream, np.float32)
    keep.append(owner)
    if shape != (rows,):
        raise ValueError("grad_loss has shape %s, expected (%d,)" % (shape, rows))
    if dtype not in _FLOATS:
        raise TypeError("grad_loss has unsupported dtype %s" % dtype)
    if address % 4 or strides[0] % 4:
        raise ValueError("grad_loss is not aligned to its item size")
    return address, strides[0]


_DISTILL_SIZE = _DISTILL.size


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


def distill_grad(grad_loss, student, values, indices, lse, *, temperature=1.0, teacher_lse=None, out=None,
                 workspace=None, stream=0):
    """The gradient of sum(grad_loss * loss) with respect to `student`, from the `lse` that
    distill_loss returned:

        out[v] = grad_loss / T * (q(v) sum of p - sum of p over the entries of index v)

    grad_loss : a number or a float32 array of one number per row (any stride, 0 too)
    out       : of the student's shape and type; may be `student` itself
    A row without entries, or with grad_loss 0, has gradient 0.  Other arguments as for distill_loss.
    """
    return _distill(_GRAD, grad_loss, student, values, indices, temperature, teacher_lse, None, lse, out, workspace,
                    stream)[2]


def distill_loss_and_grad(grad_loss, student, values, indices, *, temperature=1.0, teacher_lse=None, loss=None,
                          lse=None, out=None, workspace=None, stream=0):
    """distill_loss and distill_grad in one pass over the student's logits: (loss, lse, out).
    `loss` is not multiplied by grad_loss."""
    return _distill(_LOSS | _GRAD, grad_loss, student, values, indices, temperature, teacher_lse, loss, lse, out,
                    workspace, stream)

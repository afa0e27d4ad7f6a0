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

# A call of a few microseconds on the device should not take many on the host: arguments become plain
# tuples (address, shape, byte strides, dtype, what keeps the memory alive), found by the class of the
# argument; a torch tensor's attributes cost a tenth of what its interface dictionary does.

_foreign_dtypes = {}                         # dtype objects of other libraries -> (np.dtype, its item size)


def _foreign_dtype(dtype):
    name = str(dtype).rpartition(".")[2]
    try:
        found = bfloat16 if name == "bfloat16" else np.dtype(name)
    except TypeError:
        raise TypeError("unsupported dtype: %s" % (dtype,)) from None
    _foreign_dtypes[dtype] = found, found.itemsize
    return _foreign_dtypes[dtype]


def _view_of_own(array):
    try:
        address = array.gpu_data.device_pointer
    except AttributeError:
        address = array.device_ctypes_pointer.value or 0
    return address, array.shape, array.strides, array.dtype, array


def _view_of_tensor(tensor):
    if not tensor.is_cuda:
        return None
    dtype = tensor.dtype
    dtype, size = _foreign_dtypes.get(dtype) or _foreign_dtype(dtype)
    strides = tensor.stride()
    if len(strides) == 1:
        strides = (strides[0] * size,)
    elif len(strides) == 2:
        strides = (strides[0] * size, strides[1] * size)
    else:
        strides = tuple([n * size for n in strides])
    return tensor.data_ptr(), tensor.shape, strides, dtype, tensor


_views = {devicearray.DeviceNDArray: _view_of_own}       # class -> function


def _device_view(obj):
    """The tuple of something in device memory, None for anything else."""
    view = _views.get(obj.__class__)
    if view is not None:
        return view(obj)
    if getattr(obj, "__cuda_ndarray__", False):
        return _view_of_own(obj)
    if hasattr(obj, "is_cuda") and hasattr(obj, "data_ptr") and hasattr(obj, "stride"):
        _views[obj.__class__] = _view_of_tensor
        return _view_of_tensor(obj)
    if hasattr(obj, "__cuda_array_interface__"):
        return _view_of_own(devicearray.auto_device(obj)[0])
    return None


_several_devices = None


def _check_device(view, name):
    """Refuse memory of another device than the calling thread's."""
    global _several_devices
    if _several_devices is None:
        _several_devices = _driver.driver.get_device_count() > 1
    if _several_devices and view[0]:
        where, here = ctypes.c_int(), ctypes.c_int()
        _driver.driver.nbh_get_device(ctypes.byref(here))
        _driver.driver.nbh_pointer_device(view[0], ctypes.byref(where))
        if where.value != here.value:
            raise ValueError("%s is on device %d, the current device is %d" % (name, where.value, here.value))


def _input(obj, name, stream, dtype=None):
    """The tuple of an input; what is on the host is copied over."""
    view = _device_view(obj)
    if view is None:
        host = np.asarray(obj) if dtype is None else np.asarray(obj, dtype=dtype)
        if not host.flags["C_CONTIGUOUS"]:
            host = np.ascontiguousarray(host)
        view = _device_view(devicearray.auto_device(host, stream=stream)[0])
    if _several_devices is not False:
        _check_device(view, name)
    return view


def _output(obj, name):
    view = _device_view(obj)
    if view is None:
        raise TypeError("%s must be a device array" % name)
    if _several_devices is not False:
        _check_device(view, name)
    return view


def _as_rows(view, name, shape=None, dtypes=_ROW_DTYPE):
    """Check a 2-d operand; returns the bytes from row to row."""
    address, own_shape, strides, dtype, _ = view
    if len(own_shape) != 2:
        raise ValueError("%s must be a 2-d array, got %d-d" % (name, len(own_shape)))
    if dtype not in dtypes:
        raise TypeError("%s has unsupported dtype %s" % (name, dtype))
    if shape is not None and own_shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, tuple(own_shape), tuple(shape)))
    size = dtype.itemsize
    rows, columns = own_shape
    if columns > 1 and strides[1] != size:
        raise ValueError("the items of a row of %s must lie next to each other (strides %s)" % (name, strides))
    if address % size or (rows > 1 and strides[0] % size):
        raise ValueError("%s is not aligned to its item size" % name)
    return strides[0] if rows > 1 else 0


def _as_result_rows(view, name, shape, dtypes=_ROW_DTYPE):
    stride = _as_rows(view, name, shape, dtypes)
    if shape[0] > 1 and shape[1] and abs(stride) < shape[1] * view[3].itemsize:
        raise ValueError("the rows of %s overlap (strides %s)" % (name, view[2]))
    return stride


def _as_vector(view, name, length, dtypes):
    address, shape, strides, dtype, _ = view
    if len(shape) != 1:
        raise ValueError("%s must be a 1-d array, got %d-d" % (name, len(shape)))
    if dtype not in dtypes:
        raise TypeError("%s has unsupported dtype %s" % (name, dtype))
    n = shape[0]
    if length is not None and n != length:
        raise ValueError("%s has %d items, expected %d" % (name, n, length))
    size = dtype.itemsize
    if n > 1 and strides[0] != size:
        raise ValueError("%s must have unit stride" % name)
    if address % size:
        raise ValueError("%s is not aligned to its item size" % name)
    return view


_INTEGERS = (_int32, _int64)
_FLOATS = (_float32,)


def _extent(view):
    """First and last + 1 address of the items."""
    low, shape, strides, dtype, _ = view
    high = low
    for n, step in zip(shape, strides):
        if n == 0:
            return low, low
        if step < 0:
            low += (n - 1) * step
        else:
            high += (n - 1) * step
    return low, high + dtype.itemsize


def _refuse_overlaps(results, inputs, same=None):
    """ValueError when a result array touches an input or another result; `same`: the input that a
    result may be, item for item.  Both are lists of (tuple, name)."""
    spans = [(*_extent(view), view, name) for view, name in results]
    others = spans + [(*_extent(view), view, name) for view, name in inputs]
    for at, (low, high, out, name) in enumerate(spans):
        for other_low, other_high, other, other_name in others[at + 1:]:
            if low < other_high and other_low < high and low < high and other_low < other_high and not (
                    other is same and _same_items(out, other)) and not _beside(out, other):
                raise ValueError("%s overlaps %s" % (name, other_name))


def _same_items(out, other):
    return out[0] == other[0] and out[3] == other[3] and (out[1][0] <= 1 or out[2][0] == other[2][0])


def _beside(out, other):
    """Columns of one wider buffer lie between each other without touching."""
    if len(out[1]) == len(other[1]) == 2 and out[2][0] == other[2][0] > 0:
        pitch = out[2][0]
        gap = (other[0] - out[0]) % pitch
        return gap >= out[1][1] * out[3].itemsize and gap + other[1][1] * other[3].itemsize <= pitch
    return False


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
    """(what the caller gets back, its tuple) for a result that may have been given."""
    if obj is None or obj is True:
        obj = _new(shape, dtype, stream, handle, name)
    return obj, _output(obj, name)


def _workspace(given, nbytes, handle):
    """(address, bytes, what keeps it alive)."""
    if given is not None:
        view = _output(given, "workspace")
        low, high = _extent(view)
        items = 1
        for n in view[1]:
            items *= n
        if items * view[3].itemsize != high - low:
            raise ValueError("workspace must be contiguous")
        if high - low < nbytes or low % 16:
            raise ValueError("workspace must hold %d bytes, aligned to 16" % nbytes)
        return low, high - low, view[4]
    if not nbytes:
        return _NO_WORKSPACE
    if _capturing(handle):
        raise ValueError("a call that is captured into a graph needs a workspace of %d bytes" % nbytes)
    return devices.get_context().workspace(handle, nbytes)


_NO_WORKSPACE = (0, 0, None)


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
    view = _as_vector(_input(value, name, stream, np.float32), name, rows, _FLOATS)
    return view[0], number, view[4]


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
    shape, dtype = x[1], x[3]
    rows, vocab = shape
    if (tokens is None) != (offsets is None):
        raise ValueError("tokens and offsets come together")
    if tokens is None and not (prompt_lengths is repetition is presence is frequency is None):
        raise ValueError("penalties and prompt lengths need tokens and offsets")
    if (bias_tokens is None) != (bias_values is None) or (bias_tokens is None) != (bias_offsets is None):
        raise ValueError("bias_tokens, bias_values and bias_offsets come together")

    out, y = _result(out, "out", shape, dtype, stream, handle)
    out_stride = _as_result_rows(y, "out", shape)
    if y[3] != dtype and y[3] != _float32:
        raise TypeError("out has dtype %s, expected %s or float32" % (y[3], dtype))
    _refuse_overlaps([(y, "out")], [(x, "logits")], same=x)

    t = o = p = rep = pre = fre = bt = bo = bv = m = None        # alive until the launch is made
    history, bias = _NO_HISTORY, _NO_BIAS
    if tokens is not None:
        t = _as_vector(_input(tokens, "tokens", stream), "tokens", None, _INTEGERS)
        o = _as_vector(_input(offsets, "offsets", stream), "offsets", rows + 1, _INTEGERS)
        p = _NO_PROMPTS
        if prompt_lengths is not None:
            p = _as_vector(_input(prompt_lengths, "prompt_lengths", stream), "prompt_lengths", rows, _INTEGERS)
        rep = _per_row(repetition, "repetition", rows, stream, 1.0)
        pre = _per_row(presence, "presence", rows, stream, 0.0)
        fre = _per_row(frequency, "frequency", rows, stream, 0.0)
        history = (t[0], o[0], p[0], t[1][0], t[3].itemsize, o[3].itemsize, p[3].itemsize, rep[0], pre[0], fre[0],
                   rep[1], pre[1], fre[1])
    if bias_tokens is not None:
        bt = _as_vector(_input(bias_tokens, "bias_tokens", stream), "bias_tokens", None, _INTEGERS)
        bv = _as_vector(_input(bias_values, "bias_values", stream, np.float32), "bias_values", bt[1][0], _FLOATS)
        bo = _as_vector(_input(bias_offsets, "bias_offsets", stream), "bias_offsets", rows + 1, _INTEGERS)
        bias = (bt[0], bo[0], bv[0], bt[1][0], bt[3].itemsize, bo[3].itemsize)
    mask_address = mask_stride = 0
    if mask is not None:
        m = _input(mask, "mask", stream)
        mask_address, mask_shape, mask_strides, mask_dtype, _ = m
        if mask_dtype.kind not in "iu" or mask_dtype.itemsize != 4:
            raise TypeError("mask has dtype %s, expected 32-bit integers" % mask_dtype)
        if len(mask_shape) not in (1, 2) or (len(mask_shape) == 2 and mask_shape[0] not in (1, rows)):
            raise ValueError("mask has shape %s, expected one row of words or %d" % (tuple(mask_shape), rows))
        words = mask_shape[-1]
        if words * 32 < vocab:
            raise ValueError("mask has %d words, %d entries need %d" % (words, vocab, -(-vocab // 32)))
        if words > 1 and mask_strides[-1] != 4:
            raise ValueError("the words of a mask must lie next to each other (strides %s)" % (mask_strides,))
        if len(mask_shape) == 2 and mask_shape[0] > 1:
            mask_stride = mask_strides[0]

    if rows and vocab:
        _driver.driver.nbh_logits_adjust(
            _ADJUST.pack(_ADJUST_SIZE, x[0], y[0], rows, vocab, in_stride, out_stride, _ROW_DTYPE[dtype],
                         _ROW_DTYPE[y[3]], *history, *bias, mask_address, mask_stride), handle or None)
    return out


_ADJUST_SIZE = _ADJUST.size
_NO_PROMPTS = (0, (0,), (4,), _int32, None)
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
        dtype = _foreign_dtype(dtype)[0]
    dtype = np.dtype(dtype)
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
    (rows, vocab), dtype = x[1], x[3]
    k = _count(k, min(vocab, MOST))
    temperature = _temperature(temperature)
    shape = (rows, k)
    values, v = _result(values, "values", shape, dtype, stream, handle)
    values_stride = _as_result_rows(v, "values", shape, (dtype,))
    indices, i = _result(indices, "indices", shape, _int32, stream, handle)
    indices_stride = _as_result_rows(i, "indices", shape, (_int32,))
    results, lse_address = [(v, "values"), (i, "indices")], None
    wanted = lse is not None and lse is not False
    if wanted:
        lse, z = _result(lse, "lse", (rows,), _float32, stream, handle)
        _as_vector(z, "lse", rows, _FLOATS)
        lse_address = z[0]
        results.append((z, "lse"))
    _refuse_overlaps(results, [(x, "logits")])
    code = _ROW_DTYPE[dtype]
    if rows:
        space = _workspace(workspace, _driver.driver.lib.nbh_rows_top_workspace(rows, vocab, k, code), handle)
        _driver.driver.nbh_rows_top(x[0], rows, vocab, stride, code, k, v[0], values_stride, i[0], indices_stride,
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
    x = _input(student, "student", stream)
    stride = _as_rows(x, "student")
    shape, dtype = x[1], x[3]
    rows, vocab = shape
    v = _input(values, "values", stream)
    values_stride = _as_rows(v, "values")
    i = _input(indices, "indices", stream)
    indices_stride = _as_rows(i, "indices", v[1], _INTEGERS)
    if v[1][0] != rows:
        raise ValueError("values has %d rows, student has %d" % (v[1][0], rows))
    k = v[1][1]
    if k > MOST:
        raise ValueError("a row of values may hold %d entries, got %d" % (MOST, k))
    temperature = _temperature(temperature)
    inputs, results = [(x, "student"), (v, "values"), (i, "indices")], []
    teacher_address = grad_address = grad_stride = loss_address = out_address = out_stride = 0
    grad_value = 0.0
    if teacher_lse is not None:
        t = _as_vector(_input(teacher_lse, "teacher_lse", stream, np.float32), "teacher_lse", rows, _FLOATS)
        teacher_address = t[0]
        inputs.append((t, "teacher_lse"))
    if what & _GRAD:
        if _is_number(grad_loss):
            grad_value = _number(grad_loss, "grad_loss")
        else:
            g = _input(grad_loss, "grad_loss", stream, np.float32)
            grad_address, grad_shape, strides, grad_dtype, _ = g
            if len(grad_shape) != 1 or grad_shape[0] != rows:
                raise ValueError("grad_loss has shape %s, expected (%d,)" % (tuple(grad_shape), rows))
            if grad_dtype != _float32:
                raise TypeError("grad_loss has unsupported dtype %s" % grad_dtype)
            grad_stride = strides[0]
            if grad_address % 4 or grad_stride % 4:
                raise ValueError("grad_loss is not aligned to its item size")
            inputs.append((g, "grad_loss"))
    if what & _LOSS:
        loss, l = _result(loss, "loss", (rows,), _float32, stream, handle)
        loss_address = _as_vector(l, "loss", rows, _FLOATS)[0]
        lse, z = _result(lse, "lse", (rows,), _float32, stream, handle)
        _as_vector(z, "lse", rows, _FLOATS)
        results += [(l, "loss"), (z, "lse")]
    else:
        z = _as_vector(_input(lse, "lse", stream, np.float32), "lse", rows, _FLOATS)
        inputs.append((z, "lse"))
    if what & _GRAD:
        out, y = _result(out, "out", shape, dtype, stream, handle)
        out_address, out_stride = y[0], _as_result_rows(y, "out", shape, (dtype,))
        results.append((y, "out"))
    _refuse_overlaps(results, inputs, same=x)

    if rows:
        code = _ROW_DTYPE[dtype]
        space = _workspace(workspace, _driver.driver.lib.nbh_rows_distill_workspace(rows, vocab, k, code, what), handle)
        _driver.driver.nbh_rows_distill(
            _DISTILL.pack(_DISTILL_SIZE, what, x[0], rows, vocab, stride, code, v[0], i[0], k, values_stride,
                          _ROW_DTYPE[v[3]], indices_stride, i[3].itemsize, teacher_address, grad_address, grad_stride,
                          grad_value, temperature, loss_address, z[0], out_address, out_stride, space[0], space[1]),
            handle or None)
    return loss, lse, out


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

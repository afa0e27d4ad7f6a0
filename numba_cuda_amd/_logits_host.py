"""What the row operators over logits share between the GPU and the CPU mode.

bfloat16 on the host: NumPy has no type for it, so its items are two-byte voids (type string
"<V2", as other libraries export theirs)."""

import numpy as np

bfloat16 = np.dtype("V2")


def to_bfloat16(array):
    """`array` rounded to bfloat16, to nearest even (from float32 values)."""
    bits = np.ascontiguousarray(array, dtype=np.float32).view(np.uint32)
    rounded = (bits + (((bits >> 16) & 1) + np.uint32(0x7fff))) >> 16
    quiet = (bits >> 16) | 0x40                  # a NaN must not round to an infinity
    return np.where((bits & 0x7fffffff) > 0x7f800000, quiet, rounded).astype(np.uint16).view(bfloat16)


def from_bfloat16(array):
    """The float32 values of an array of bfloat16 items."""
    bits = np.ascontiguousarray(array).view(np.uint16).astype(np.uint32) << 16
    return bits.view(np.float32)


def host_array(obj, dtype=None):
    """The compact array of an input on the host.  An empty list holds no integers: NumPy makes float64 of it."""
    a = np.ascontiguousarray(obj, dtype=dtype)
    return a if a.size or dtype is not None or hasattr(obj, "dtype") else a.astype(np.int64)


def refuse_overlaps(results, inputs, same=None):
    """ValueError when a result array touches an input or another result.  Both are lists of blocks
    (address, rows, bytes of a row, bytes from row to row, name); `same`: the input that a result may
    be, byte for byte."""
    spans = []
    for block in results + inputs:
        address, rows, width, step, _ = block
        reach = (rows - 1) * step
        low, high = (address + reach, address + width) if reach < 0 else (address, address + reach + width)
        spans.append((low, high if rows and width else low, block))
    for at, (low, high, out) in enumerate(spans[:len(results)]):
        for other_low, other_high, other in spans[at + 1:]:
            if low < other_high and other_low < high and low < high and other_low < other_high and not (
                    other is same and out[:3] == other[:3] and (out[1] <= 1 or out[3] == other[3])) and not beside(
                    out, other):
                raise ValueError("%s overlaps %s" % (out[4], other[4]))


def beside(out, other):
    """Columns of one wider buffer lie between each other without touching."""
    pitch = out[3]
    if pitch != other[3] or pitch <= 0:
        return False
    gap = (other[0] - out[0]) % pitch
    return gap >= out[2] and gap + other[2] <= pitch

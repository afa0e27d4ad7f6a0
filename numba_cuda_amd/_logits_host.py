"""bfloat16 on the host: NumPy has no type for it, so its items are two-byte voids (type string
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

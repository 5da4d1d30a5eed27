"""Products in 8-bit integers with a scale for each row of both operands: a linear layer's (or the
experts') product on the integer tensor cores.  The reference has no low-precision product.

Neither call has a gradient.  Where gradients are recorded, an operand that requires one is refused: pass it
detached, or call under `torch.no_grad()`.
"""
import ctypes

import torch

from .._cabi import check, lib, stream_ptr
from . import _calls


def quantize_rows(x, rows=None):
    """The rows of `x` in 8 bits: ``q = round(127 * x / max|x|)`` (exact quotient, half to even) and
    ``scales = max|x| / 127``, so that ``q * scales[:, None]`` stands for the row.

    `x` (n, d) in float32, float16 or bfloat16.  With `rows` (m int32), row i is taken from
    ``x[rows[i]]``, or is zero where `rows` lies outside ``[0, n)``: the gather into expert order in the
    same pass.  Returns ``(q (m, d) int8, scales (m,) float32)``; the rows of `q` lie at a pitch of a multiple
    of 16 bytes.  Rows of zeros have scale 0.  A row that holds an infinity or NaN has scale NaN and zeros,
    so that whatever is computed from it is NaN.  Quantise weights the same way, one row per output feature.
    """
    return _calls.quantize_rows(x, rows)


def int8_matmul(a, a_scales, b, b_scales, bias=None, offsets=None, out_dtype=torch.bfloat16):
    """``out[i, j] = a_scales[i] * b_scales[j] * sum_f a[i, f] * b[j, f]  (+ bias[j])``.

    `a` (m, d) and `b` (n, d) int8, scales and `bias` float32; the sum is exact.  With `offsets` (g + 1
    int32, ascending, on the device) `b` is (g, n, d), `b_scales` and `bias` (g, n), and rows
    ``offsets[g]:offsets[g + 1]`` of `a` meet ``b[g]``: the experts' products, with nothing read back to the
    host.  Rows ahead of ``offsets[0]`` and behind ``offsets[-1]`` become zeros.  `out_dtype` is float32, float16 or bfloat16.

    Rows are read in pieces of 16 bytes: operands as `quantize_rows` returns them, or with d a multiple
    of 16, are read in place; others are copied first.  At most 131071 features and 1024 groups.
    """
    return _calls.int8_matmul(a, a_scales, b, b_scales, bias, offsets, out_dtype)


def check_int8_waits(device=None):
    """Raises KmbError if a bounded wait inside `int8_matmul` ran out on `device` since the last call of
    this function (the output tiles concerned hold NaN).  Waits for the device's current stream."""
    flag = ctypes.c_int(0)
    with torch.cuda.device(device):
        check(lib.kmb_int8_wait_error(ctypes.byref(flag), stream_ptr(device)), "kmb_int8_wait_error")

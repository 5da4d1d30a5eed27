"""Products in 8-bit integers with a scale for each row of both operands: a linear layer's (or the
experts') product on the integer tensor cores.  The reference has no low-precision product.
"""
import ctypes

import torch

from .._cabi import check, launch, lib, require_cuda_tensor, row_dtype_code, stream_ptr

#: Features that a sum of products of 8-bit integers may run over before it could leave 32 bits.
MAX_FEATURES = 131071


def _pitched(t, name):
    """`t` with rows at a pitch of a multiple of 16 bytes, as the kernel's loads need them: itself if it
    is laid out so (as `quantize_rows` returns it), else a copy."""
    d = t.shape[-1]
    if t.numel() and t.data_ptr() % 16 == 0 and (d == 1 or t.stride(-1) == 1):
        pitch = t.stride(-2)
        if pitch % 16 == 0 and pitch >= d and (t.dim() == 2 or t.shape[0] == 1
                                               or t.stride(0) == t.shape[1] * pitch):
            return t, pitch
    pitch = -(-d // 16) * 16
    buf = torch.empty((*t.shape[:-1], pitch), dtype=torch.int8, device=t.device)
    buf[..., :d].copy_(t)
    return buf[..., :d], pitch


def quantize_rows(x, rows=None):
    """The rows of `x` in 8 bits: ``q = round(127 * x / max|x|)`` (exact quotient, half to even) and
    ``scales = max|x| / 127``, so that ``q * scales[:, None]`` stands for the row.

    `x` (n, d) in float32, float16 or bfloat16.  With `rows` (m int32), row i is taken from
    ``x[rows[i]]``, or is zero where `rows` lies outside ``[0, n)``: the gather into expert order in the
    same pass.  Returns ``(q (m, d) int8, scales (m,) float32)``; the rows of `q` lie at a pitch of a multiple
    of 16 bytes.  Rows of zeros have scale 0.  A row that holds an infinity or NaN has scale NaN and zeros,
    so that whatever is computed from it is NaN.  Quantise weights the same way, one row per output feature.
    """
    require_cuda_tensor(x, "x", contiguous=False)
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must have shape (n, d) with d >= 1, got {tuple(x.shape)}")
    code = row_dtype_code(x.dtype, "x")
    x = x if x.is_contiguous() else x.contiguous()
    n, d = x.shape
    m = n
    if rows is not None:
        require_cuda_tensor(rows, "rows", torch.int32)
        if rows.dim() != 1 or rows.device != x.device:
            raise ValueError("rows must be a vector on the device of x")
        m = rows.shape[0]
    pitch = -(-d // 16) * 16
    dev = x.device
    q = torch.empty((m, pitch), dtype=torch.int8, device=dev)
    scales = torch.empty(m, dtype=torch.float32, device=dev)
    launch("kmb_quantize_rows", dev, code, x.data_ptr(), n, d, None if rows is None else rows.data_ptr(), m,
           q.data_ptr(), pitch, scales.data_ptr())
    return (q if pitch == d else q[:, :d]), scales


def int8_matmul(a, a_scales, b, b_scales, bias=None, offsets=None, out_dtype=torch.bfloat16):
    """``out[i, j] = a_scales[i] * b_scales[j] * sum_f a[i, f] * b[j, f]  (+ bias[j])``.

    `a` (m, d) and `b` (n, d) int8, scales and `bias` float32; the sum is exact.  With `offsets` (g + 1
    int32, ascending, on the device) `b` is (g, n, d), `b_scales` and `bias` (g, n), and rows
    ``offsets[g]:offsets[g + 1]`` of `a` meet ``b[g]``: the experts' products, with nothing read back to the
    host.  Rows behind ``offsets[-1]`` become zeros.  `out_dtype` is float32, float16 or bfloat16.

    Rows are read in pieces of 16 bytes: operands as `quantize_rows` returns them, or with d a multiple
    of 16, are read in place; others are copied first.  At most 131071 features and 1024 groups.
    """
    require_cuda_tensor(a, "a", torch.int8, contiguous=False)
    require_cuda_tensor(b, "b", torch.int8, contiguous=False)
    code = row_dtype_code(out_dtype, "out_dtype")
    grouped = offsets is not None
    if a.dim() != 2 or b.dim() != (3 if grouped else 2):
        raise ValueError(f"a must be (m, d) and b (n, d), or (g, n, d) with offsets; got {tuple(a.shape)} and "
                         f"{tuple(b.shape)}")
    m, d = a.shape
    g, n = (b.shape[0], b.shape[1]) if grouped else (1, b.shape[0])
    if b.shape[-1] != d:
        raise ValueError(f"a and b disagree on the number of features: {d} and {b.shape[-1]}")
    wanted = [(a_scales, "a_scales", (m,)), (b_scales, "b_scales", b.shape[:-1])]
    if bias is not None:
        wanted.append((bias, "bias", b.shape[:-1]))
    for t, name, shape in wanted:
        require_cuda_tensor(t, name, torch.float32)
        if t.shape != shape:
            raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if grouped:
        require_cuda_tensor(offsets, "offsets", torch.int32)
        if offsets.shape != (g + 1,):
            raise ValueError(f"offsets must have shape ({g + 1},), got {tuple(offsets.shape)}")
    for t in (b, a_scales, b_scales, bias, offsets):
        if t is not None and t.device != a.device:
            raise ValueError(f"all operands must be on {a.device}, got {t.device}")
    if d > MAX_FEATURES:
        raise ValueError(f"at most {MAX_FEATURES} features (sums are held in 32 bits), got {d}")
    dev = a.device
    out = torch.empty((m, n), dtype=out_dtype, device=dev)
    if m == 0 or n == 0:
        return out
    if d == 0 or g == 0:
        raise ValueError("d and the number of groups must be at least 1")
    a, lda = _pitched(a, "a")
    b, ldb = _pitched(b, "b")
    launch("kmb_int8_matmul", dev, code, a.data_ptr(), lda, a_scales.data_ptr(), b.data_ptr(), ldb,
           b_scales.data_ptr(), None if bias is None else bias.data_ptr(),
           None if offsets is None else offsets.data_ptr(), g, out.data_ptr(), m, n, d)
    return out


def check_int8_waits(device=None):
    """Raises KmbError if a bounded wait inside `int8_matmul` ran out on `device` since the last call of
    this function (the output tiles concerned hold NaN).  Waits for the device's current stream."""
    flag = ctypes.c_int(0)
    with torch.cuda.device(device):
        check(lib.kmb_int8_wait_error(ctypes.byref(flag), stream_ptr(device)), "kmb_int8_wait_error")

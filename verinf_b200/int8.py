"""The quantised model's own arithmetic, beside the field products that prove it.

`int8_quantize_rows` turns rows of activations (or of a weight, one row an output channel) into int8 with one scale a row;
`int8_matmul` multiplies int8 matrices with exact 32-bit sums and gives the scaled product, the sums, or the sums as field
elements: the witness that `gl_matmul` gives for the operands lifted by the signed-to-field map (prover/loader.py:52-58), from
one pass over one byte plane instead of 64 plane products.

As elsewhere in the package: CUDA tensors, outputs allocated with torch (or given as `out`), kernels on torch's current stream
of the tensors' device, RuntimeError for what is refused.
"""
import ctypes as C

import torch

from ._lib import LIB, check, on_device, raw_stream

# element types of the C ABI (enum in include/verinf_b200.h)
DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int32: 3, torch.uint64: 4}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
MAX_K = 131071        # int8 products that a 32-bit sum holds


def _matrix(t, what, name, dtypes):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{what}: {name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{what}: {name} has dtype {t.dtype}, expected one of {', '.join(map(str, dtypes))}")
    if t.dim() != 2:
        raise RuntimeError(f"{what}: {name} must be 2-D")


def _rows_apart(t, what, name):
    """Elements from a row of a 2-D tensor to the next; the entries of a row must lie together."""
    if t.size(1) > 1 and t.stride(1) != 1:
        raise RuntimeError(f"{what}: the entries of a row of {name} must lie together (stride {t.stride(1)})")
    return t.stride(0) if t.size(0) > 1 else max(t.size(1), 1)


def int8_quantize_rows(x, out=None):
    """x (m, k), fp32 / fp16 / bf16, rows any distance apart -> (q int8 (m, k), scale fp32 (m,)).

    scale[r] = max_j |x[r, j]| / 127 and q[r, j] = the whole number nearest to 127 x[r, j] / max_j |x[r, j]|, ties to even: of
    the exact quotient, so that whoever quantises the same row gets the same whole numbers.  A row of zeros has scale 0; one
    that holds a NaN or an infinity has scale NaN and zeros.  `out`: a pair (q, scale) to write into; the rows of q may be any
    distance apart."""
    what = "int8_quantize_rows"
    _matrix(x, what, "x", _FLOATS)
    m, k = x.shape
    xs = _rows_apart(x, what, "x")
    if xs < k:
        x, xs = x.contiguous(), k                       # expanded rows
    if out is None:
        q = torch.empty((m, k), dtype=torch.int8, device=x.device)
        scale = torch.empty((m,), dtype=torch.float32, device=x.device)
        qs = k
    else:
        q, scale = out
        _matrix(q, what, "out[0]", (torch.int8,))
        if q.shape != x.shape or q.device != x.device:
            raise RuntimeError(f"{what}: out[0] must have x's shape and device")
        qs = _rows_apart(q, what, "out[0]")
        if qs < k:
            raise RuntimeError(f"{what}: rows of out[0] overlap")
        if not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 or scale.shape != (m,) or \
                scale.device != x.device or not scale.is_contiguous():
            raise RuntimeError(f"{what}: out[1] must be a contiguous fp32 tensor of {m} scales on x's device")
    with on_device(x.device):
        check(LIB.vi_int8_quantize_rows(x.data_ptr(), DTYPE_CODES[x.dtype], m, k, xs, q.data_ptr(), qs, scale.data_ptr(),
                                        raw_stream(x.device)))
    return q, scale


def _scales(s, n, dev, what, name):
    if s is None:
        return None
    if not isinstance(s, torch.Tensor) or s.dtype != torch.float32 or s.device != dev or s.shape != (n,) or not s.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be a contiguous fp32 tensor of {n} scales on the operands' device")
    return s.data_ptr()


def int8_matmul(A, B, scale_a=None, scale_b=None, dtype=torch.int32, out=None):
    """A (m, k) . B (k, n) of int8 matrices, summed exactly (k <= 131071).

    dtype fp32 / fp16 / bf16: (sum * scale_a[i]) * scale_b[j] in fp32, rounded once to the type; scales are fp32 vectors, one
    a token (row of A) and one a channel (column of B), and a missing one counts as ones.  dtype int32: the sums; dtype
    uint64: the sums as field elements, negative ones as p - |sum|; these two take no scales.

    The rows of A may be any distance apart.  B is row-major with rows any distance apart, or the transposed view of a weight
    stored by output channel (`weight.t()`), its channels any distance apart.  Rows (channels) that start on 16-byte
    boundaries are read in place; others are copied on every call.  `out`: a tensor of `dtype` to write into, rows any
    distance apart; it must not share memory with the operands."""
    what = "int8_matmul"
    _matrix(A, what, "A", (torch.int8,))
    _matrix(B, what, "B", (torch.int8,))
    if A.size(1) != B.size(0):
        raise RuntimeError(f"{what}: inner dim mismatch")
    if A.device != B.device:
        raise RuntimeError(f"{what}: operands on different devices")
    if dtype not in DTYPE_CODES:
        raise RuntimeError(f"{what}: dtype must be float32, float16, bfloat16, int32 or uint64")
    m, k = A.shape
    n = B.size(1)
    if k > MAX_K:
        raise RuntimeError(f"{what}: k = {k}, but 32-bit sums hold at most {MAX_K} products")
    if dtype not in _FLOATS and (scale_a is not None or scale_b is not None):
        raise RuntimeError(f"{what}: whole-number outputs take no scales")
    dev = A.device
    lda = _rows_apart(A, what, "A")
    if (B.stride(1) == 1 or n == 1) and (B.stride(0) >= n or k == 1):
        by_channel, ldb = 0, (B.stride(0) if k > 1 else n)
    elif (B.stride(0) == 1 or k == 1) and (B.stride(1) >= k or n == 1):
        by_channel, ldb = 1, (B.stride(1) if n > 1 else k)
    elif B.stride(0) and B.stride(1):
        raise RuntimeError(f"{what}: the rows or the columns of B must lie together (strides {B.stride()})")
    else:
        B = B.contiguous()                              # expanded
        by_channel, ldb = 0, n
    if lda < k:
        A, lda = A.contiguous(), k
    sa, sb = _scales(scale_a, m, dev, what, "scale_a"), _scales(scale_b, n, dev, what, "scale_b")
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=dev)
        ldc = n
    else:
        _matrix(out, what, "out", (dtype,))
        if out.shape != (m, n) or out.device != dev:
            raise RuntimeError(f"{what}: out must be ({m}, {n}) on the operands' device")
        ldc = _rows_apart(out, what, "out")
        if ldc < n:
            raise RuntimeError(f"{what}: rows of out overlap")
    a, b = A.data_ptr(), B.data_ptr()
    room, nb = None, LIB.vi_int8_matmul_scratch_bytes(a, lda, b, ldb, by_channel, m, k, n)
    if nb:
        room = torch.empty((nb,), dtype=torch.int8, device=dev)      # of the current stream: calls on two streams share nothing
    with on_device(dev):
        check(LIB.vi_int8_matmul(a, lda, b, ldb, by_channel, sa, sb, out.data_ptr(), DTYPE_CODES[dtype], ldc, m, k, n,
                                 room.data_ptr() if nb else None, nb, raw_stream(dev)))
    return out


def check_async_errors(device=None):
    """Raises if a product launched earlier on the device gave up on one of its bounded device-side waits (its output is then
    incomplete).  Waits for the device."""
    code = C.c_int(0)
    with torch.cuda.device(device):
        check(LIB.vi_int8_matmul_status(C.byref(code)))
    if code.value:
        raise RuntimeError(f"int8_matmul: a device-side wait expired (code {code.value}); the product written by that call is "
                           "incomplete")

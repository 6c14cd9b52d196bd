"""The quantised model's own arithmetic, beside the field products that prove it.

`int8_quantize_rows` turns rows of activations (or of a weight, one row an output channel) into int8 with one scale a row;
`int8_matmul` multiplies int8 matrices with exact 32-bit sums and gives the scaled product, the sums, or the sums as field
elements: the witness that `gl_matmul` gives for the operands lifted by the signed-to-field map (prover/loader.py:52-58), from
one pass over one byte plane instead of 64 plane products.

As elsewhere in the package: CUDA tensors, outputs allocated with torch (or given as `out`), kernels on torch's current stream
of the tensors' device, RuntimeError for what is refused.  Outputs carry no gradient: nothing in the package is trained.
"""
import ctypes as C

import torch

from ._lib import LIB, check, current_device, empty_strided, raw_stream

# element types of the C ABI (enum in include/verinf_b200.h)
DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int32: 3, torch.uint64: 4}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_INT8 = (torch.int8,)
MAX_K = 131071        # int8 products that a 32-bit sum holds


def matrix(t, what, name, dtypes):
    """(rows, columns, elements from a row to the next) of a 2-D CUDA tensor whose rows' entries lie together."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{what}: {name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{what}: {name} has dtype {t.dtype}, expected one of {', '.join(map(str, dtypes))}")
    shape = t.shape
    if len(shape) != 2:
        raise RuntimeError(f"{what}: {name} must be 2-D")
    rows, cols = shape
    apart, step = t.stride()
    if step != 1 and cols > 1:
        raise RuntimeError(f"{what}: the entries of a row of {name} must lie together (stride {step})")
    return rows, cols, apart if rows > 1 else cols


def _output(out, shape, dev, what, name, dtypes):
    """Row distance of a tensor to be written."""
    rows, cols, apart = matrix(out, what, name, dtypes)
    if (rows, cols) != shape or out.device != dev:
        raise RuntimeError(f"{what}: {name} must be {shape[0]} x {shape[1]} on the inputs' device")
    if apart < cols:
        raise RuntimeError(f"{what}: rows of {name} overlap")
    return apart


def _vector(s, n, dev, what, name):
    if not isinstance(s, torch.Tensor) or s.dtype is not torch.float32 or s.device != dev or s.shape != (n,) or not s.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be a contiguous fp32 tensor of {n} scales on the inputs' device")
    return s.data_ptr()


def int8_quantize_rows(x, out=None):
    """x (m, k), fp32 / fp16 / bf16, rows any distance apart -> (q int8 (m, k), scale fp32 (m,)).

    scale[r] = max_j |x[r, j]| / 127 and q[r, j] = the whole number nearest to 127 x[r, j] / max_j |x[r, j]|, ties to even: of
    the exact quotient, so that whoever quantises the same row gets the same whole numbers.  A row of zeros has scale 0; one
    that holds a NaN or an infinity has scale NaN and zeros.  `out`: a pair (q, scale) to write into; the rows of q may be any
    distance apart; neither shares memory with x or the other (a long row is read twice, after parts of it are written)."""
    index = x.get_device() if isinstance(x, torch.Tensor) else -1
    if index >= 0 and index != current_device():
        with torch.cuda.device(index):
            return int8_quantize_rows(x, out)
    what = "int8_quantize_rows"
    m, k, xs = matrix(x, what, "x", _FLOATS)
    if out is None:
        q, qs = empty_strided((m, k), (k, 1), torch.int8), k
        scale = empty_strided((m,), (1,), torch.float32)
        scale_ptr = scale.data_ptr()
    else:
        q, scale = out
        qs = _output(q, (m, k), x.device, what, "out[0]", _INT8)
        scale_ptr = _vector(scale, m, x.device, what, "out[1]")
    rc = LIB.vi_int8_quantize_rows(x.data_ptr(), DTYPE_CODES[x.dtype], m, k, xs, q.data_ptr(), qs, scale_ptr, raw_stream(index))
    if rc:
        check(rc)
    return q, scale


def _weight(B, what):
    """(k, n, by channel or not, distance of rows or channels) of a (k, n) operand that lies either way, copied if it is
    expanded."""
    if not isinstance(B, torch.Tensor) or not B.is_cuda:
        raise RuntimeError(f"{what}: B must be a CUDA tensor")
    if B.dtype is not torch.int8:
        raise RuntimeError(f"{what}: B has dtype {B.dtype}, expected torch.int8")
    shape = B.shape
    if len(shape) != 2:
        raise RuntimeError(f"{what}: B must be 2-D")
    k, n = shape
    s0, s1 = B.stride()
    if n == 1 and s0 == 1:                              # a column is one channel: a row of k instead of k rows of one
        return B, k, n, 1, k
    if (s1 == 1 or n == 1) and (s0 >= n or k == 1):
        return B, k, n, 0, s0 if k > 1 else n
    if (s0 == 1 or k == 1) and (s1 >= k or n == 1):
        return B, k, n, 1, s1 if n > 1 else k
    if s0 and s1:
        raise RuntimeError(f"{what}: the rows or the columns of B must lie together (strides {B.stride()})")
    return B.contiguous(), k, n, 0, n


def int8_matmul(A, B, scale_a=None, scale_b=None, dtype=torch.int32, out=None):
    """A (m, k) . B (k, n) of int8 matrices, summed exactly (k <= 131071).

    dtype fp32 / fp16 / bf16: (sum * scale_a[i]) * scale_b[j] in fp32, rounded once to the type; scales are fp32 vectors, one
    a token (row of A) and one a channel (column of B), and a missing one counts as ones.  dtype int32: the sums; dtype
    uint64: the sums as field elements, negative ones as p - |sum|; these two take no scales.

    The rows of A may be any distance apart.  B is row-major with rows any distance apart, or the transposed view of a weight
    stored by output channel (`weight.t()`), its channels any distance apart.  Rows (channels) that start on 16-byte
    boundaries are fastest; others are shifted on their way or copied, on every call.  `out`: a tensor of `dtype` to write
    into, rows any distance apart; it must not share memory with the operands or the scales."""
    index = A.get_device() if isinstance(A, torch.Tensor) else -1
    if index >= 0 and index != current_device():
        with torch.cuda.device(index):
            return int8_matmul(A, B, scale_a, scale_b, dtype, out)
    what = "int8_matmul"
    m, k, lda = matrix(A, what, "A", _INT8)
    B, kb, n, by_channel, ldb = _weight(B, what)
    if k != kb:
        raise RuntimeError(f"{what}: inner dim mismatch")
    if B.get_device() != index:
        raise RuntimeError(f"{what}: operands on different devices")
    code = DTYPE_CODES.get(dtype)
    if code is None:
        raise RuntimeError(f"{what}: dtype must be float32, float16, bfloat16, int32 or uint64")
    if k > MAX_K:
        raise RuntimeError(f"{what}: k = {k}, but 32-bit sums hold at most {MAX_K} products")
    if code > 2 and (scale_a is not None or scale_b is not None):
        raise RuntimeError(f"{what}: whole-number outputs take no scales")
    if lda < k:
        A, lda = A.contiguous(), k                      # expanded
    sa = None if scale_a is None else _vector(scale_a, m, A.device, what, "scale_a")
    sb = None if scale_b is None else _vector(scale_b, n, A.device, what, "scale_b")
    if out is None:
        out, ldc = empty_strided((m, n), (n, 1), dtype), n
    else:
        ldc = _output(out, (m, n), A.device, what, "out", (dtype,))
    a, b, room, nb = A.data_ptr(), B.data_ptr(), None, 0
    if (a | b | lda | ldb) & 15:                        # an operand may have to be copied
        nb = LIB.vi_int8_matmul_scratch_bytes(a, lda, b, ldb, by_channel, m, k, n)
        if nb:
            room = empty_strided((nb,), (1,), torch.int8)      # of the current stream: calls on two streams share nothing
    rc = LIB.vi_int8_matmul(a, lda, b, ldb, by_channel, sa, sb, out.data_ptr(), code, ldc, m, k, n, room.data_ptr() if nb else None,
                            nb, raw_stream(index))
    if rc:
        check(rc)
    return out


def check_async_errors(device=None):
    """Raises if a product launched earlier on the device gave up on one of its bounded device-side waits (its output is then
    incomplete).  Waits for all streams of the device, so it is not called while one is captured."""
    code = C.c_int(0)
    with torch.cuda.device(device):
        check(LIB.vi_int8_matmul_status(C.byref(code)))
    if code.value:
        raise RuntimeError(f"int8_matmul: a device-side wait expired (code {code.value}); the product written by that call is "
                           "incomplete")

"""The quantised model's operators: int8 rows, int8 products, token log probabilities, against plain implementations in 64
bits; what they refuse; a run of them together.  Tolerances are counted in roundings: half a step is 2^-24 of the value in
fp32, 2^-11 in fp16, 2^-8 in bf16."""
import ctypes as C
import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

P = (1 << 64) - (1 << 32) + 1
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLOATS = [torch.float32, torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from verinf_b200 import _lib
    return _lib


@pytest.fixture(scope="module")
def i8():
    from verinf_b200 import int8
    return int8


@pytest.fixture(scope="module")
def lp():
    from verinf_b200 import logprobs
    return logprobs


# ---- refusals of the C ABI, before any kernel runs (no GPU) -------------------------------------------------------
def _err(lib):
    return lib.LIB.vi_last_error().decode()


def _buf():
    b = (C.c_uint64 * 64)()
    return b, C.cast(b, C.c_void_p).value


def test_quantize_refusals_without_gpu(lib):
    L = lib.LIB
    keep, p = _buf()
    assert L.vi_int8_quantize_rows(p, 3, 1, 4, 4, p, 4, p, None) != 0 and "dtype" in _err(lib)
    assert L.vi_int8_quantize_rows(p, 0, -1, 4, 4, p, 4, p, None) != 0 and "negative" in _err(lib)
    assert L.vi_int8_quantize_rows(p, 0, 1 << 31, 4, 4, p, 4, p, None) != 0 and "rows" in _err(lib)
    assert L.vi_int8_quantize_rows(p, 0, 2, 4, -4, p, 4, p, None) != 0 and "negative" in _err(lib)
    assert L.vi_int8_quantize_rows(p, 0, 2, 4, 4, p, 3, p, None) != 0 and "overlap" in _err(lib)
    assert L.vi_int8_quantize_rows(p + 2, 0, 1, 4, 4, p, 4, p, None) != 0 and "aligned" in _err(lib)
    assert L.vi_int8_quantize_rows(p, 0, 1, 4, 4, p, 4, None, None) != 0 and "scale" in _err(lib)
    assert L.vi_int8_quantize_rows(None, 0, 1, 4, 4, p, 4, p, None) != 0 and "null" in _err(lib)
    assert L.vi_int8_quantize_rows(None, 0, 0, 4, 4, None, 4, None, None) == 0


def test_matmul_refusals_without_gpu(lib):
    L = lib.LIB
    keep, p = _buf()

    def call(A=p, lda=4, B=p, ldb=4, nk=0, sa=None, sb=None, Cp=p, out=3, ldc=4, m=2, k=4, n=4):
        return L.vi_int8_matmul(A, lda, B, ldb, nk, sa, sb, Cp, out, ldc, m, k, n, None, 0, None)
    assert call(m=-1) != 0 and "negative" in _err(lib)
    assert call(out=5) != 0 and "output type" in _err(lib)
    assert call(out=-1) != 0 and "output type" in _err(lib)
    assert call(k=131072) != 0 and "131071" in _err(lib)
    assert call(out=3, sa=p) != 0 and "no scales" in _err(lib)
    assert call(out=4, sb=p) != 0 and "no scales" in _err(lib)
    assert call(Cp=None) != 0 and "output" in _err(lib)
    assert call(Cp=p + 2) != 0 and "misaligned output" in _err(lib)
    assert call(ldc=3) != 0 and "overlap" in _err(lib)
    assert call(A=None) != 0 and "null input" in _err(lib)
    assert call(out=0, sa=p + 1) != 0 and "scales" in _err(lib)
    assert call(lda=3) != 0 and "operand rows overlap" in _err(lib)
    assert call(nk=1, k=5, lda=5) != 0 and "operand rows overlap" in _err(lib)
    assert call(A=p + 1, lda=3001, ldb=2001, m=700, k=3001, n=2001, ldc=2001) != 0 and "scratch" in _err(lib)
    assert L.vi_int8_matmul_scratch_bytes(16, 16, 32, 16, 0, 2, 4, 4) == 0
    assert L.vi_int8_matmul_scratch_bytes(16, 17, 33, 16, 1, 2, 17, 5) == 0          # shifted on the way
    assert L.vi_int8_matmul_scratch_bytes(16, 3001, 32, 2001, 0, 700, 3001, 2001) == 700 * 3008 + 3001 * 2016
    assert L.vi_int8_matmul_scratch_bytes(16, 3008, 33, 3008, 1, 700, 3001, 2001) == 2001 * 3008
    assert L.vi_int8_matmul_status(None) != 0 and "null" in _err(lib)
    assert call(m=0, A=None, Cp=None) == 0
    assert call(n=0, A=None, Cp=None) == 0


def test_matmul_size_limits_without_gpu(lib):
    """Sizes whose last tile would end beyond 31-bit indices are refused; the scratch of the largest allowed ones is known."""
    L = lib.LIB
    keep, p = _buf()
    most = (1 << 31) - 256
    for m, n in [(most + 1, 16), (16, most + 1), (1 << 40, 1)]:
        assert L.vi_int8_matmul_scratch_bytes(p + 1, 17, p, 16, 1, m, 16, n) == 0
        assert L.vi_int8_matmul(p + 1, 17, p, 16, 1, None, None, p, 3, n, m, 16, n, None, 0, None) != 0 and "2^31 - 256" in _err(lib)
    assert L.vi_int8_matmul_scratch_bytes(p + 1, 131072, 16, 131072, 1, most, 131071, 16) == most * 131072
    assert L.vi_int8_matmul_scratch_bytes(16, 131072, 16, 131072, 1, most, 131071, most) == 0


def test_logprobs_refusals_without_gpu(lib):
    L = lib.LIB
    keep, p = _buf()

    def call(x=p, dtype=0, rows=1, vocab=4, stride=4, tok=p, top=0, t=1.0, a=p, b=p, tl=p, tt=p):
        return L.vi_token_logprobs(x, dtype, rows, vocab, stride, tok, top, t, a, b, tl, tt, None)
    assert call(dtype=3) != 0 and "dtype" in _err(lib)
    assert call(rows=-1) != 0
    assert call(vocab=0) != 0 and "vocab" in _err(lib)
    assert call(vocab=1 << 31) != 0 and "limited" in _err(lib)
    assert call(top=33) != 0 and "top" in _err(lib)
    assert call(top=-1) != 0 and "top" in _err(lib)
    for t in (0.0, -1.0, float("nan"), float("inf")):
        assert call(t=t) != 0 and "temperature" in _err(lib)
    assert call(x=None) != 0 and "null" in _err(lib)
    assert call(top=1, tl=None) != 0 and "null" in _err(lib)
    assert call(x=p + 2) != 0 and "aligned" in _err(lib)
    assert call(tok=p + 4) != 0 and "misaligned" in _err(lib)
    assert call(rows=2, stride=-4) != 0 and "stride" in _err(lib)
    assert call(rows=0, x=None, tok=None) == 0


def test_python_refusals_without_gpu(i8, lp):
    with pytest.raises(RuntimeError, match="CUDA"):
        i8.int8_quantize_rows(torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="CUDA"):
        i8.int8_matmul(torch.zeros(2, 3, dtype=torch.int8), torch.zeros(3, 2, dtype=torch.int8))
    with pytest.raises(RuntimeError, match="CUDA"):
        lp.token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))


# ---- rows to int8 --------------------------------------------------------------------------------------------------
def _quantize_64(x):
    """In 64 bits the quotient of 31-bit by 24-bit numbers never rounds onto a border that it is not on: it differs from a
    half-integer by at least 2^-33 of itself."""
    x = x.detach().cpu().double()
    big = x.abs().amax(1, keepdim=True) if x.size(1) else torch.zeros(x.size(0), 1, dtype=torch.float64)
    bad = ~torch.isfinite(x).all(1)
    safe = torch.where((big > 0) & torch.isfinite(big), big, 1.0)
    q = torch.where(bad[:, None], 0.0, torch.nan_to_num(127 * x / safe, 0, 0, 0)).round().to(torch.int8)
    scale = big[:, 0].float() / np.float32(127)                     # one division in fp32
    return q, torch.where(bad, float("nan"), scale)


def _check_quantize(i8, x, **kw):
    q, s = i8.int8_quantize_rows(x, **kw)
    wq, ws = _quantize_64(x)
    assert torch.equal(q.cpu(), wq)
    assert torch.equal(torch.nan_to_num(s.cpu(), -1), torch.nan_to_num(ws, -1))


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 7), (3, 8), (2, 129), (5, 1000), (1, 4096), (33, 5003), (2, 16384), (2, 40001), (1000, 96)])
def test_quantize_sizes(i8, dtype, m, k):
    g = torch.Generator().manual_seed(m * 7919 + k)
    x = (torch.randn(m, k, generator=g) * torch.exp(3 * torch.randn(m, 1, generator=g))).to(dtype).cuda()
    _check_quantize(i8, x)


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_borders(i8, dtype):
    """Rows whose quotients fall on borders exactly, or next to them: maxima 127 and 254 with halves, neighbours of halves."""
    halves = torch.arange(-127, 127).double() + 0.5
    rows = [torch.cat([halves, torch.tensor([127.0])]), torch.cat([2 * halves, torch.tensor([-254.0])]),
            torch.cat([halves * 4, torch.tensor([127.0 * 4])])]
    near = [torch.nextafter(halves.float(), torch.full_like(halves.float(), s)).double() for s in (-1e9, 1e9)]
    rows += [torch.cat([n, torch.tensor([127.0])]) for n in near]
    x = torch.stack(rows).to(dtype)
    _check_quantize(i8, x.cuda())
    odd = torch.stack([torch.cat([halves * f, torch.tensor([127.0 * f])]) for f in (1 / 3, 0.7, 1.1, 97.3)]).to(dtype)
    _check_quantize(i8, odd.cuda())


@gpu
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 7), (torch.float16, 10)])
@pytest.mark.parametrize("gap", [0, 1, 2, 4, 7])
def test_quantize_every_quotient_of_16_bits(i8, dtype, bits, gap):
    """Rows with every significand as their maximum, in them every significand `gap` binades lower, against whole numbers:
    127 x / a = 127 i 2^-gap / j for significands i and j.  fp16 values near 1, so that none is subnormal."""
    n = 1 << bits
    j = torch.arange(n, 2 * n, device="cuda")
    i = torch.arange(n, 2 * n, device="cuda").repeat(n, 1)
    i = torch.where(i <= j[:, None] << gap, i, 0)                    # not above the maximum
    x = torch.cat([i * 2.0 ** (-gap - bits), -(j[:, None] * 2.0 ** -bits)], 1)
    q, _ = i8.int8_quantize_rows(x.to(dtype))
    num, den = 127 * i, j[:, None] << gap
    low, rest = num // den, num % den * 2
    want = low + ((rest > den) | ((rest == den) & (low % 2 == 1)))
    assert (x.to(dtype).double() == x).all()
    assert torch.equal(q[:, :-1].long(), want) and (q[:, -1] == -127).all()


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_extremes(i8, dtype):
    """The type's largest, smallest and subnormal values, rows of zeros, rows with NaN and infinities."""
    f = torch.finfo(dtype)
    tiny = f.smallest_normal * f.eps                                # the least subnormal value
    g = torch.Generator().manual_seed(5)
    base = torch.randn(8, 300, generator=g).double().clamp(-1, 1)
    base[:, 0] = 1
    x = torch.zeros(12, 300, dtype=dtype)
    x[0] = (base[0] * f.max).to(dtype)
    x[1] = (base[1] * f.smallest_normal).to(dtype)
    x[2] = (base[2] * tiny * 5).to(dtype)
    x[3, 17] = tiny
    x[4, 5] = -f.max
    x[4, 6] = tiny
    x[6] = base[3].to(dtype); x[6, 299] = float("nan")
    x[7] = base[4].to(dtype); x[7, 0] = float("inf")
    x[8] = base[5].to(dtype); x[8, 131] = -float("inf")
    x[9] = (base[6] * f.smallest_normal * 64).to(dtype)
    x[10] = -0.0
    x[11] = (base[7] * f.smallest_normal * 3).to(dtype)
    _check_quantize(i8, x.cuda())


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("offset,pitch", [(0, 1040), (0, 1033), (1, 1040), (3, 1029), (8, 1040)])
def test_quantize_strides_and_out(i8, dtype, offset, pitch):
    g = torch.Generator().manual_seed(offset + pitch)
    k = 1003
    buf = torch.randn(9, pitch + 16, generator=g).to(dtype).cuda()
    x = buf[:, offset:offset + k]
    _check_quantize(i8, x)
    room = torch.full((9, pitch), 77, dtype=torch.int8, device="cuda")
    scale = torch.empty(9, device="cuda")
    q, s = i8.int8_quantize_rows(x, out=(room[:, 5:5 + k], scale))
    wq, ws = _quantize_64(x)
    assert torch.equal(room[:, 5:5 + k].cpu(), wq) and torch.equal(scale.cpu(), ws)
    assert (room[:, :5] == 77).all() and (room[:, 5 + k:] == 77).all()
    _check_quantize(i8, x[:1].expand(4, k))


@gpu
def test_quantize_empty_and_refusals(i8):
    q, s = i8.int8_quantize_rows(torch.empty(0, 5, device="cuda"))
    assert q.shape == (0, 5) and s.shape == (0,)
    q, s = i8.int8_quantize_rows(torch.empty(3, 0, device="cuda"))
    assert q.shape == (3, 0) and (s == 0).all()
    x = torch.zeros(4, 6, device="cuda")
    q, s = torch.empty(4, 6, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    for bad, words in [((x.double(),), "dtype"), ((x[0],), "2-D"), ((x.t(),), "lie together")]:
        with pytest.raises(RuntimeError, match=words):
            i8.int8_quantize_rows(*bad)
    for out, words in [((q[:3], s), "must be 4 x 6"), ((q.to(torch.int32), s), "dtype"), ((q[:1].expand(4, 6), s), "overlap"),
                       ((q, s[:3]), "scales"), ((q, s.double()), "scales"), ((q, s.cpu()), "scales"), ((q.cpu(), s), "CUDA"),
                       ((torch.empty(6, 4, dtype=torch.int8, device="cuda").t(), s), "lie together")]:
        with pytest.raises(RuntimeError, match=words):
            i8.int8_quantize_rows(x, out=out)


# ---- product --------------------------------------------------------------------------------------------------------
def _sums_64(A, B):
    return (A.cpu().double() @ B.cpu().double()).to(torch.int64)        # |sum| < 2^31: whole in 64-bit floats


def _field(S):
    return np.where(S.numpy() < 0, S.numpy() + np.int64(P - (1 << 64)), S.numpy())


def _rand8(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)


def _weight(g, k, n, layout, pad):
    """(k, n) int8 on the GPU: row-major ("kn") or by channel ("nk"), `pad` bytes behind each row or channel."""
    r, c = (k, n) if layout == "kn" else (n, k)
    buf = _rand8(g, r, c + pad).cuda()[:, :c]
    return buf if layout == "kn" else buf.t()


def _check_matmul(i8, A, B, dtypes=None, g=None, out_pad=0):
    m, n = A.size(0), B.size(1)
    S = _sums_64(A, B)
    for dtype in dtypes or [torch.int32, torch.uint64] + FLOATS:
        out = None
        if out_pad:
            room = torch.full((m, n + out_pad), 7, device="cuda").to(dtype) if dtype != torch.uint64 else \
                torch.full((m, n + out_pad), 7, dtype=torch.int64, device="cuda").view(torch.uint64)
            out = room[:, :n]
        if dtype == torch.int32:
            assert torch.equal(i8.int8_matmul(A, B, dtype=dtype, out=out).cpu().to(torch.int64), S)
        elif dtype == torch.uint64:
            got = i8.int8_matmul(A, B, dtype=dtype, out=out).view(torch.int64).cpu().numpy()
            assert np.array_equal(got, _field(S))
        else:
            sa = torch.rand(m, generator=g) * 0.05 + 1e-3
            sb = torch.rand(n, generator=g) * 0.02 + 1e-4
            got = i8.int8_matmul(A, B, sa.cuda(), sb.cuda(), dtype=dtype, out=out).cpu().double()
            want = S.double() * sa.double()[:, None] * sb.double()
            # roundings: the sum to fp32, two products, the output type (fp32: the second product already is it)
            tol = want.abs() * (3 * HALF[torch.float32] + (HALF[dtype] if dtype != torch.float32 else 0)) * 1.001
            tol = tol + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            big = want.abs() > torch.finfo(dtype).max
            assert ((got - want).abs() <= tol)[~big].all() and torch.isinf(got[big & (want.abs() > 2 * torch.finfo(dtype).max)]).all()
        if out_pad:
            assert (room.view(torch.int64 if dtype == torch.uint64 else dtype)[:, n:] == 7).all()


@gpu
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 16, 8), (2, 3, 5), (7, 33, 9), (1, 4096, 512), (3, 1000, 130), (16, 128, 128),
                                   (17, 257, 129), (31, 515, 1001), (64, 1024, 256), (65, 48, 300), (128, 384, 640), (129, 1001, 515),
                                   (255, 64, 31), (300, 2048, 384), (513, 640, 272), (700, 3001, 2001), (2, 1925, 1098), (20, 77, 1125)])
def test_matmul_sizes(i8, layout, m, k, n):
    g = torch.Generator().manual_seed(m + 31 * k + 101 * n)
    _check_matmul(i8, _rand8(g, m, k).cuda(), _weight(g, k, n, layout, 0), g=g)


@gpu
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("m", [1, 5, 40, 200])
@pytest.mark.parametrize("pad,a_pad,offset", [(0, 0, 1), (16, 32, 0), (5, 3, 0), (11, 0, 7), (0, 9, 0)])
def test_matmul_strides(i8, layout, m, pad, a_pad, offset):
    g = torch.Generator().manual_seed(m + pad + a_pad + offset)
    k, n = 272, 336
    A = _rand8(g, m, k + a_pad + offset).cuda()[:, offset:offset + k]
    B = _weight(g, k + offset, n + offset, layout, pad)[offset:, offset:]
    _check_matmul(i8, A, B, [torch.int32, torch.bfloat16], g)
    _check_matmul(i8, A, B, g=g, out_pad=3)


@gpu
@pytest.mark.parametrize("m", [1, 33, 300])
def test_matmul_extreme_sums(i8, m):
    """The largest sums: every product 2^14 at the longest k, either sign."""
    k, n = 131071, 24
    A = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    B = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    B[1::2] = 127
    got = i8.int8_matmul(A, B.t())
    assert (got[:, 0::2] == 16384 * k).all() and (got[:, 1::2] == -16256 * k).all()
    got = i8.int8_matmul(A, B.t(), dtype=torch.uint64).view(torch.int64)
    assert (got[:, 0::2] == 16384 * k).all() and (got[:, 1::2] == P - (1 << 64) - 16256 * k).all()


@gpu
def test_matmul_scales(i8):
    """Missing scales are ones, an infinite or NaN scale reaches its row or column only, results beyond fp16 are infinite."""
    g = torch.Generator().manual_seed(3)
    A, B = _rand8(g, 20, 64).cuda(), _weight(g, 64, 40, "nk", 0)
    S = _sums_64(A, B)
    assert torch.equal(i8.int8_matmul(A, B, dtype=torch.float32).cpu(), S.float())
    sa = torch.ones(20, device="cuda"); sa[4] = float("nan")
    y = i8.int8_matmul(A, B, sa, dtype=torch.float32).cpu()
    assert torch.isnan(y[4]).all() and torch.equal(y[[3, 5]], S[[3, 5]].float())
    sb = torch.full((40,), 2.0, device="cuda"); sb[7] = 1e30
    y = i8.int8_matmul(A, B, None, sb, dtype=torch.float16).cpu()
    assert torch.isinf(y[:, 7][S[:, 7] != 0]).all() and torch.equal(y[:, 6], (2 * S[:, 6]).half())


@gpu
def test_matmul_empty_and_refusals(i8):
    z = lambda *s: torch.zeros(s, dtype=torch.int8, device="cuda")
    assert i8.int8_matmul(z(0, 4), z(4, 3)).shape == (0, 3)
    assert i8.int8_matmul(z(2, 4), z(4, 0)).shape == (2, 0)
    assert (i8.int8_matmul(z(2, 0), z(0, 3)) == 0).all()
    assert (i8.int8_matmul(z(2, 0), z(0, 3), torch.full((2,), 3.0, device="cuda"), dtype=torch.bfloat16) == 0).all()
    g = torch.Generator().manual_seed(1)
    A = _rand8(g, 1, 40).cuda().expand(6, 40)                      # expanded operands
    B = _rand8(g, 40, 1).cuda().expand(40, 24)
    assert torch.equal(i8.int8_matmul(A, B).cpu().long(), _sums_64(A, B))
    B = _rand8(g, 1, 24).cuda().expand(40, 24)
    assert torch.equal(i8.int8_matmul(A, B).cpu().long(), _sums_64(A, B))
    one = torch.ones
    for args, kw, words in [((z(2, 3), z(4, 2)), {}, "inner dim"), ((z(2, 3).float(), z(3, 2)), {}, "dtype"), ((z(2, 3)[0], z(3, 2)), {}, "2-D"),
                            ((z(2, 3), z(3, 2).cpu()), {}, "CUDA"), ((z(2, 3), z(3, 2)), dict(dtype=torch.float64), "dtype must be"),
                            ((z(2, 3), z(3, 2), one(2, device="cuda")), {}, "no scales"),
                            ((z(2, 3), z(3, 2), one(3, device="cuda")), dict(dtype=torch.float16), "scale_a"),
                            ((z(2, 3), z(3, 2), one(2)), dict(dtype=torch.float16), "scale_a"),
                            ((z(2, 3), z(3, 2), None, one(2, device="cuda").double()), dict(dtype=torch.float16), "scale_b"),
                            ((z(3, 2).t(), z(3, 2)), {}, "lie together"), ((z(2, 3), z(6, 4)[::2, ::2]), {}, "lie together"),
                            ((z(1, 131072), z(131072, 1)), {}, "131071"),
                            ((z(2, 3), z(3, 2)), dict(out=torch.empty(2, 2, device="cuda")), "out"),
                            ((z(2, 3), z(3, 2)), dict(out=torch.empty(2, 3, dtype=torch.int32, device="cuda")), "out must"),
                            ((z(2, 3), z(3, 2)), dict(out=torch.empty(1, 2, dtype=torch.int32, device="cuda").expand(2, 2)), "overlap")]:
        with pytest.raises(RuntimeError, match=words):
            i8.int8_matmul(*args, **kw)


@gpu
@pytest.mark.parametrize("m,n", [(1, 1), (3, 700), (2000, 5)])
def test_matmul_without_terms(i8, m, n):
    """k = 0: sums of 0, NaN where a scale is not finite; rows of the output any distance apart."""
    A, B = torch.empty(m, 0, dtype=torch.int8, device="cuda"), torch.empty(0, n, dtype=torch.int8, device="cuda")
    sa, sb = torch.ones(m, device="cuda"), torch.full((n,), 2.0, device="cuda")
    sa[m // 2], sb[n // 2] = math.nan, -math.inf
    bad = (torch.arange(m) == m // 2)[:, None] | (torch.arange(n) == n // 2)
    for dtype in FLOATS:
        room = torch.full((m, n + 3), 7.0, device="cuda", dtype=dtype)
        y = i8.int8_matmul(A, B, sa, sb, dtype=dtype, out=room[:, :n]).cpu()
        assert torch.isnan(y[bad]).all() and (y[~bad] == 0).all() and (room[:, n:] == 7).all()
        assert (i8.int8_matmul(A, B.t().contiguous().t(), dtype=dtype) == 0).all()
    for dtype in (torch.int32, torch.uint64):
        assert (i8.int8_matmul(A, B, dtype=dtype).view(torch.int32) == 0).all()


@gpu
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_matmul_witness_is_the_field_product(i8, layout):
    from verinf_b200 import cuda_primitives as cp
    g = torch.Generator().manual_seed(8)
    A, B = _rand8(g, 200, 700).cuda(), _weight(g, 700, 333, layout, 0)
    lift = lambda t: torch.where(t < 0, t.long() + (P - (1 << 64)), t.long()).contiguous().view(torch.uint64)
    want = cp.gl_matmul(lift(A), lift(B))
    assert torch.equal(i8.int8_matmul(A, B, dtype=torch.uint64).view(torch.int64), want.view(torch.int64))


# ---- log probabilities ------------------------------------------------------------------------------------------------
def _logprobs_64(x, tokens, top, temperature):
    x = x.cpu().double()
    rows, vocab = x.shape
    tokens = tokens.cpu()
    lp, ent = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    tl, tt = torch.full((rows, top), -math.inf, dtype=torch.float64), torch.full((rows, top), -1, dtype=torch.int64)
    log_z, width = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    for r in range(rows):
        v, t = x[r], int(tokens[r])
        if torch.isnan(v).any() or (v == math.inf).any():
            lp[r] = ent[r] = math.nan
            tl[r] = math.nan
        elif (v == -math.inf).all():
            lp[r] = -math.inf
        else:
            z = (v - v.max()) / temperature
            e = z.exp()
            s = e.sum()
            log_z[r] = s.log()
            w = (e * torch.where(e > 0, z, 0.0)).sum() / s
            width[r] = -w
            ent[r] = s.log() - w
            lp[r] = z[max(0, min(t, vocab - 1))] - s.log()
            order = torch.sort(v, descending=True, stable=True)[1][:top]
            order = order[v[order] > -math.inf]
            tt[r, :len(order)] = order
            tl[r, :len(order)] = z[order] - s.log()
        if t < 0:
            lp[r] = 0
        elif t >= vocab:
            lp[r] = math.nan
    return lp, ent, tl, tt, log_z, width


def _near(got, want, tol):
    # the value is an fp32 number: one of more than 2^128 (1 - 2^-25) in size is infinite there, as -2 * 3.4e38 is
    got, want = got.cpu().double(), want.float().double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    return bool((same | ((got - want).abs() <= tol)).all())


def _check_logprobs(lp_mod, x, tokens, top=0, temperature=1.0):
    out = lp_mod.token_logprobs(x, tokens, top=top, temperature=temperature)
    lp, ent, tl, tt, log_z, width = _logprobs_64(x, tokens, top, temperature)
    assert torch.equal(out.top_token.cpu(), tt)
    # Half steps of fp32.  An exponential: its argument is a difference, a product and a rounded constant (3 half steps of
    # |z|, and only |z| < 24 counts: the rest is below half a step of the sum) and the function itself (4).  The sum: one
    # rounding a term of a thread's chain (vocab / 256 terms) and of the tree, rescaling included (64).  The logarithm and
    # the difference: 4 each of their values; z of the token itself: 3.
    u = HALF[torch.float32]
    rel = (3 * 24 + 4 + x.size(1) / 256 + 64) * u
    assert _near(out.logprob, lp, rel + u * (8 * log_z + 4 * torch.nan_to_num(lp, 0, 0, 0).abs()))
    assert _near(out.entropy, ent, rel * (1 + 2 * width) + 8 * u * (log_z + width))
    assert _near(out.top_logprob, tl, rel + u * (8 * log_z[:, None] + 4 * torch.nan_to_num(tl, 0, 0, 0).abs()))


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 5), (2, 7, 32), (4, 8, 3), (2, 31, 8), (5, 255, 20), (9, 1000, 32), (3, 4099, 20),
                                            (2, 32000, 20), (1, 70001, 32), (300, 513, 4), (2, 202045, 20), (2, 2048, 0)])
def test_logprobs_sizes(lp, dtype, rows, vocab, top):
    g = torch.Generator().manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).cuda()
    tokens = torch.randint(0, vocab, (rows,), generator=g).cuda()
    _check_logprobs(lp, x, tokens, top)
    _check_logprobs(lp, x, tokens, top, temperature=0.6)


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_logprobs_masks_and_special_rows(lp, dtype, low):
    vocab, top = 3001, 20
    g = torch.Generator().manual_seed(11)
    low = -math.inf if low == "inf" else torch.finfo(dtype).min
    x = (torch.randn(14, vocab, generator=g) * 4).to(dtype)
    tokens = torch.randint(0, vocab, (14,), generator=g)
    x[0, torch.rand(vocab, generator=g) < 0.9] = low
    x[1] = low                                        # nothing left
    x[2] = low; x[2, 1234] = 3.5                      # one token left, the one asked for or another
    tokens[2] = 1234
    x[3] = low; x[3, 77] = -20
    x[4, 2000] = math.nan
    x[5, 3000] = math.inf
    x[6] = 1.25                                       # all alike
    tokens[7] = -1
    tokens[8] = vocab
    tokens[9] = -100
    x[10] = low; x[10, 5:12] = 0.5; x[10, 3000] = 0.5  # fewer than the list holds
    x[11] = 0; x[11, ::3] = -0.0                      # equal zeros of either sign
    x[12] = torch.finfo(dtype).max * torch.tensor([1, 0.5, -1]).repeat(vocab)[:vocab]
    x[13] = torch.linspace(-9, 9, vocab)
    _check_logprobs(lp, x.to(dtype).cuda(), tokens.cuda(), top)


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_logprobs_orders_and_crowded_lists(lp, dtype):
    """Rising and falling rows, runs of equal values, and rows whose allowed entries crowd in a few threads' shares."""
    vocab = 70000
    x = torch.full((7, vocab), -math.inf)
    x[0] = torch.linspace(-5, 5, vocab)
    x[1] = torch.linspace(5, -5, vocab)
    x[2] = (torch.arange(vocab) // 100 % 7).float()
    i = torch.arange(vocab)
    for r, step in ((3, 512), (4, 1024), (5, 2048)):
        at = i % step < 16
        x[r, at] = torch.arange(int(at.sum())).float() / 512
    x[6] = 2.0
    tokens = torch.tensor([69999, 0, 5, 512, 1024, 2048, 33])
    _check_logprobs(lp, x.to(dtype).cuda(), tokens.cuda(), 32)
    _check_logprobs(lp, x.to(dtype).cuda(), tokens.cuda(), 1, temperature=2.0)


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("offset,pitch", [(0, 4016), (0, 4003), (1, 4016), (8, 4016), (3, 4005)])
def test_logprobs_strides(lp, dtype, offset, pitch):
    g = torch.Generator().manual_seed(offset + pitch)
    x = (torch.randn(6, pitch + 16, generator=g) * 3).to(dtype).cuda()
    x[:, offset + 3999:] = 100.0                       # behind the vocabulary: must not be read as part of it
    x[:, :offset] = 100.0
    tokens = torch.randint(0, 3999, (6,), generator=g).cuda()
    _check_logprobs(lp, x[:, offset:offset + 3999], tokens, 8)
    _check_logprobs(lp, x[2:3, offset:offset + 3999].expand(5, 3999), tokens[:5].contiguous(), 3)


@gpu
@pytest.mark.parametrize("temperature", [1e-6, 0.05, 30.0, 1e6])
def test_logprobs_temperatures(lp, temperature):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 1500, generator=g) * 5
    x[1] *= 1000
    x[2] = (x[2] * 8).round() / 8
    tokens = x.argmax(1)
    tokens[3] = 7
    out = lp.token_logprobs(x.cuda(), tokens.cuda(), top=5, temperature=temperature)
    # c = 1 / T is rounded: a difference of |z| costs two more half steps, beside those counted for T = 1
    w = _logprobs_64(x, tokens, 5, temperature)
    u = HALF[torch.float32]
    rel = (5 * 24 + 4 + 1500 / 256 + 64) * u
    assert torch.equal(out.top_token.cpu(), w[3])
    assert _near(out.logprob, w[0], rel + u * (8 * w[4] + 6 * w[0].abs()))
    assert _near(out.entropy, w[1], rel * (1 + 2 * w[5]) + 8 * u * (w[4] + w[5]))
    assert _near(out.top_logprob, w[2], rel + u * (8 * w[4][:, None] + 6 * w[2].abs()))


@gpu
def test_logprobs_refusals(lp):
    x, t = torch.zeros(3, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    assert lp.token_logprobs(x[:0], t[:0], top=4).top_token.shape == (0, 4)
    for args, kw, words in [((x.double(), t), {}, "dtype"), ((x[0], t), {}, "2-D"), ((x, t[:2]), {}, "tokens"), ((x, t.int()), {}, "tokens"),
                            ((x, t.cpu()), {}, "tokens"), ((x, t), dict(top=33), "top"), ((x, t), dict(top=-1), "top"),
                            ((x, t), dict(top=2.0), "top"), ((x, t), dict(temperature=0.0), "temperature"),
                            ((x, t), dict(temperature=math.nan), "temperature"), ((torch.zeros(8, 3, device="cuda").t(), t), {}, "lie together"),
                            ((x[:, :0], t), {}, "vocab")]:
        with pytest.raises(RuntimeError, match=words):
            lp.token_logprobs(*args, **kw)


# ---- together, as they are used ------------------------------------------------------------------------------------------
def _answer(i8, lp, hidden, weight, sw, tokens, out=None):
    q, s = i8.int8_quantize_rows(hidden, out=out)
    logits = i8.int8_matmul(q, weight.t(), s, sw, dtype=torch.float32)
    witness = i8.int8_matmul(q, weight.t(), dtype=torch.uint64)
    return (q, s, logits, witness) + tuple(lp.token_logprobs(logits, tokens, top=5))


@gpu
@pytest.mark.parametrize("m", [1, 9, 150])
def test_answers_of_a_quantised_head(i8, lp, m):
    """Hidden states to int8, the head product as logits and as witness, log probabilities of the answers: each against 64
    bits from its own inputs, a second run on another stream and a captured and replayed one the same bit for bit."""
    g = torch.Generator().manual_seed(m)
    d, vocab = 1024, 5003
    hidden = torch.randn(m, d, generator=g).bfloat16().cuda()
    weight, sw = i8.int8_quantize_rows((torch.randn(vocab, d, generator=g) * 0.1).cuda())
    tokens = torch.randint(0, vocab, (m,), generator=g).cuda()
    first = _answer(i8, lp, hidden, weight, sw, tokens)
    q, s, logits, witness = first[:4]
    wq, ws = _quantize_64(hidden)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    S = _sums_64(q, weight.t())
    assert np.array_equal(witness.view(torch.int64).cpu().numpy(), _field(S))
    want = S.double() * ws.double()[:, None] * sw.cpu().double()
    assert ((logits.cpu().double() - want).abs() <= 3.01 * HALF[torch.float32] * want.abs()).all()
    _check_logprobs(lp, logits, tokens, 5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _answer(i8, lp, hidden, weight, sw, tokens)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    inputs = torch.zeros_like(hidden)
    with torch.cuda.graph(graph):
        captured = _answer(i8, lp, inputs, weight, sw, tokens)
    inputs.copy_(hidden)
    graph.replay()
    torch.cuda.synchronize()
    as_bits = lambda t: t.view(torch.int64) if t.dtype == torch.uint64 else t
    for a, b, c in zip(first, again, captured):
        assert torch.equal(as_bits(a), as_bits(b)) and torch.equal(as_bits(a), as_bits(c))


@gpu
def test_two_streams_at_once(i8, lp):
    """Calls on two streams share nothing, operands that have to be copied first among them."""
    g = torch.Generator().manual_seed(4)
    streams = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for j in range(2):
        A, B = _rand8(g, 120 + j, 1001).cuda(), _weight(g, 1001, 515 + j, ("kn", "nk")[j], 0)
        x = torch.randn(70, 5003 + j, generator=g).cuda()
        t = torch.randint(0, 5003, (70,), generator=g).cuda()
        work.append((A, B, x, t))
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(6):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                A, B, x, t = work[j]
                results[j].append((i8.int8_matmul(A, B), i8.int8_quantize_rows(x)[0], lp.token_logprobs(x, t, top=7)))
    torch.cuda.synchronize()
    for j in range(2):
        A, B, x, t = work[j]
        S, q = _sums_64(A, B), _quantize_64(x)[0]
        for y, qq, out in results[j]:
            assert torch.equal(y.cpu().long(), S) and torch.equal(qq.cpu(), q)
            assert all(torch.equal(a, b) for a, b in zip(out, results[j][0][2]))
        _check_logprobs(lp, x, t, 7)


@gpu
def test_pairs_beside_clusters(i8):
    """A product of pairs of blocks and one whose terms are shared by clusters, small enough to lie on the same SMs, on two
    streams at once, many times: neither waits for tensor memory that the other holds while it waits."""
    g = torch.Generator().manual_seed(12)
    streams = [torch.cuda.Stream() for _ in range(2)]
    work = [(_rand8(g, 32, 1024).cuda(), _weight(g, 1024, 11008, "nk", 0)), (_rand8(g, 16, 4096).cuda(), _weight(g, 4096, 1024, "nk", 0))]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(60):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                results[j].append(i8.int8_matmul(*work[j]))
    torch.cuda.synchronize()
    i8.check_async_errors()
    for (A, B), ys in zip(work, results):
        S = _sums_64(A, B)
        assert all(torch.equal(y.cpu().long(), S) for y in ys)


@gpu
def test_captured_streams_that_join(i8, lp):
    """A captured product whose operands are quantised on two streams that join, one of them from a copied tensor."""
    g = torch.Generator().manual_seed(13)
    x, y = torch.zeros(40, 512, device="cuda"), torch.zeros(300, 512, device="cuda")
    host = torch.zeros(300, 512).pin_memory()
    tokens = torch.zeros(40, dtype=torch.int64, device="cuda")

    def step():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y.copy_(host, non_blocking=True)
            wq, ws = i8.int8_quantize_rows(y)
        q, s = i8.int8_quantize_rows(x)
        torch.cuda.current_stream().wait_stream(side)
        logits = i8.int8_matmul(q, wq.t(), s, ws, dtype=torch.float32)
        return (q, wq, i8.int8_matmul(q, wq.t()), logits) + tuple(lp.token_logprobs(logits, tokens, top=3))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, wq, sums, logits, *_ = out = step()
    for _ in range(3):
        x.copy_(torch.randn(40, 512, generator=g))
        host.copy_(torch.randn(300, 512, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q.cpu(), _quantize_64(x)[0]) and torch.equal(wq.cpu(), _quantize_64(host)[0])
        assert torch.equal(sums.cpu().long(), _sums_64(q, wq.t()))
        assert all(torch.equal(a, b) for a, b in zip(out[4:], lp.token_logprobs(logits, tokens, top=3)))


@gpu
def test_two_graphs_of_one_product(i8):
    """Two captured products, of operands that have to be copied, replayed in turn and at once, keep their own copies."""
    g = torch.Generator().manual_seed(6)
    A = [_rand8(g, 33, 515).cuda() for _ in range(2)]
    B = [_weight(g, 515, 301, "kn", 0) for _ in range(2)]
    graphs, outs = [], []
    for j in range(2):
        i8.int8_matmul(A[j], B[j])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(i8.int8_matmul(A[j], B[j]))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for _ in range(3):
        graphs[0].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(outs[j].cpu().long(), _sums_64(A[j], B[j]))
            A[j].copy_(_rand8(g, 33, 515))


@gpu
def test_offsets_past_32_bits(i8, lp):
    """Matrices of more than 2^32 entries, looked at in their first and last rows."""
    x = torch.zeros(70000, 65536, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(9)
    ends = [0, 1, 65535, 65536, 69998, 69999]
    x[ends] = torch.randn(len(ends), 65536, generator=g, device="cuda").bfloat16()
    q, s = i8.int8_quantize_rows(x)
    wq, ws = _quantize_64(x[ends])
    assert torch.equal(q[ends].cpu(), wq) and torch.equal(s[ends].cpu(), ws) and int(q.count_nonzero(1).sum()) == int((wq != 0).sum())
    tokens = torch.arange(70000, device="cuda") % 65536
    out = lp.token_logprobs(x, tokens, top=3)
    part = lp.token_logprobs(x[ends].contiguous(), tokens[ends].contiguous(), top=3)
    assert all(torch.equal(a[ends], b) for a, b in zip(out, part))
    assert torch.equal(out.top_token[2], torch.tensor([0, 1, 2], device="cuda"))
    del x, q, out
    A = torch.randint(-128, 128, (140000, 64), generator=g, device="cuda", dtype=torch.int8)
    B = torch.randint(-128, 128, (64, 32768), generator=g, device="cuda", dtype=torch.int8)
    y = i8.int8_matmul(A, B)
    ends = [0, 65535, 65536, 131071, 131072, 139999]
    assert torch.equal(y[ends].cpu().long(), _sums_64(A[ends], B))


@gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_other_device_than_the_current_one(i8, lp):
    g = torch.Generator().manual_seed(4)
    with torch.cuda.device(0):
        x = torch.randn(9, 300, generator=g).to("cuda:1")
        q, s = i8.int8_quantize_rows(x)
        y = i8.int8_matmul(q, q.t())
        out = lp.token_logprobs(x, torch.zeros(9, dtype=torch.int64, device="cuda:1"), top=2)
        assert q.device == y.device == out.entropy.device == x.device and torch.cuda.current_device() == 0
        assert torch.equal(y.cpu().long(), _sums_64(q, q.t()))
        with pytest.raises(RuntimeError, match="different devices"):
            i8.int8_matmul(q, q.t().to("cuda:0"))


@gpu
def test_no_wait_expired(i8):
    i8.check_async_errors()


@gpu
def test_quantised_head_workload():
    """The review of answered tokens at a small size: the committed witness is that of the field product."""
    from verinf_b200 import cuda_primitives as cp, int8, workloads as w
    dev = torch.device("cuda:0")
    out = w.quantised_head(dev, seq=40, d=256, vocab=1000, seed=3)
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    hidden = torch.randn(40, 256, device=dev, generator=g).to(torch.bfloat16)
    weight, _ = int8.int8_quantize_rows(torch.randn(1000, 256, device=dev, generator=g) * (2.5 / 16))
    q, _ = int8.int8_quantize_rows(hidden)
    lift = lambda t: w._signed_to_field(t.to(torch.int64)).contiguous()
    rows = w._pack_rows(cp.gl_matmul(lift(q), lift(weight.t().contiguous())).reshape(-1))
    root, _, _ = cp.commit_rows(rows, w.K_DEG, w.N_LIG, master_seed=torch.arange(32, dtype=torch.uint8, device=dev))
    assert bytes(root.cpu().tolist()).hex() == out["root"]
    assert 0 < out["mean_entropy_bits"] < math.log2(1000) and out["mean_bits"] > 0


@gpu
def test_errors_are_asked_for_behind_every_stream(i8):
    """A product on a side stream that is still waiting to run has ended when its errors have been asked for."""
    g = torch.Generator().manual_seed(14)
    A, B = _rand8(g, 32, 1024).cuda(), _weight(g, 1024, 512, "nk", 0)
    i8.int8_matmul(A, B)
    side, ended = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)              # about a tenth of a second
        y = i8.int8_matmul(A, B)
        ended.record()
    assert not ended.query()
    i8.check_async_errors()
    assert ended.query()
    assert torch.equal(y.cpu().long(), _sums_64(A, B))


@gpu
@pytest.mark.parametrize("temperature", [1.0, 2.5, 1000.0, 1e6])
def test_logprobs_of_values_far_apart(lp, temperature):
    """fp32 values whose difference is beyond fp32, while that over the temperature is not: likely and unlikely tokens, short rows and
    rows of a cluster."""
    most = torch.finfo(torch.float32).max
    for vocab in (5, 70001):
        x = torch.full((6, vocab), -math.inf)
        x[:, :5] = torch.tensor([[most, -most, -most / 2, 0.0, 1.0], [-most, most, most, -0.75 * most, -math.inf], [-most] * 5,
                                 [-most, 3.0, 2.5, 2.0, -math.inf], [2e38, -2e38, -1.5e38, 1.5e38, 1.9e38],
                                 [-most, -most / 2, -math.inf, -math.inf, -math.inf]])
        tokens = torch.tensor([1, 0, 3, 0, 1, 0])
        out = lp.token_logprobs(x.cuda(), tokens.cuda(), top=5, temperature=temperature)
        want = _logprobs_64(x, tokens, 5, temperature)
        # of ln p: the difference, 1 / T, their product and the difference with the logarithm of the sum, half a step each, and what
        # these four make together; the sum itself as in _check_logprobs, its constant rounded too
        u = HALF[torch.float32]
        rel = (5 * 24 + 4 + vocab / 256 + 64) * u
        assert torch.equal(out.top_token.cpu(), want[3])
        for got, w in ((out.logprob, want[0]), (out.top_logprob, want[2])):
            assert _near(got, w, rel + u * (8 * want[4].reshape([-1] + [1] * (w.dim() - 1)) + 5 * torch.nan_to_num(w, 0, 0, 0).abs()))
        assert _near(out.entropy, want[1], rel * (1 + 2 * want[5]) + 8 * u * (want[4] + want[5]))


def test_import_without_torchs_short_calls():
    """A torch that lacks the calls which the entry points prefer has the public ones, and the package imports."""
    prog = """
import torch
hidden = []
for place, name in ((torch._C, "_cuda_getDevice"), (torch._C, "_cuda_getCurrentRawStream"), (torch._C._dynamo.guards, "_empty_strided_cuda")):
    if hasattr(place, name):
        hidden.append((place, name, getattr(place, name)))
        delattr(place, name)
from verinf_b200 import _lib, int8, logprobs
for place, name, call in hidden:                 # the public calls may use them
    assert call not in (_lib.current_device, _lib.raw_stream, _lib.empty_strided)
    setattr(place, name, call)
try:
    int8.int8_quantize_rows(torch.zeros(2, 3))
except RuntimeError as e:
    assert "CUDA" in str(e)
if torch.cuda.is_available():
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert _lib.raw_stream(0) == side.cuda_stream and _lib.current_device() == 0
        x = torch.tensor([[1.0, -2.0]], device="cuda")
        q, s = int8.int8_quantize_rows(x)
        assert q.tolist() == [[64, -127]]
        assert int8.int8_matmul(q, q.t()).item() == 64 * 64 + 127 * 127
        assert logprobs.token_logprobs(x, torch.tensor([0], device="cuda"), top=1).top_token.item() == 0
print("imported")
"""
    root = Path(__file__).resolve().parents[1]
    out = subprocess.run([sys.executable, "-c", prog], cwd=root, capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and out.stdout.strip() == "imported", out.stderr[-2000:]


@gpu
def test_torchs_public_calls_do_as_well():
    """The same on the GPU: the kernels run on the current stream that the public calls name."""
    test_import_without_torchs_short_calls()


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("vocab", [3, 2999])
def test_logprobs_the_token_comes_before_the_row(lp, dtype, vocab):
    """No token and a token outside the vocabulary beside rows with a NaN, with +inf, of -inf alone and ordinary ones; entropy says
    which rows are valid."""
    rows = torch.zeros(4, vocab)
    rows[0, vocab - 1], rows[1, 0], rows[2] = math.nan, math.inf, -math.inf
    tokens = torch.tensor([-1, -(1 << 62), vocab, (1 << 40) + 1, 1])
    out = lp.token_logprobs(rows.repeat(5, 1).to(dtype).cuda(), tokens.repeat_interleave(4).cuda(), top=2)
    logprob, entropy = out.logprob.cpu().view(5, 4), out.entropy.cpu().view(5, 4)
    # equal entries: the sum, its logarithm and the difference, counted as in _check_logprobs
    tol = (4 + vocab / 256 + 64 + 12 * math.log(vocab)) * HALF[torch.float32]
    assert (logprob[:2] == 0).all() and torch.isnan(logprob[2:4]).all()
    assert torch.isnan(logprob[4, :2]).all() and logprob[4, 2] == -math.inf and abs(logprob[4, 3] + math.log(vocab)) < tol
    assert torch.isnan(entropy[:, :2]).all() and (entropy[:, 2] == 0).all() and ((entropy[:, 3] - math.log(vocab)).abs() < tol).all()
    lists, ids = out.top_logprob.cpu().view(5, 4, 2), out.top_token.cpu().view(5, 4, 2)
    assert torch.isnan(lists[:, :2]).all() and (lists[:, 2] == -math.inf).all() and (ids[:, :3] == -1).all()
    assert (ids[:, 3] == torch.tensor([0, 1])).all()


# ---- many rows: a block of 64 or 128 threads a row -------------------------------------------------------------------------
def _logprobs_rows_64(x, tokens, top, temperature):
    """What _logprobs_64 gives, for all rows at once (where x is)."""
    x = x.double() + 0.0                                             # -0 counts as 0
    rows, vocab = x.shape
    bad, none = (torch.isnan(x) | (x == math.inf)).any(1), (x == -math.inf).all(1)
    x = torch.where(bad[:, None], 0.0, x)
    z = (x - torch.where(none[:, None], 0.0, x.amax(1, keepdim=True))) / temperature
    e = z.exp()
    s = torch.where(none, 1.0, e.sum(1))
    log_z, width = s.log(), -(e * torch.where(e > 0, z, 0.0)).sum(1) / s
    ent = torch.where(bad, math.nan, log_z + width)
    lp = z.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0] - log_z
    lp = torch.where(tokens < 0, 0.0, torch.where((tokens >= vocab) | bad, math.nan, lp))
    tt = x.sort(dim=1, descending=True, stable=True)[1][:, :top]
    tl = z.gather(1, tt) - log_z[:, None]
    tt = torch.where((tl == -math.inf) | bad[:, None], -1, tt)
    tl = torch.where(bad[:, None], math.nan, tl)
    short = top - tt.size(1)                                         # fewer entries than the list holds
    if short > 0:
        tt = torch.cat([tt, tt.new_full((rows, short), -1)], 1)
        tl = torch.cat([tl, torch.where(bad[:, None], math.nan, -math.inf).double().expand(rows, short)], 1)
    return lp, ent, tl, tt, log_z, width


def _check_many_rows(lp_mod, x, tokens, tops, temperature):
    lp, ent, tl, tt, log_z, width = _logprobs_rows_64(x, tokens, 32, temperature)
    # as in _check_logprobs, with a rounded 1 / T (two half steps more of a difference) and the longest chain, that of 64 threads
    u = HALF[torch.float32]
    rel = (5 * 24 + 4 + x.size(1) / 64 + 64) * u
    t = lambda want, steps: (rel + u * (8 * log_z.reshape([-1] + [1] * (want.dim() - 1)) + steps * torch.nan_to_num(want, 0, 0, 0).abs())).cpu()
    for top in tops:
        out = lp_mod.token_logprobs(x, tokens, top=top, temperature=temperature)
        assert torch.equal(out.top_token, tt[:, :top])
        assert _near(out.logprob, lp.cpu(), t(lp, 6))
        assert _near(out.entropy, ent.cpu(), (rel * (1 + 2 * width) + 8 * u * (log_z + width)).cpu())
        assert _near(out.top_logprob, tl[:, :top].cpu(), t(tl[:, :top], 6))


@gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,vocab,offset,pitch,masked,temperature",
                         [(512, 1, 0, 1, "no", 1.0), (513, 31, 0, 31, "no", 0.7), (2000, 300, 1, 305, "inf", 1.0), (515, 4001, 0, 4001, "lowest", 1.5),
                          (700, 4096, 0, 4096, "no", 1.0), (600, 8200, 3, 8209, "inf", 0.7), (1100, 9001, 0, 9008, "lowest", 1.0),
                          (520, 33000, 0, 33000, "no", 1.0), (516, 32001, 5, 32011, "inf", 1.3)])
def test_logprobs_many_rows(lp, dtype, rows, vocab, offset, pitch, masked, temperature):
    """Every row against 64 bits, lists on both sides of the change of the number of groups; rows that are masked in part or whole,
    hold fewer entries than the list, equal ones, a NaN or infinity, or crowd their large entries in a few threads' shares."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = torch.randn(rows, vocab, device="cuda", generator=g) * 3
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 12), device="cuda", generator=g), torch.rand(rows, 12, device="cuda", generator=g) * 9)
    low = torch.finfo(dtype).min if masked == "lowest" else -math.inf
    if masked != "no":
        x[torch.rand(rows, vocab, device="cuda", generator=g) < 0.4] = low
    i = torch.arange(vocab, device="cuda")
    x[3] = low
    x[4, vocab // 2] = math.nan
    x[5, vocab - 1] = math.inf
    x[6] = 1.25
    x[7] = torch.where(i % 2 == 0, 0.0, -0.0)
    x[8] = torch.where(i % max(1, vocab // 7) == 0, 2.0 + 0.25 * (i % 5), -math.inf)
    x[9] = torch.linspace(-9, 9, vocab, device="cuda")
    x[10] = torch.linspace(9, -9, vocab, device="cuda")
    for r, step in ((11, 512), (12, 1024), (13, 2048)):
        x[r] = torch.where(i % step < 16, (i // step).float() / 64 + i % 16, -math.inf)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    tokens[20], tokens[21], tokens[rows - 1] = -1, vocab, 0
    buf = torch.full((rows, pitch + offset), 100.0, dtype=dtype, device="cuda")       # behind the vocabulary: not part of it
    view = buf[:, offset:offset + vocab]
    view.copy_(x.to(dtype))
    _check_many_rows(lp, view, tokens, (0, 1, 5, 16, 17, 32), temperature)


# ---- operands that are copied first ------------------------------------------------------------------------------------
def _scratch_bytes(i8, lib, A, B):
    """What int8_matmul asks for these operands."""
    m, k, lda = i8.matrix(A, "", "A", (torch.int8,))
    B, k, n, by_channel, ldb = i8._weight(B, "")
    return lib.LIB.vi_int8_matmul_scratch_bytes(A.data_ptr(), lda, B.data_ptr(), ldb, by_channel, m, k, n)


def _laid(g, rows, cols, offset, pitch):
    """rows x cols int8 on the GPU whose first entry is `offset` bytes behind the 16-byte grid, rows `pitch` bytes apart."""
    buf = _rand8(g, rows * pitch + 32).cuda()
    assert buf.data_ptr() % 16 == 0 and pitch >= cols
    return torch.as_strided(buf, (rows, cols), (pitch, 1), offset)


def _on_grid(n):
    return (n + 15) // 16 * 16


@gpu
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("off", ["A", "B", "both"])
@pytest.mark.parametrize("m,k,n", [(120, 4001, 1003), (300, 2001, 1500), (700, 3001, 2001), (256, 1203, 2001)])
def test_matmul_copied_operands(i8, lib, layout, off, m, k, n):
    """One operand or both off the 16-byte grid, by their rows' distance or their first byte, at sizes where they are copied; then
    clusters, single blocks and pairs make the product.  On the grid, nothing is asked for."""
    g = torch.Generator().manual_seed(m + k + n)
    rows, cols = (k, n) if layout == "kn" else (n, k)

    def operands(offset, a_pitch, b_pitch):
        b = _laid(g, rows, cols, offset if off != "A" else 0, b_pitch if off != "A" else _on_grid(cols))
        return _laid(g, m, k, offset if off != "B" else 0, a_pitch if off != "B" else _on_grid(k)), b if layout == "kn" else b.t()

    for offset, a_pitch, b_pitch in [(0, k, cols), (1, _on_grid(k), _on_grid(cols)), (15, _on_grid(k), _on_grid(cols) + 16), (7, k + 2, cols + 6)]:
        A, B = operands(offset, a_pitch, b_pitch)
        assert _scratch_bytes(i8, lib, A, B) >= (m * k if off != "B" else 0) + (k * n if off != "A" else 0)
        _check_matmul(i8, A, B, [torch.int32, torch.uint64, torch.bfloat16], g, out_pad=3)
    A, B = operands(0, _on_grid(k), _on_grid(cols))
    assert _scratch_bytes(i8, lib, A, B) == 0


@gpu
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("m,k,n", [(1, 515, 1001), (5, 515, 1001), (31, 515, 1001), (17, 515, 3001), (700, 515, 301)])
def test_matmul_copied_tokens_alone(i8, lib, layout, m, k, n):
    """Few tokens off the grid beside a weight on it: copied, and the product made by single blocks."""
    g = torch.Generator().manual_seed(m + k + n)
    rows, cols = (k, n) if layout == "kn" else (n, k)
    for offset, pitch in [(1, _on_grid(k)), (8, k), (15, k + 10)]:
        A, b = _laid(g, m, k, offset, pitch), _laid(g, rows, cols, 0, _on_grid(cols))
        B = b if layout == "kn" else b.t()
        assert _scratch_bytes(i8, lib, A, B) == m * _on_grid(k)
        _check_matmul(i8, A, B, g=g)


@gpu
def test_two_streams_and_two_graphs_with_copies(i8, lib):
    """Products whose operands are copied first, on two streams at once and in two captured graphs replayed in turn and at once: each
    call has copies of its own."""
    g = torch.Generator().manual_seed(16)
    shapes = [(300, 2001, 1501, "kn"), (120, 4001, 1003, "nk")]
    A = [_rand8(g, m, k).cuda() for m, k, n, _ in shapes]
    B = [_weight(g, k, n, layout, 0) for m, k, n, layout in shapes]
    for a, b in zip(A, B):
        assert _scratch_bytes(i8, lib, a, b) >= a.numel() + b.numel()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(8):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                results[j].append(i8.int8_matmul(A[j], B[j]))
                results[j].append(i8.int8_matmul(A[j].neg(), B[j]))       # another operand into the room that is free again
    torch.cuda.synchronize()
    for j in range(2):
        S, N = _sums_64(A[j], B[j]), _sums_64(A[j].neg(), B[j])
        assert all(torch.equal(y.cpu().long(), (S, N)[i % 2]) for i, y in enumerate(results[j]))
    graphs, outs = [], []
    for j in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(i8.int8_matmul(A[j], B[j]))
        graphs.append(graph)
    for _ in range(3):
        graphs[0].replay()
        streams[0].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[0]):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(outs[j].cpu().long(), _sums_64(A[j], B[j]))
            A[j].copy_(_rand8(g, *A[j].shape))
            B[j].copy_(_rand8(g, *B[j].shape))


@gpu
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("m,k,n", [(1001, 1200, 20000), (2001, 304, 9008), (4095, 128, 5008), (515, 2064, 30000), (777, 1040, 32000)])
def test_matmul_many_tiles_a_pair(i8, layout, m, k, n):
    """More tiles than three rounds of 74 pairs of blocks even at the largest tile of 256 x 256, and numbers of slices that no ring of 6, 7 or 8
    stages divides evenly: both accumulators, the wait for one that is written out, and a ring that goes on from tile to tile.  The whole
    result, with remainders of every size."""
    assert -(-m // 256) * -(-n // 256) > 3 * 74
    g = torch.Generator().manual_seed(m + k + n)
    A, B = _rand8(g, m, k).cuda(), _weight(g, k, n, layout, 0)
    S = (A.double() @ B.double()).to(torch.int64)                    # whole in 64 bits
    assert torch.equal(i8.int8_matmul(A, B), S.to(torch.int32))
    lifted = torch.where(S < 0, S + (P - (1 << 64)), S)
    assert torch.equal(i8.int8_matmul(A, B, dtype=torch.uint64).view(torch.int64), lifted)
    sa, sb = torch.rand(m, generator=g).cuda() + 0.01, torch.rand(n, generator=g).cuda() * 1e-3
    want = S.double() * sa.double()[:, None] * sb.double()
    for dtype in (torch.float32, torch.bfloat16):
        y = i8.int8_matmul(A, B, sa, sb, dtype=dtype).double()
        # roundings: the sum to fp32, two products, the output type where it is shorter
        tol = want.abs() * (3 * HALF[torch.float32] + (HALF[dtype] if dtype != torch.float32 else 0)) * 1.001 + 1e-37
        assert ((y - want).abs() <= tol).all()
    i8.check_async_errors()


@gpu
def test_first_calls_inside_a_capture():
    """In a process that has called nothing before, the first call of each operator may be a captured one: kernels, their shared memory
    and tensor maps are set up on the way."""
    prog = """
import torch
from verinf_b200 import int8, logprobs
x = torch.zeros(300, 512, device="cuda")
w = torch.zeros(1024, 512, device="cuda")
a = torch.zeros(40, 515, dtype=torch.int8, device="cuda")
b = torch.zeros(515, 301, dtype=torch.int8, device="cuda")
c = torch.zeros(700, 2001, dtype=torch.int8, device="cuda")
d = torch.zeros(2001, 1500, dtype=torch.int8, device="cuda")
tokens = torch.zeros(300, dtype=torch.int64, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q, s = int8.int8_quantize_rows(x)
    wq, ws = int8.int8_quantize_rows(w)
    logits = int8.int8_matmul(q, wq.t(), s, ws, dtype=torch.float32)
    one = int8.int8_matmul(q[:1], wq.t())
    shifted, copied = int8.int8_matmul(a, b), int8.int8_matmul(c, d)
    out = logprobs.token_logprobs(logits, tokens, top=3)
for t in (x, w):
    t.normal_()
for t in (a, b, c, d):
    t.random_(-128, 128)
graph.replay()
torch.cuda.synchronize()
sums = lambda p, r: (p.double() @ r.double()).to(torch.int32)
assert torch.equal(one, sums(q[:1], wq.t())) and torch.equal(shifted, sums(a, b)) and torch.equal(copied, sums(c, d))
assert torch.equal(logits, sums(q, wq.t()).float() * s[:, None] * ws)
again = logprobs.token_logprobs(logits, tokens, top=3)
assert all(torch.equal(p, r) for p, r in zip(out, again))
assert torch.equal(q, int8.int8_quantize_rows(x)[0]) and int(q.abs().max()) == 127
int8.check_async_errors()
print("captured")
"""
    root = Path(__file__).resolve().parents[1]
    out = subprocess.run([sys.executable, "-c", prog], cwd=root, capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and out.stdout.strip() == "captured", out.stderr[-2000:]


@gpu
def test_two_threads_at_once(i8, lp):
    """Calls from two threads, each on a stream of its own, products that are copied and shifted among them, and errors asked for
    meanwhile."""
    import threading
    g = torch.Generator().manual_seed(18)
    shapes = [[(300, 2001, 1501), (33, 515, 301), (1, 4096, 512)], [(120, 4001, 1003), (333, 1001, 515), (513, 640, 272)]]
    work = [[(_rand8(g, m, k).cuda(), _rand8(g, k, n).cuda()) for m, k, n in s] for s in shapes]
    rows = [torch.randn(70, 5003, generator=g).cuda() for _ in range(2)]
    tokens = torch.arange(70, device="cuda")
    torch.cuda.synchronize()
    results, failures = [[], []], []

    def run(j):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(12):
                    for A, B in work[j]:
                        results[j].append(i8.int8_matmul(A, B))
                    results[j].append((i8.int8_quantize_rows(rows[j])[0], lp.token_logprobs(rows[j], tokens, top=7)))
                    if i % 4 == j:
                        i8.check_async_errors()
                torch.cuda.current_stream().synchronize()
        except BaseException as e:
            failures.append(e)

    threads = [threading.Thread(target=run, args=(j,)) for j in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for j in range(2):
        sums = [_sums_64(A, B) for A, B in work[j]]
        q, out = _quantize_64(rows[j])[0], lp.token_logprobs(rows[j], tokens, top=7)
        for i, y in enumerate(results[j]):
            if i % 4 < 3:
                assert torch.equal(y.cpu().long(), sums[i % 4])
            else:
                assert torch.equal(y[0].cpu(), q) and all(torch.equal(a, b) for a, b in zip(y[1], out))

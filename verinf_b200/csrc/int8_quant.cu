// Rows of activations (or of a weight, one row an output channel) to int8 with one scale a row.
//
// a_r = max_j |x_rj|, scale_r = a_r / 127, q_rj = the whole number nearest to 127 x_rj / a_r, ties to even.  The nearest
// whole number is that of the exact quotient: v = x (127 / a) is off by a few units of 2^-23 v, so only where v lies within
// 10^-4 of a border between two whole numbers is the remainder 127 x - q a formed (exactly, see round_quotient) and
// compared with a / 2.  A result that does not depend on how the quotient was rounded is what a witness needs: another
// program that quantises the same activations commits to the same whole numbers.
//
// Bound by HBM: a row is read once and stays in the registers of its block (up to 64 KB of row), the maximum meets in shared
// memory, and the row leaves as bytes.  A longer row is read twice, the second time from L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/verinf_b200.h"
#include "common.cuh"

namespace {

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// VEC consecutive elements of a row
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

struct RowScale {
    float p, a, inv;     // x p and a = (row maximum) p without rounding, p a power of two; 127 / a
};

// p brings the maximum to [1, 2) (a subnormal one to [2^-23, 1)), so that neither 127 x nor 127 / a can overflow.
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23);                                    // biased exponent, 0 for a subnormal maximum
    RowScale s;
    s.p = e >= 254 ? __uint_as_float(0x00400000u)                            // 2^-127
                   : __uint_as_float((uint32_t)(254 - (e ? e : 1)) << 23);   // 2^(127 - e)
    s.a = __uint_as_float(amax_bits) * s.p;
    s.inv = __fdiv_rn(127.0f, s.a);
    return s;
}

// Nearest whole number to 127 x / a, ties to even; |x| <= a.
__device__ __forceinline__ int round_quotient(float x, const RowScale& s) {
    const float magic = 12582912.0f;                                         // 1.5 * 2^23: adding it rounds to a whole number
    const float xs = x * s.p, v = xs * s.inv;
    const float t = v + magic;
    float q = t - magic;
    if (fabsf(v - q) > 0.4999f) {
        // hi + lo = 127 xs exactly.  q a differs from hi by about a / 2 < 1, both are multiples of 2^-24 (for a subnormal
        // maximum of 2^-23), so the difference has at most 24 bits and the fused multiply-add is exact.
        const float hi = 127.0f * xs, lo = __fmaf_rn(127.0f, xs, -hi);
        const float rem = __fmaf_rn(-q, s.a, hi);
        const float side = rem < 0.0f ? -1.0f : 1.0f;
        const float over = (fabsf(rem) - 0.5f * s.a) + lo * side;            // sign: beyond, on, or before the border
        if (over > 0.0f || (over == 0.0f && ((int)q & 1))) q += side;
    }
    return (int)q;
}

constexpr int QT_CACHED = 4;      // packs of a row that a thread keeps

// One block a row.  VEC elements are loaded at a time (16 bytes where every row starts on 16 bytes, else one element).
template <typename T, int VEC>
__global__ void __launch_bounds__(1024) k_int8_quantize(const T* __restrict__ x, int64_t x_stride, int64_t k, int8_t* __restrict__ q,
                                                        int64_t q_stride, float* __restrict__ scale, int q_vec) {
    using P = Pack<T, VEC>;
    constexpr int KEEP = VEC == 1 ? 4 * QT_CACHED : QT_CACHED;
    __shared__ uint32_t part[32];
    const int64_t r = blockIdx.x;
    const T* xr = x + r * x_stride;
    int8_t* qr = q + r * q_stride;
    const int tid = threadIdx.x, nt = blockDim.x;
    const int64_t nvec = k / VEC;                  // whole packs; the last k % VEC elements are taken one by one
    P keep[KEEP];
    uint32_t amax = 0;                             // bits of |x|: ordered as numbers, infinity and NaN above all
    auto take = [&](T e) { amax = max(amax, __float_as_uint(as_float(e)) & 0x7FFFFFFFu); };
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int64_t i = tid + (int64_t)j * nt;
        if (i < nvec) keep[j] = reinterpret_cast<const P*>(xr)[i];
    }
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        if (tid + (int64_t)j * nt < nvec) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) take(keep[j].v[e]);
        }
    }
    for (int64_t i = tid + (int64_t)KEEP * nt; i < nvec; i += nt) {
        const P p = reinterpret_cast<const P*>(xr)[i];
#pragma unroll
        for (int e = 0; e < VEC; ++e) take(p.v[e]);
    }
    for (int64_t i = nvec * VEC + tid; i < k; i += nt) take(xr[i]);
    amax = __reduce_max_sync(0xFFFFFFFFu, amax);
    if ((tid & 31) == 0) part[tid >> 5] = amax;
    __syncthreads();
    amax = __reduce_max_sync(0xFFFFFFFFu, (tid & 31) < (nt >> 5) ? part[tid & 31] : 0u);

    const bool bad = amax >= 0x7F800000u, zero = amax == 0;
    if (tid == 0) scale[r] = bad ? __uint_as_float(0x7FC00000u) : __fdiv_rn(__uint_as_float(amax), 127.0f);
    const RowScale s = row_scale(bad || zero ? 0x3F800000u : amax);
    auto whole = [&](T e) { return bad ? 0 : round_quotient(as_float(e), s); };
    auto put = [&](int64_t i, const P& p) {
        Pack<int8_t, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = (int8_t)whole(p.v[e]);
        if (q_vec) reinterpret_cast<Pack<int8_t, VEC>*>(qr)[i] = o;
        else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) qr[i * VEC + e] = o.v[e];
        }
    };
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int64_t i = tid + (int64_t)j * nt;
        if (i < nvec) put(i, keep[j]);
    }
    for (int64_t i = tid + (int64_t)KEEP * nt; i < nvec; i += nt) put(i, reinterpret_cast<const P*>(xr)[i]);
    for (int64_t i = nvec * VEC + tid; i < k; i += nt) qr[i] = (int8_t)whole(xr[i]);
}

template <typename T>
int launch(const void* x, int64_t m, int64_t k, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, cudaStream_t st) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const bool wide = ((uintptr_t)x) % 16 == 0 && (x_stride * (int64_t)sizeof(T)) % 16 == 0;
    const int64_t packs = wide ? (k + VEC - 1) / VEC : k;
    const int keep = wide ? QT_CACHED : 4 * QT_CACHED;
    int64_t nt = (packs + keep - 1) / keep;
    nt = nt < 32 ? 32 : nt > 1024 ? 1024 : (nt + 31) / 32 * 32;
    if (wide) {
        const int q_vec = ((uintptr_t)q) % VEC == 0 && q_stride % VEC == 0;
        k_int8_quantize<T, VEC><<<(unsigned)m, (unsigned)nt, 0, st>>>((const T*)x, x_stride, k, q, q_stride, scale, q_vec);
    } else {
        k_int8_quantize<T, 1><<<(unsigned)m, (unsigned)nt, 0, st>>>((const T*)x, x_stride, k, q, q_stride, scale, 1);
    }
    return vi::check_launch("k_int8_quantize");
}

}  // namespace

extern "C" int vi_int8_quantize_rows(const void* x, int dtype, int64_t m, int64_t k, int64_t x_stride, int8_t* q, int64_t q_stride,
                                     float* scale, void* stream) {
    VI_REQUIRE(dtype == VI_F32 || dtype == VI_F16 || dtype == VI_BF16, "int8_quantize_rows: dtype must be VI_F32, VI_F16 or VI_BF16");
    VI_REQUIRE(m >= 0 && k >= 0, "int8_quantize_rows: negative size");
    VI_REQUIRE(m <= 0x7FFFFFFF, "int8_quantize_rows: more than 2^31 - 1 rows");
    if (m == 0) return VI_OK;
    VI_REQUIRE(scale && ((uintptr_t)scale) % 4 == 0, "int8_quantize_rows: null or misaligned scale");
    VI_REQUIRE(k == 0 || (x && q), "int8_quantize_rows: null pointer");
    VI_REQUIRE(((uintptr_t)x) % (dtype == VI_F32 ? 4 : 2) == 0, "int8_quantize_rows: x is not aligned to its type");
    VI_REQUIRE(m == 1 || (x_stride >= 0 && q_stride >= k), "int8_quantize_rows: negative distance of rows, or output rows that overlap");
    cudaStream_t st = (cudaStream_t)stream;
    if (m == 1) { x_stride = 0; q_stride = 0; }
    if (dtype == VI_F32) return launch<float>(x, m, k, x_stride, q, q_stride, scale, st);
    if (dtype == VI_F16) return launch<__half>(x, m, k, x_stride, q, q_stride, scale, st);
    return launch<__nv_bfloat16>(x, m, k, x_stride, q, q_stride, scale, st);
}

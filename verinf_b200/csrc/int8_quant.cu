// Rows of activations (or of a weight, one row an output channel) to int8 with one scale a row.
//
// a_r = max_j |x_rj|, scale_r = a_r / 127, q_rj = the whole number nearest to 127 x_rj / a_r, ties to even: nearest to the
// exact quotient, however it was computed.  A result that does not depend on roundings is what a witness needs: another
// program that quantises the same activations commits to the same whole numbers.
//
// Bound by HBM: a row is read once and stays in the registers of its block (up to 128 KB of row), the maximum meets in shared
// memory, and the row leaves as bytes; a longer row is read twice, the second time from L2.  11008 x 4096 fp32 34 us (6.7 TB/s),
// bf16 21.7 us (6.2 TB/s); 1000 x 11008 bf16 7.0 us (4.7 TB/s: 192 threads of 64 registers, so five blocks an SM and 740 of the 1000 at
// once; the others follow as a short second wave, and load and store phases hardly overlap).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/verinf_b200.h"
#include "common.cuh"
#include "f32x2.cuh"
#include "launch.cuh"
#include "packs.cuh"

namespace {

using namespace vf2;

// The entries of a 16-byte pack as fp32 in pairs, and the bits of the largest |x|, which are ordered as the numbers are,
// infinity and NaN above all.
__device__ __forceinline__ uint32_t word(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
__device__ __forceinline__ uint32_t largest16(const uint4& w) {
    const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
    return max(m & 0xFFFFu, m >> 16);
}
__device__ __forceinline__ float2 halves(uint32_t w) {
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}
template <typename T> struct Entries;
template <> struct Entries<float> {
    using Raw = uint32_t;
    static __device__ __forceinline__ void pair(const uint4& w, int i, float& a, float& b) {
        a = __uint_as_float(word(w, 2 * i));
        b = __uint_as_float(word(w, 2 * i + 1));
    }
    static __device__ __forceinline__ uint32_t largest(const uint4& w) {
        return max(max(w.x & 0x7FFFFFFFu, w.y & 0x7FFFFFFFu), max(w.z & 0x7FFFFFFFu, w.w & 0x7FFFFFFFu));
    }
};
template <> struct Entries<__half> {
    using Raw = uint16_t;
    static __device__ __forceinline__ void pair(const uint4& w, int i, float& a, float& b) {
        const float2 f = halves(word(w, i));
        a = f.x;
        b = f.y;
    }
    static __device__ __forceinline__ uint32_t largest(const uint4& w) { return __float_as_uint(halves(largest16(w)).x); }
};
template <> struct Entries<__nv_bfloat16> {
    using Raw = uint16_t;
    static __device__ __forceinline__ void pair(const uint4& w, int i, float& a, float& b) {
        a = __uint_as_float(word(w, i) << 16);
        b = __uint_as_float(word(w, i) & 0xFFFF0000u);
    }
    static __device__ __forceinline__ uint32_t largest(const uint4& w) { return largest16(w) << 16; }
};

struct RowScale {
    float p127, a, inv;     // 127 p, a = (row maximum) p, 1 / a
};

// p = 2^j brings the maximum to [1, 2), a smaller one than 2^-119 to [2^-30, 1): neither 127 p nor 1 / a overflows, and 127 x p
// of a 16-bit type is exact (where it could underflow, 127 x / a rounds to 0 whatever its last bits are).
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    const int e = max((int)(amax_bits >> 23), 8);                            // biased exponent, 2^-119 at least
    const float p = e == 254 ? __uint_as_float(0x00400000u)                  // 2^-127
                             : __uint_as_float((uint32_t)(254 - e) << 23);   // 2^(127 - e)
    return {127.0f * p, __uint_as_float(amax_bits) * p, __fdiv_rn(1.0f, __uint_as_float(amax_bits) * p)};
}

constexpr float QT_MAGIC = 12582912.0f;      // 1.5 * 2^23: adding it rounds to a whole number, ties to even, which then stands in the low bits

// Whole numbers of the two entries of a pair; their low bytes count.
// 16-bit types: hi = 127 x p is exact, and v = hi (1 / a) off by at most 2^-23 of itself.  A quotient of significands of at
// most 11 bits that is on a border (n + 1/2, n < 127) has 8 bits, one that is not differs from every border by 2^-20 of itself
// or more.  So v is rounded to 21 bits (9 v - (9 v - v), the split of Veltkamp), which puts back onto the border what belongs
// there and moves nothing else across one, and then to a whole number.  Every pair of significands is a test.
__device__ __forceinline__ void whole_pair(float x0, float x1, const RowScale& s, uint32_t& q0, uint32_t& q1) {
    const uint64_t v = mul2(mul2(pack2(x0, x1), pack2(s.p127, s.p127)), pack2(s.inv, s.inv));
    const uint64_t v9 = mul2(v, pack2(9.0f, 9.0f)), minus = pack2(-1.0f, -1.0f);
    const uint64_t w = fma2(fma2(v, minus, v9), minus, v9);
    float a, b;
    unpack2(add2(w, pack2(QT_MAGIC, QT_MAGIC)), a, b);
    q0 = __float_as_uint(a);
    q1 = __float_as_uint(b);
}

template <typename T, int N>
__device__ __forceinline__ void whole_numbers(const uint4& w, const RowScale& s, uint32_t (&q)[N]) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        float a, b;
        Entries<T>::pair(w, e / 2, a, b);
        whole_pair(a, b, s, q[e], q[e + 1]);
    }
}
// fp32: t = hi (1 / a) rounded to a whole number is right unless the quotient is within 10^-4 of a border, which the size of
// the remainder hi - q a tells.  There 127 x p = hi + lo, and the remainder, at most about a / 2 < 1 and a multiple of 2^-24 (of
// 2^-31 and less than 2^-7 for a small maximum), is exact: the nearest whole number is the next one on its side if with lo it
// is beyond a / 2, or on it and q is odd.
template <>
__device__ __forceinline__ void whole_numbers<float, 4>(const uint4& w, const RowScale& s, uint32_t (&q)[4]) {
    float worst = 0.0f;
    const uint64_t p2 = pack2(s.p127, s.p127), inv2 = pack2(s.inv, s.inv), a2 = pack2(s.a, s.a), magic2 = pack2(QT_MAGIC, QT_MAGIC), minus = pack2(-1.0f, -1.0f);
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
        float a, b, r0, r1, t0, t1;
        Entries<float>::pair(w, e / 2, a, b);
        const uint64_t hi = mul2(pack2(a, b), p2), t = fma2(hi, inv2, magic2);
        unpack2(fma2(fma2(t, minus, magic2), a2, hi), r0, r1);
        unpack2(t, t0, t1);
        worst = fmaxf(worst, fmaxf(fabsf(r0), fabsf(r1)));
        q[e] = __float_as_uint(t0);
        q[e + 1] = __float_as_uint(t1);
    }
    if (worst > 0.4999f * s.a) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float y = __uint_as_float(word(w, e)), hi = y * s.p127, lo = __fmaf_rn(y, s.p127, -hi), t = __fmaf_rn(hi, s.inv, QT_MAGIC);
            const float rem = __fmaf_rn(QT_MAGIC - t, s.a, hi);
            const float over = (fabsf(rem) - 0.5f * s.a) + copysignf(1.0f, rem) * lo;      // beyond, on, or before the border
            if (over > 0.0f || (over == 0.0f && (q[e] & 1))) q[e] += rem < 0.0f ? -1 : 1;
        }
    }
}

__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The N low bytes of a pack's whole numbers to `to`, those in [lo, hi) of them.  The lanes of a warp hold packs side by side: if
// all are whole, their bytes leave in words on the grid of N bytes, off which `to` is by the same `off` for every lane: a lane
// takes the last `off` bytes of the lane before it in front of its own.
template <int N>
__device__ __forceinline__ void store(int8_t* to, const uint32_t (&q)[N], int lo, int hi) {
    const int off = (int)((uintptr_t)to % N), lane = threadIdx.x & 31;
    uint64_t w = bytes4(q[0], q[1], q[2], q[3]);
    if (N == 8) w |= (uint64_t)bytes4(q[4 % N], q[5 % N], q[6 % N], q[7 % N]) << 32;
    const bool all = __all_sync(0xFFFFFFFFu, lo == 0 && hi == N);
    if (all && off == 0) {
        if (N == 8) *reinterpret_cast<uint64_t*>(to) = w;
        else *reinterpret_cast<uint32_t*>(to) = (uint32_t)w;
    } else if (all) {
        const uint64_t before = __shfl_up_sync(0xFFFFFFFFu, w, 1);
        if (lane) {
            const uint64_t v = w << (8 * off) | before >> (8 * (N - off));
            if (N == 8) *reinterpret_cast<uint64_t*>(to - off) = v;
            else *reinterpret_cast<uint32_t*>(to - off) = (uint32_t)v;
        }
        if (lane == 0 || lane == 31) {               // the first lane's bytes before its next word, the last one's behind it
            const int from = lane ? N - off : 0, end = lane ? N : N - off;
            for (int e = from; e < end; ++e) to[e] = (int8_t)(uint8_t)(w >> (8 * e));
        }
    } else {
        for (int e = lo; e < hi; ++e) to[e] = (int8_t)(uint8_t)(w >> (8 * e));
    }
}

constexpr int QT_KEEP = 8;        // packs of a row that a thread keeps

// blockDim.x threads a row, blockDim.y rows a block (more than one only where a warp has a row).  ALIGNED: every row of x starts
// on 16 bytes and every row of q on N, so that only a row's last pack can be a part of one (that saves the tests of each pack:
// 11008 x 4096 fp32 40 -> 35 us).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(1024) k_int8_quantize(const T* __restrict__ x, int64_t x_stride, int64_t m, int64_t k, int8_t* __restrict__ q,
                                                        int64_t q_stride, float* __restrict__ scale) {
    using E = Entries<T>;
    constexpr int N = 16 / (int)sizeof(T);
    __shared__ uint32_t part[32];
    const int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    vi::await_inputs();
    if (r >= m) return;
    const vpk::Row<typename E::Raw> row(x + r * x_stride, k);
    int8_t* qr = q + r * q_stride;
    const int tid = threadIdx.x, nt = blockDim.x;
    const int64_t whole = k / N;                      // ALIGNED: packs of the row alone
    const bool last = ALIGNED && k % N && tid == nt - 1;
    uint4 keep[QT_KEEP];
    uint32_t amax = 0;
    if (ALIGNED) {
        const uint4* packs = reinterpret_cast<const uint4*>(x + r * x_stride);
#pragma unroll
        for (int j = 0; j < QT_KEEP; ++j)
            if (tid + j * nt < whole) keep[j] = __ldg(packs + tid + j * nt);
#pragma unroll
        for (int j = 0; j < QT_KEEP; ++j)
            if (tid + j * nt < whole) amax = max(amax, E::largest(keep[j]));
        for (int64_t i = tid + QT_KEEP * nt; i < whole; i += nt) amax = max(amax, E::largest(__ldg(packs + i)));
        if (last) amax = max(amax, E::largest(vpk::edge_pack(row.x, whole * N, k, 0)));
    } else {
#pragma unroll
        for (int j = 0; j < QT_KEEP; ++j) {
            keep[j] = {0, 0, 0, 0};
            if (tid + j * nt < row.count) keep[j] = row.load(tid + j * nt, 0);
        }
#pragma unroll
        for (int j = 0; j < QT_KEEP; ++j) amax = max(amax, E::largest(keep[j]));
        for (int64_t i = tid + QT_KEEP * nt; i < row.count; i += nt) amax = max(amax, E::largest(row.load(i, 0)));
    }
    vi::release_next();
    amax = __reduce_max_sync(0xFFFFFFFFu, amax);
    if (nt > 32) {
        if ((tid & 31) == 0) part[tid >> 5] = amax;
        __syncthreads();
        amax = __reduce_max_sync(0xFFFFFFFFu, (tid & 31) < nt >> 5 ? part[tid & 31] : 0u);
    }

    const bool bad = amax >= 0x7F800000u;
    if (tid == 0) scale[r] = bad ? __uint_as_float(0x7FC00000u) : __fdiv_rn(__uint_as_float(amax), 127.0f);
    if (bad || amax == 0) {
        for (int64_t i = tid; i < k; i += nt) qr[i] = 0;
        return;
    }
    const RowScale s = row_scale(amax);
    if (ALIGNED) {
        const uint4* packs = reinterpret_cast<const uint4*>(x + r * x_stride);
        auto put = [&](int64_t p, const uint4& w) {
            uint32_t o[N];
            whole_numbers<T, N>(w, s, o);
            if (N == 8) reinterpret_cast<uint2*>(qr)[p] = {bytes4(o[0], o[1], o[2], o[3]), bytes4(o[4 % N], o[5 % N], o[6 % N], o[7 % N])};
            else reinterpret_cast<uint32_t*>(qr)[p] = bytes4(o[0], o[1], o[2], o[3]);
        };
#pragma unroll
        for (int j = 0; j < QT_KEEP; ++j)
            if (tid + j * nt < whole) put(tid + j * nt, keep[j]);
        for (int64_t i = tid + QT_KEEP * nt; i < whole; i += nt) put(i, __ldg(packs + i));
        if (last) {
            uint32_t o[N];
            whole_numbers<T, N>(vpk::edge_pack(row.x, whole * N, k, 0), s, o);
#pragma unroll
            for (int e = 0; e < N - 1; ++e)
                if (whole * N + e < k) qr[whole * N + e] = (int8_t)(uint8_t)o[e];
        }
    } else {
        auto put = [&](int64_t p, const uint4& w) {  // by whole warps; lanes behind the row have nothing to store
            uint32_t o[N];
            whole_numbers<T, N>(w, s, o);
            const int64_t at = row.first(p), left = k - at;
            store<N>(qr + at, o, at < 0 ? (int)-at : 0, left < 0 ? 0 : left < N ? (int)left : N);
        };
#pragma unroll
        for (int j = 0; j < QT_KEEP; ++j)
            if ((tid & ~31) + j * nt < row.count) put(tid + j * nt, keep[j]);
        for (int64_t i = tid + QT_KEEP * nt; (i & ~(int64_t)31) < row.count; i += nt) put(i, i < row.count ? row.load(i, 0) : uint4{0, 0, 0, 0});
    }
}

// As many threads as the row needs with QT_KEEP packs each: with 1024 threads an SM that is 128 KB in flight, which HBM needs
// (4 packs a thread and twice the threads a row: 11008 x 4096 fp32 44 instead of 35 us).
template <typename T>
int launch(const void* x, int64_t m, int64_t k, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, cudaStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    const int64_t want = ((k + N - 1) / N + QT_KEEP - 1) / QT_KEEP;
    const unsigned nt = want <= 32 ? 32 : want >= 1024 ? 1024 : (unsigned)(want + 31) / 32 * 32;
    const unsigned rows = nt == 32 ? 8 : 1;
    const bool aligned = ((uintptr_t)x) % 16 == 0 && x_stride % N == 0 && ((uintptr_t)q) % N == 0 && q_stride % N == 0;
    return vi::launch_early("k_int8_quantize", aligned ? k_int8_quantize<T, true> : k_int8_quantize<T, false>, dim3((unsigned)((m + rows - 1) / rows)),
                            dim3(nt, rows), 0, 1, true, st, (const T*)x, x_stride, m, k, q, q_stride, scale);
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

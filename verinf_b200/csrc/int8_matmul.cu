// int8 x int8 product with whole-number sums: scaled per token and channel, raw, or as field elements.
//
// S = A.B, A (m, k) and B (k, n) int8; |S| <= 2^14 k < 2^31 for k <= 131071, so 32-bit sums are exact in any order.
// out = S sa_i sb_j in fp32, rounded once to the output type; or S; or S mod p (negative sums as p - |S|).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/verinf_b200.h"
#include "common.cuh"
#include "gl.cuh"

namespace {

constexpr int64_t I8_MAX_K = 131071;

template <typename T> struct Out;
template <> struct Out<float> { static __device__ __forceinline__ float make(int s, float sc) { return (float)s * sc; } };
template <> struct Out<__half> { static __device__ __forceinline__ __half make(int s, float sc) { return __float2half_rn((float)s * sc); } };
template <> struct Out<__nv_bfloat16> { static __device__ __forceinline__ __nv_bfloat16 make(int s, float sc) { return __float2bfloat16_rn((float)s * sc); } };
template <> struct Out<int32_t> { static __device__ __forceinline__ int32_t make(int s, float) { return s; } };
// p - |s| = s - (2^32 - 1) in 64-bit words
template <> struct Out<uint64_t> { static __device__ __forceinline__ uint64_t make(int s, float) { return (uint64_t)(int64_t)s - (s < 0 ? vgl::EPS : 0ull); } };

// 64 x 64 outputs a block, 4 x 4 a thread, slices of 32 terms in shared memory, four products an instruction.
template <typename T>
__global__ void __launch_bounds__(256) k_int8_tile(const int8_t* __restrict__ A, int64_t lda, const int8_t* __restrict__ B, int64_t bk, int64_t bn,
                                                   const float* __restrict__ sa, const float* __restrict__ sb, T* __restrict__ C, int64_t ldc,
                                                   int64_t m, int64_t k, int64_t n) {
    __shared__ int As[64][9], Bs[64][9];
    const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 64;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    int acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k; k0 += 32) {
        for (int i = tid; i < 64 * 32; i += 256) {
            const int64_t r = r0 + (i >> 5), kk = k0 + (i & 31);
            reinterpret_cast<int8_t*>(&As[i >> 5][0])[i & 31] = r < m && kk < k ? A[r * lda + kk] : (int8_t)0;
            const int cl = bn == 1 ? (i & 63) : (i >> 5), kl = bn == 1 ? (i >> 6) : (i & 31);      // neighbours read neighbours
            const int64_t c = c0 + cl, kb = k0 + kl;
            reinterpret_cast<int8_t*>(&Bs[cl][0])[kl] = c < n && kb < k ? B[kb * bk + c * bn] : (int8_t)0;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            int a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] = As[ty + 16 * i][w]; b[i] = Bs[tx + 16 * i][w]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t r = r0 + ty + 16 * i, c = c0 + tx + 16 * j;
            if (r < m && c < n) C[r * ldc + c] = Out<T>::make(acc[i][j], (sa ? sa[r] : 1.0f) * (sb ? sb[c] : 1.0f));
        }
}

template <typename T>
int launch_tile(const int8_t* A, int64_t lda, const int8_t* B, int64_t bk, int64_t bn, const float* sa, const float* sb, void* C, int64_t ldc,
                int64_t m, int64_t k, int64_t n, cudaStream_t st) {
    dim3 grid((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64));
    k_int8_tile<T><<<grid, 256, 0, st>>>(A, lda, B, bk, bn, sa, sb, (T*)C, ldc, m, k, n);
    return vi::check_launch("k_int8_tile");
}

}  // namespace

extern "C" int vi_int8_matmul(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb, int b_by_channel, const float* sa, const float* sb,
                              void* C, int out_type, int64_t ldc, int64_t m, int64_t k, int64_t n, void* stream) {
    VI_REQUIRE(m >= 0 && k >= 0 && n >= 0, "int8_matmul: negative size");
    VI_REQUIRE(out_type >= VI_F32 && out_type <= VI_FIELD, "int8_matmul: unknown output type");
    VI_REQUIRE(k <= I8_MAX_K, "int8_matmul: k = %lld, but 32-bit sums hold at most 131071 products", (long long)k);
    VI_REQUIRE(out_type < VI_I32 || (!sa && !sb), "int8_matmul: whole-number outputs take no scales");
    if (m == 0 || n == 0) return VI_OK;
    static const int out_bytes[] = {4, 2, 2, 4, 8};
    VI_REQUIRE(C && ((uintptr_t)C) % out_bytes[out_type] == 0, "int8_matmul: null or misaligned output");
    VI_REQUIRE(m == 1 || ldc >= n, "int8_matmul: output rows overlap (stride below n)");
    VI_REQUIRE(k == 0 || (A && B), "int8_matmul: null input");
    VI_REQUIRE(((uintptr_t)sa) % 4 == 0 && ((uintptr_t)sb) % 4 == 0, "int8_matmul: misaligned scales");
    VI_REQUIRE((m + 63) / 64 <= 65535 && (n + 63) / 64 <= 0x7FFFFFFF, "int8_matmul: matrix too large for one launch");
    cudaStream_t st = (cudaStream_t)stream;
    const int64_t bk = b_by_channel ? 1 : ldb, bn = b_by_channel ? ldb : 1;
    switch (out_type) {
        case VI_F32: return launch_tile<float>(A, lda, B, bk, bn, sa, sb, C, ldc, m, k, n, st);
        case VI_F16: return launch_tile<__half>(A, lda, B, bk, bn, sa, sb, C, ldc, m, k, n, st);
        case VI_BF16: return launch_tile<__nv_bfloat16>(A, lda, B, bk, bn, sa, sb, C, ldc, m, k, n, st);
        case VI_I32: return launch_tile<int32_t>(A, lda, B, bk, bn, sa, sb, C, ldc, m, k, n, st);
        default: return launch_tile<uint64_t>(A, lda, B, bk, bn, sa, sb, C, ldc, m, k, n, st);
    }
}

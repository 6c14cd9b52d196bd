// int8 x int8 product with whole-number sums: scaled per token and channel, raw, or as field elements.
//
// S = A.B, A (m, k) and B (k, n) int8; |S| <= 2^14 k < 2^31 for k <= 131071, so 32-bit sums are exact in any order.
// out = S sa_i sb_j in fp32, rounded once to the output type; or S; or S mod p (negative sums as p - |S|).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "../../include/verinf_b200.h"
#include "common.cuh"
#include "gl.cuh"
#include "launch.cuh"
#include "umma.cuh"

namespace {

using namespace vumma;

constexpr int64_t I8_MAX_K = 131071, I8_MAX_MN = (int64_t(1) << 31) - 256;      // tiles that reach beyond the end keep 31-bit indices
constexpr int I8_MAX_SMEM = 227 * 1024;

template <typename T> struct Out;
template <> struct Out<float> { static __device__ __forceinline__ float make(int s, float a, float b) { return (float)s * a * b; } };
template <> struct Out<__half> { static __device__ __forceinline__ __half make(int s, float a, float b) { return __float2half_rn((float)s * a * b); } };
template <> struct Out<__nv_bfloat16> { static __device__ __forceinline__ __nv_bfloat16 make(int s, float a, float b) { return __float2bfloat16_rn((float)s * a * b); } };
template <> struct Out<int32_t> { static __device__ __forceinline__ int32_t make(int s, float, float) { return s; } };
// p - |s| = s - (2^32 - 1) in 64-bit words
template <> struct Out<uint64_t> { static __device__ __forceinline__ uint64_t make(int s, float, float) { return (uint64_t)(int64_t)s - (s < 0 ? vgl::EPS : 0ull); } };

// ---- tcgen05 ---------------------------------------------------------------------------------------------------
// A tile is 128 channels by `nt` tokens: the weight is the operand with 128 rows, so a lane of tensor memory is a channel, a
// column a token, and a warp writes 32 neighbouring channels of one token.
constexpr int I8_TN = 128, I8_KS = 128, I8_THREADS = 256, I8_MAX_STAGES = 8, I8_MAX_SPLIT = 8;
constexpr int I8_W_BYTES = I8_TN * I8_KS;
constexpr int I8_TAIL = 2 * I8_MAX_STAGES * 8 + 64 + 256 * 4;      // barriers, tensor-memory slot, scales of the tokens

__device__ int g_i8_status, g_i8_taken;                              // first wait that expired, 0 = none; what the last question took
__global__ void k_int8_take_status() { g_i8_taken = atomicExch(&g_i8_status, 0); }

struct Plan { bool pair, direct; int nt, split, stages; };
__host__ __device__ inline int i8_stage_bytes(int nt) { return I8_W_BYTES + nt * I8_KS; }

// 128-byte rows, 128-byte swizzle, groups of 8 rows 1024 bytes apart: K-major tiles (rows = channels or tokens), and tiles
// of a row-major weight (rows = terms; one atom is 128 channels wide, so the leading offset is never used).
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// s8 x s8 -> s32; bit 15: the first operand is MN-major
__device__ __forceinline__ uint32_t idesc_s8(int nt, bool kn) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (kn ? 1u << 15 : 0u) | ((uint32_t)(nt >> 3) << 17) | ((uint32_t)(I8_TN >> 4) << 24);
}

// A thread's channel of 16 tokens, `out` the first of them and ldc from each to the next: `tokens` of them exist.
template <typename T>
__device__ __forceinline__ void write_out(T* out, int64_t ldc, const uint32_t (&sum)[16], const float* sa, float sb, int tokens) {
    if (tokens >= 16) {
        T v[16];
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 a = *reinterpret_cast<const float4*>(sa + j);
            v[j] = Out<T>::make((int)sum[j], a.x, sb);
            v[j + 1] = Out<T>::make((int)sum[j + 1], a.y, sb);
            v[j + 2] = Out<T>::make((int)sum[j + 2], a.z, sb);
            v[j + 3] = Out<T>::make((int)sum[j + 3], a.w, sb);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) out[j * ldc] = v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 15; ++j) {
            if (j < tokens) out[0] = Out<T>::make((int)sum[j], sa[j], sb);
            out += ldc;
        }
    }
}

// ---- rows off the 16-byte grid ------------------------------------------------------------------------------------
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int by) {      // 16 of 32 bytes, from `by` on
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (by & 8) { w[0] = w[2]; w[1] = w[3]; w[2] = w[4]; w[3] = w[5]; w[4] = w[6]; w[5] = w[7]; }
    if (by & 4) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = w[4]; w[4] = w[5]; }
    const int bits = 8 * (by & 3);
    return {__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits)};
}

__device__ __forceinline__ uint4 first_bytes(const uint4& v, int n) {       // zero from byte n (1 .. 15) on
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = n - 4 * i;
        o[i] = left >= 4 ? w[i] : left <= 0 ? 0u : w[i] & ((1u << (8 * left)) - 1);
    }
    return {o[0], o[1], o[2], o[3]};
}

struct Operands {
    const int8_t *A, *B;
    int64_t lda, ldb;
};

// Tiles of `rows` x 128 bytes whose rows start anywhere, made as TMA with the 128-byte swizzle would bring them.  TMA reads no
// such rows, but a cp.async reads any cell of the 16-byte grid: the nine cells that hold a row's 128 bytes go to shared memory
// as they are, some slices ahead, and are shifted from there into place.  Six warps, each with every sixth row from end to end,
// so that a warp waits for nothing but its own copies.  Only cells with bytes of the row are read.
constexpr int I8_LOADERS = I8_THREADS / 32 - 2, I8_CELLS = 9, I8_RAW_STAGES = 3, I8_DIRECT_STAGES = 2;
struct Tile {
    const int8_t* src;
    int64_t pitch, row0, rows_end, len;      // first row, end of the rows, bytes of a row
    int rows;
};
// Row r of a warp's rows is row id + 6 r of the tile.  Three rows a step, a lane with one of their 27 cells.
__device__ __forceinline__ void fetch_cells(const Tile& t, int64_t c0, uint32_t raw, int id, int lane) {
    const int cell = lane % I8_CELLS, r0 = id + I8_LOADERS * (lane / I8_CELLS);
    const int64_t rows = t.rows_end - t.row0;
    const int end = lane >= 3 * I8_CELLS ? 0 : rows < t.rows ? (int)rows : t.rows;
    uintptr_t row = (uintptr_t)(t.src + (t.row0 + r0) * t.pitch);
    const uintptr_t step = 3 * I8_LOADERS * t.pitch;
    uint32_t to = raw + (r0 * I8_CELLS + cell) * 16;
#pragma unroll 4
    for (int r = r0; r < end; r += 3 * I8_LOADERS) {
        const uintptr_t at = ((row + c0) & ~(uintptr_t)15) + 16 * cell;
        if (at < row + t.len) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(at) : "memory");
        row += step;
        to += 3 * I8_LOADERS * I8_CELLS * 16;
    }
}
// Four rows a step, eight cells of the tile each.  `last`: zero behind the row's end (one of the two operands has to be).
template <bool LAST>
__device__ __forceinline__ void shift_cells(const Tile& t, int64_t c0, const uint8_t* raw, uint8_t* dst, int id, int lane) {
    const int c = lane & 7, r0 = id + I8_LOADERS * (lane >> 3);
    uint32_t by = (uint32_t)(uintptr_t)(t.src + c0) + (uint32_t)(t.row0 + r0) * (uint32_t)t.pitch;      // low bits of the row's address
    const uint32_t step = 4 * I8_LOADERS * (uint32_t)t.pitch;
    const uint4* from = reinterpret_cast<const uint4*>(raw) + r0 * I8_CELLS + c;
#pragma unroll 2
    for (int r = r0; r < t.rows; r += 4 * I8_LOADERS) {
        uint4 v = shifted(from[0], from[1], by & 15);
        if (LAST) {
            const int64_t left = t.len - c0 - 16 * c;
            if (left <= 0) v = {0, 0, 0, 0};
            else if (left < 16) v = first_bytes(v, (int)left);
        }
        *reinterpret_cast<uint4*>(dst + r * 128 + ((c ^ (r & 7)) << 4)) = v;
        by += step;
        from += 4 * I8_LOADERS * I8_CELLS;
    }
}

__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

enum { I8_ERR_FULL = 1, I8_ERR_EMPTY = 2, I8_ERR_ACC = 3 };

// One tile a block, or, with split > 1, one tile a cluster whose blocks each take a share of the terms; the sums meet through
// distributed shared memory (whole numbers: the order does not matter).  For few tokens, where the weight's bytes, the latency of
// the first loads and of the join, and uneven shares bind: 1 x 4096 x 11008 10.5 us (4.3 TB/s), 16 x 11008 x 4096 11.8 us (3.9 TB/s).
// Whole blocks of clusters do not fill the machine: 344 of 128 KB on 132 SMs put 384 KB on the busiest, where an even share of 148
// is 298 KB, and 256 of 176 KB in clusters of eight on 120 SMs put 528 KB there.
// DIRECT: operands off the 16-byte grid, brought by warps 2 .. 7 instead of TMA.
template <typename T, bool KN, bool DIRECT>
__global__ void __launch_bounds__(I8_THREADS) k_int8_umma(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Operands in,
                                                          const float* __restrict__ sa, const float* __restrict__ sb, T* __restrict__ C, int64_t ldc,
                                                          int64_t m, int64_t k, int64_t n, int t_tiles, int slices, int nt, int split, int stages) {
    extern __shared__ uint8_t i8_raw[];
    uint8_t* base = (uint8_t*)(((uintptr_t)i8_raw + 1023) & ~(uintptr_t)1023);
    const int stage_bytes = i8_stage_bytes(nt);
    uint64_t* bars = (uint64_t*)(base + stages * stage_bytes);
    float* sa_s = (float*)(bars + 2 * I8_MAX_STAGES + 8);
    volatile uint32_t* tmem_slot = (volatile uint32_t*)(bars + 2 * I8_MAX_STAGES + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    const uint32_t ring = smem_u32(base), full0 = smem_u32(bars), empty0 = smem_u32(bars + I8_MAX_STAGES), accb = smem_u32(bars + 2 * I8_MAX_STAGES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)blockIdx.x % split, tile = (int)blockIdx.x / split;
    const int64_t n0 = (int64_t)(tile / t_tiles) * I8_TN, m0 = (int64_t)(tile % t_tiles) * nt;
    const int s0 = (int)((int64_t)slices * rank / split), s1 = (int)((int64_t)slices * (rank + 1) / split);
    uint32_t cols = 32;
    while ((int)cols < nt) cols <<= 1;

    if (tid == 0) {
        for (int s = 0; s < stages; ++s) { mbar_init(full0 + 8 * s, DIRECT ? I8_LOADERS : 1); mbar_init(empty0 + 8 * s, 1); }
        mbar_init(accb, 1);
        *abort_flag = 0;
        if (!DIRECT) {
            prefetch_map(&map_w);
            prefetch_map(&map_x);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (!DIRECT && tid == 0) {     // the weight's first tiles on their way while the kernel before this one ends
        for (int s = s0; s < s1 && s < s0 + stages; ++s) {
            if (KN) prefetch_tile(&map_w, (int32_t)n0, s * I8_KS);
            else prefetch_tile(&map_w, s * I8_KS, (int32_t)n0);
        }
    }
    vi::await_inputs();
    for (int j = tid; j < nt; j += I8_THREADS) sa_s[j] = sa && m0 + j < m ? sa[m0 + j] : 1.0f;
    const int quad = warp & 3, half = warp >> 2;
    const int64_t ch = n0 + 32 * quad + lane;
    const float sbv = sb && ch < n ? sb[ch] : 1.0f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (DIRECT && warp >= 2) {
        uint8_t* raw = base + stages * stage_bytes + I8_TAIL;
        const int raw_bytes = (I8_TN + nt) * I8_CELLS * 16, w_raw = I8_TN * I8_CELLS * 16, id = warp - 2;
        const Tile x = {in.A, in.lda, m0, m, k, nt};
        auto weight = [&](int s) { return KN ? Tile{in.B, in.ldb, (int64_t)s * I8_KS, k, n, I8_KS} : Tile{in.B, in.ldb, n0, n, k, I8_TN}; };
        auto fetch = [&](int s) {
            if (s < s1) {
                const uint32_t to = smem_u32(raw) + (s % I8_RAW_STAGES) * raw_bytes;
                fetch_cells(weight(s), KN ? n0 : (int64_t)s * I8_KS, to, id, lane);
                fetch_cells(x, (int64_t)s * I8_KS, to + w_raw, id, lane);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int st = 0;
        uint32_t par = 0;
        for (int s = s0; s < s0 + I8_RAW_STAGES - 1; ++s) fetch(s);
        for (int s = s0; s < s1; ++s) {
            fetch(s + I8_RAW_STAGES - 1);         // into the cells that this warp shifted out of in the step before
            asm volatile("cp.async.wait_group %0;" ::"n"(I8_RAW_STAGES - 1) : "memory");
            __syncwarp();
            if (__any_sync(~0u, s - s0 >= stages && !mbar_wait_soon(empty0 + 8 * st, par ^ 1))) { *abort_flag = I8_ERR_EMPTY; break; }
            const uint8_t* from = raw + (s % I8_RAW_STAGES) * raw_bytes;
            uint8_t* dst = base + st * stage_bytes;
            shift_cells<false>(weight(s), KN ? n0 : (int64_t)s * I8_KS, from, dst, id, lane);
            if (s + 1 < slices) shift_cells<false>(x, (int64_t)s * I8_KS, from + w_raw, dst + I8_W_BYTES, id, lane);
            else shift_cells<true>(x, (int64_t)s * I8_KS, from + w_raw, dst + I8_W_BYTES, id, lane);
            fence_to_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full0 + 8 * st);
            if (++st == stages) { st = 0; par ^= 1; }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (!DIRECT && warp == 0) {
        int st = 0;
        uint32_t par = 0, dst = ring;
        for (int s = s0; s < s1; ++s) {
            if (s - s0 >= stages && __any_sync(~0u, !mbar_wait_soon(empty0 + 8 * st, par ^ 1))) { *abort_flag = I8_ERR_EMPTY; break; }
            if (elect_one()) {
                const uint32_t fb = full0 + 8 * st;
                mbar_expect_tx(fb, stage_bytes);
                if (KN) tma_load_2d(dst, &map_w, (int32_t)n0, s * I8_KS, fb);
                else tma_load_2d(dst, &map_w, s * I8_KS, (int32_t)n0, fb);
                tma_load_2d(dst + I8_W_BYTES, &map_x, s * I8_KS, (int32_t)m0, fb);
            }
            dst += stage_bytes;
            if (++st == stages) { st = 0; par ^= 1; dst = ring; }
        }
    } else if (warp == 1) {
        int st = 0;
        uint32_t par = 0, at = 0;                                      // at: the stage, in the descriptors' 16 bytes
        const uint32_t idesc = idesc_s8(nt, KN);
        const uint64_t w0 = desc_sw128(ring), x0 = desc_sw128(ring + I8_W_BYTES);
        for (int s = s0; s < s1; ++s) {
            if (__any_sync(~0u, !mbar_wait_soon(full0 + 8 * st, par))) { *abort_flag = I8_ERR_FULL; break; }
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < I8_KS / 32; ++kk)
                    umma_i8(tmem, w0 + at + kk * (KN ? 32 * 128 / 16 : 2), x0 + at + kk * 2, idesc, s > s0 || kk > 0);
                if (s + stages < s1) umma_commit(empty0 + 8 * st);        // the last ones are not loaded again
                if (s + 1 == s1) umma_commit(accb);
            }
            at += stage_bytes / 16;
            if (++st == stages) { st = 0; par ^= 1; at = 0; }
        }
    }
    __syncwarp();
    bool ok = mbar_wait_soon(accb, 0);
    vi::release_next();
    if (!ok && *abort_flag == 0) *abort_flag = I8_ERR_ACC;
    tc_fence_after();
    ok = ok && *abort_flag == 0;
    T* out = C + m0 * ldc + ch;
    const int tokens = ch >= n ? 0 : m - m0 < nt ? (int)(m - m0) : nt;
    if (ok) {
        for (int q = half; q < nt / 16; q += 2) {
            uint32_t r[16];
            tmem_ld16(tmem + ((uint32_t)(32 * quad) << 16) + 16 * q, r);
            tmem_ld_wait();
            if (split == 1) write_out(out + 16 * q * ldc, ldc, r, sa_s + 16 * q, sbv, tokens - 16 * q);
            else {
#pragma unroll
                for (int j = 0; j < 16; ++j) ((uint32_t*)base)[(16 * q + j) * I8_TN + 32 * quad + lane] = r[j];
            }
        }
    }
    if (split > 1) {
        // This block's tensor memory is free before it waits for the others: two blocks of a pair on another stream, each beside
        // a block of this cluster, could otherwise hold what one of them waits for while the other waits for theirs.
        tc_fence_before();
        __syncthreads();
        if (warp == 1 && *abort_flag == 0) tmem_free(tmem, cols);
        __syncwarp();
        cluster_sync();
        const int per = nt / split, j1 = (rank + 1) * per < tokens ? (rank + 1) * per : tokens;
        if (ok) {
            for (int j = rank * per + half; j < j1; j += 2) {
                uint32_t part[I8_MAX_SPLIT], v = 0;
#pragma unroll
                for (int p = 0; p < I8_MAX_SPLIT; ++p)        // all on their way before the first is added
                    part[p] = p < split ? cluster_ld(ring + (j * I8_TN + 32 * quad + lane) * 4, p) : 0u;
#pragma unroll
                for (int p = 0; p < I8_MAX_SPLIT; ++p) v += part[p];
                out[j * ldc] = Out<T>::make((int)v, sa_s[j], sbv);
            }
        }
        __syncwarp();
        cluster_sync();            // no block leaves while another reads its sums
    }
    if (*abort_flag) {
        if (tid == 0) atomicCAS(&g_i8_status, 0, (int)*abort_flag);
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);        // copies in flight land in this block's shared memory
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1 && (split == 1 || *abort_flag)) tmem_free(tmem, cols);
}

// ---- pairs of blocks, persistent --------------------------------------------------------------------------------
// A tile is 256 channels by `nt` tokens, 128 channels a block; each block brings its channels and half of the tokens, so that
// the tokens cross from L2 once a pair.  Two accumulators a block (2 x 256 columns of tensor memory): while eight warps write
// one tile out, the products of the next one run.  Bound by the tensor pipe and its feeding, about 0.32 us a slice of 256 tokens (0.26
// of them the products'): 1000 x 4096 x 11008 35 us (2.6 P operations a second; 215 tiles of 224 tokens on 74 pairs), 4096 x 5120 x
// 8192 104 us (3.3 P; 512 tiles).  The warps that load and that issue the products run their loops whole and elect the lane that
// issues: with a loop of one lane each slice costs 0.07 us more (39 and 113 us).
constexpr int I8_PAIR_THREADS = 320, I8_PAIR_STAGES = 8;
constexpr int I8_PAIR_TAIL = (2 * I8_PAIR_STAGES + 4 + 1) * 8 + 24 + 8 * 256 * 4;      // barriers, slots, the tokens' scales for each writing warp
__host__ __device__ inline int i8_pair_stage_bytes(int nt) { return I8_W_BYTES + nt / 2 * I8_KS; }

template <typename T, bool KN>
__global__ void __launch_bounds__(I8_PAIR_THREADS)
k_int8_pair(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const float* __restrict__ sa,
            const float* __restrict__ sb, T* __restrict__ C, int64_t ldc, int64_t m, int64_t n, int t_tiles, int tiles, int slices, int nt, int stages) {
    extern __shared__ uint8_t i8_raw[];
    uint8_t* base = (uint8_t*)(((uintptr_t)i8_raw + 1023) & ~(uintptr_t)1023);
    const int stage_bytes = i8_pair_stage_bytes(nt);
    uint64_t* bars = (uint64_t*)(base + stages * stage_bytes);
    volatile uint32_t* tmem_slot = (volatile uint32_t*)(bars + 2 * I8_PAIR_STAGES + 4);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    const uint32_t ring = smem_u32(base), full0 = smem_u32(bars), empty0 = smem_u32(bars + I8_PAIR_STAGES),
                   acc_full0 = smem_u32(bars + 2 * I8_PAIR_STAGES), acc_empty0 = acc_full0 + 16;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)blockIdx.x & 1, first = (int)blockIdx.x >> 1, step = (int)gridDim.x >> 1;

    if (tid == 0) {
        for (int s = 0; s < stages; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(acc_full0 + 8 * a, 1); mbar_init(acc_empty0 + 8 * a, 16); }
        *abort_flag = 0;
        prefetch_map(&map_w);
        prefetch_map(&map_x);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {                // the weight's first tiles on their way while the kernel before this one ends
        const int32_t n0 = (first / t_tiles) * 2 * I8_TN + rank * I8_TN;
        for (int s = 0; s < slices && s < stages; ++s) {
            if (KN) prefetch_tile(&map_w, n0, s * I8_KS);
            else prefetch_tile(&map_w, s * I8_KS, n0);
        }
    }
    vi::await_inputs();
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        {
            int st = 0, filled = 0;
            uint32_t par = 0, dst = ring;
            const uint32_t full_first = cluster_addr(full0, 0);       // the pair's first block's
            for (int t = first; t < tiles && !*abort_flag; t += step) {
                const int32_t n0 = (t / t_tiles) * 2 * I8_TN + rank * I8_TN, m0 = (t % t_tiles) * nt + rank * (nt / 2);
                for (int s = 0; s < slices; ++s) {
                    if (filled == stages) {
                        if (__any_sync(~0u, !mbar_wait_soon(empty0 + 8 * st, par ^ 1))) { *abort_flag = I8_ERR_EMPTY; break; }
                    } else ++filled;
                    if (elect_one()) {
                        const uint32_t fb = full_first + 8 * st;
                        if (rank == 0) mbar_expect_tx(full0 + 8 * st, 2 * stage_bytes);
                        if (KN) tma_load_2d_pair(dst, &map_w, n0, s * I8_KS, fb);
                        else tma_load_2d_pair(dst, &map_w, s * I8_KS, n0, fb);
                        tma_load_2d_pair(dst + I8_W_BYTES, &map_x, s * I8_KS, m0, fb);
                    }
                    dst += stage_bytes;
                    if (++st == stages) { st = 0; par ^= 1; dst = ring; }
                }
            }
            // the last commits arrive here: stay until they have
            const bool wrapped = filled == stages;
            if (!wrapped) st = 0;
            for (int i = 0; i < filled && !*abort_flag; ++i) {
                if (!mbar_wait_soon(empty0 + 8 * st, wrapped ? par ^ 1 : 0)) *abort_flag = I8_ERR_EMPTY;
                if (++st == stages) { st = 0; par ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            int st = 0, acc = 0, used = 0;
            uint32_t par = 0, acc_par = 0;
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | (KN ? 1u << 15 : 0u) | ((uint32_t)(nt >> 3) << 17) | ((uint32_t)(2 * I8_TN >> 4) << 24);
            const uint64_t w0 = desc_sw128(ring), x0 = desc_sw128(ring + I8_W_BYTES);
            uint32_t at = 0;                                           // of the stage, in the descriptors' 16 bytes
            for (int t = first; t < tiles && !*abort_flag; t += step) {
                if (used >= 2 && __any_sync(~0u, !mbar_wait_soon(acc_empty0 + 8 * acc, acc_par ^ 1))) { *abort_flag = I8_ERR_ACC; break; }
                ++used;
                tc_fence_after();
                const uint32_t d = tmem + 256 * acc;
                for (int s = 0; s < slices; ++s) {
                    if (__any_sync(~0u, !mbar_wait_soon(full0 + 8 * st, par))) { *abort_flag = I8_ERR_FULL; break; }
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < I8_KS / 32; ++kk)
                            umma_i8_pair(d, w0 + at + kk * (KN ? 32 * 128 / 16 : 2), x0 + at + kk * 2, idesc, s > 0 || kk > 0);
                        umma_commit_pair(empty0 + 8 * st);
                    }
                    at += stage_bytes / 16;
                    if (++st == stages) { st = 0; par ^= 1; at = 0; }
                }
                if (elect_one()) umma_commit_pair(acc_full0 + 8 * acc);
                if (++acc == 2) { acc = 0; acc_par ^= 1; }
            }
        }
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2;
        float* sa_s = (float*)(bars + 2 * I8_PAIR_STAGES + 6) + 256 * (warp - 2);      // 16-byte aligned
        int acc = 0;
        uint32_t acc_par = 0;
        for (int t = first; t < tiles; t += step) {
            const int64_t ch = (int64_t)(t / t_tiles) * 2 * I8_TN + rank * I8_TN + 32 * quad + lane, m0 = (int64_t)(t % t_tiles) * nt;
            const float sbv = sb && ch < n ? sb[ch] : 1.0f;
            __syncwarp();
            for (int j = lane; j < nt; j += 32) sa_s[j] = sa && m0 + j < m ? sa[m0 + j] : 1.0f;      // while the products run
            __syncwarp();
            if (!mbar_wait_soon(acc_full0 + 8 * acc, acc_par)) { *abort_flag = I8_ERR_ACC; break; }
            if (*abort_flag) break;
            tc_fence_after();
            const uint32_t from = tmem + 256 * acc + ((uint32_t)(32 * quad) << 16);
            T* out = C + m0 * ldc + ch;
            const int tokens = ch >= n ? 0 : m - m0 < nt ? (int)(m - m0) : nt;
            for (int q = half; q < nt / 16; q += 2) {
                uint32_t r[16];
                tmem_ld16(from + 16 * q, r);
                tmem_ld_wait();
                write_out(out + 16 * q * ldc, ldc, r, sa_s + 16 * q, sbv, tokens - 16 * q);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(cluster_addr(acc_empty0 + 8 * acc, 0));
            if (++acc == 2) { acc = 0; acc_par ^= 1; }
        }
    }
    __syncwarp();
    vi::release_next();
    if (*abort_flag) {
        if (lane == 0) atomicCAS(&g_i8_status, 0, (int)*abort_flag);
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
    tc_fence_before();
    cluster_sync();            // the other block's arrivals and the pair's products have ended
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// No terms (k = 0): sums of 0, which a scale that is not finite turns into NaN as it does elsewhere.
template <typename T>
__global__ void __launch_bounds__(256) k_int8_no_terms(const float* __restrict__ sa, const float* __restrict__ sb, T* __restrict__ C, int64_t ldc, int64_t m, int64_t n) {
    vi::await_inputs();
    for (int64_t i = blockIdx.x; i < m; i += gridDim.x)
        for (int64_t j = threadIdx.x; j < n; j += 256) C[i * ldc + j] = Out<T>::make(0, sa ? sa[i] : 1.0f, sb ? sb[j] : 1.0f);
}

// rows x len bytes, rows `pitch` bytes apart; box: 128 bytes x box_rows
int make_map(CUtensorMap* map, const int8_t* ptr, int64_t rows, int64_t len, int64_t pitch, int box_rows) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return vi::fail(VI_ERR_CUDA, "int8_matmul: cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[2] = {(cuuint64_t)len, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {(cuuint32_t)I8_KS, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return vi::fail(VI_ERR_CUDA, "int8_matmul: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return VI_OK;
}

struct Product {
    const int8_t *A, *B;
    int64_t lda, ldb;
    bool by_channel;
    const float *sa, *sb;
    void* C;
    int64_t ldc, m, k, n;
};

// Shared memory beyond 48 KB is granted to a kernel once a device (`done`: a bit for each of the first 64; others every time).
int grant_smem(const void* kernel, std::atomic<uint64_t>& done) {
    int dev = 0;
    VI_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return VI_OK;
    VI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, I8_MAX_SMEM));
    done.fetch_or(bit, std::memory_order_relaxed);
    return VI_OK;
}

template <typename T, bool KN, bool DIRECT>
int launch_umma(const Product& p, const Plan& plan, cudaStream_t st) {
    static std::atomic<uint64_t> granted{0};
    CUtensorMap map_w = {}, map_x = {};
    int rc = VI_OK;
    if (!DIRECT) {
        rc = KN ? make_map(&map_w, p.B, p.k, p.n, p.ldb, I8_KS) : make_map(&map_w, p.B, p.n, p.k, p.ldb, I8_TN);
        if (rc == VI_OK) rc = make_map(&map_x, p.A, p.m, p.k, p.lda, plan.nt);
    }
    const int smem = plan.stages * i8_stage_bytes(plan.nt) + 1024 + I8_TAIL + (DIRECT ? I8_RAW_STAGES * (I8_TN + plan.nt) * I8_CELLS * 16 : 0);
    if (rc == VI_OK) rc = grant_smem((const void*)k_int8_umma<T, KN, DIRECT>, granted);
    if (rc) return rc;
    const int64_t t_tiles = (p.m + plan.nt - 1) / plan.nt, n_tiles = (p.n + I8_TN - 1) / I8_TN;
    VI_REQUIRE(t_tiles * n_tiles * plan.split <= 0x7FFFFFFF, "int8_matmul: matrix too large for one launch");
    return vi::launch_early("k_int8_umma", k_int8_umma<T, KN, DIRECT>, dim3((unsigned)(t_tiles * n_tiles * plan.split)), dim3(I8_THREADS), (size_t)smem,
                            plan.split, true, st, map_w, map_x, Operands{p.A, p.B, p.lda, p.ldb}, p.sa, p.sb, (T*)p.C, p.ldc, p.m, p.k, p.n, (int)t_tiles,
                            (int)((p.k + I8_KS - 1) / I8_KS), plan.nt, plan.split, plan.stages);
}

template <typename T, bool KN>
int launch_pair(const Product& p, const Plan& plan, cudaStream_t st) {
    static std::atomic<uint64_t> granted{0};
    CUtensorMap map_w, map_x;
    int rc = KN ? make_map(&map_w, p.B, p.k, p.n, p.ldb, I8_KS) : make_map(&map_w, p.B, p.n, p.k, p.ldb, I8_TN);
    if (rc) return rc;
    rc = make_map(&map_x, p.A, p.m, p.k, p.lda, plan.nt / 2);
    if (rc) return rc;
    const int smem = plan.stages * i8_pair_stage_bytes(plan.nt) + 1024 + I8_PAIR_TAIL;
    rc = grant_smem((const void*)k_int8_pair<T, KN>, granted);
    if (rc) return rc;
    const int64_t t_tiles = (p.m + plan.nt - 1) / plan.nt, tiles = t_tiles * ((p.n + 2 * I8_TN - 1) / (2 * I8_TN));
    VI_REQUIRE(tiles <= 0x3FFFFFFF, "int8_matmul: matrix too large for one launch");
    return vi::launch_early("k_int8_pair", k_int8_pair<T, KN>, dim3((unsigned)(2 * (tiles < 74 ? tiles : 74))), dim3(I8_PAIR_THREADS), (size_t)smem, 2, true, st,
                            map_w, map_x, p.sa, p.sb, (T*)p.C, p.ldc, p.m, p.n, (int)t_tiles, (int)tiles, (int)((p.k + I8_KS - 1) / I8_KS), plan.nt,
                            plan.stages);
}

template <typename T>
int launch_product(const Product& p, const Plan& plan, cudaStream_t st) {
    if (p.k == 0)
        return vi::launch_early("k_int8_no_terms", k_int8_no_terms<T>, dim3((unsigned)std::min<int64_t>(p.m, 148 * 8)), dim3(256), 0, 1, true, st, p.sa, p.sb,
                                (T*)p.C, p.ldc, p.m, p.n);
    if (plan.direct) return p.by_channel ? launch_umma<T, false, true>(p, plan, st) : launch_umma<T, true, true>(p, plan, st);
    if (!plan.pair) return p.by_channel ? launch_umma<T, false, false>(p, plan, st) : launch_umma<T, true, false>(p, plan, st);
    return p.by_channel ? launch_pair<T, false>(p, plan, st) : launch_pair<T, true>(p, plan, st);
}

// blocks of clusters of `split` that run at once, `room` on an SM
inline int blocks_at_once(int split, int room) { return (split <= 2 ? 148 : split == 4 ? 132 : 120) * room; }

// Which kernel and tile: the least of estimated times, in us.  The estimate knows what bounds these kernels: the bytes that must
// come from HBM (5.4 MB a us, to pairs 6.3 MB); of single blocks the operand bytes of all tiles on their way to the busiest SM (one
// block's at 61 KB a us, several blocks' together at 91 KB) or its products, 1850 columns a us; of pairs a slice's time, 0.18 us
// and 0.10 us for 256 tokens, or the write-out; a fixed part for set-up and end, the last write-out, rounds, the barriers of a
// split, and how many blocks run at once (clusters of 4 and 8 leave SMs unused).  Its constants are fitted to 1145 measured plans
// of 76 shapes (m 1 .. 3986, k 32 .. 11008, n 16 .. 32000, both layouts): 16 % off where a plan is not far from the best, and the
// chosen plan takes 1.5 % longer than the best on average, 21 % at worst (932 x 704 x 48, 7.2 us).  Among them (us): 16 x 4096 x
// 11008 split 4 11.6, unsplit 14.7, in pairs 11.5; 200 x 4096 x 11008 in pairs 15.3, else 17.2; 200 x 11008 x 4096 split 4 of 128
// tokens 19.1, in pairs 22.6; 1000 x 4096 x 11008 in pairs of 224 tokens 35.7, of 256 36.0, of 128 42, single blocks 48.5.  A pair
// makes 32 tokens at least, so up to 16 tokens go to single blocks (1 x 4096 x 11008 11.1 / 11.7, 1 x 4096 x 4096 6.9 / 10.6,
// 1 x 4096 x 32000 24.1 / 23.5).
//
// `off_grid`: bytes of the operands that TMA cannot read in place.  They are copied first (4.7 MB a us, read and written, and a
// launch more: 4 us, most of it the host's), or, where a tile has few slices, shifted on their way: about 4.4 us for a block's first
// slice and its end and 1.3 us for each other one, 1.7 us with two blocks an SM (fitted to 406 measured plans of 52 shapes, 9 % off;
// us with / without a copy, without the host's part, the better plan of each: 15 x 77 x 1125 5.3 / 4.1, 2 x 1925 x 1098 7.7 / 6.2,
// 172 x 581 x 516 6.5 / 8.0, 16 x 11007 x 4095 30 / 25, 100 x 4095 x 11007 33 / 63).
Plan make_plan(int m, int k, int n, int64_t off_grid) {
    const int slices = (k + I8_KS - 1) / I8_KS, n128 = (n + 127) / 128, n256 = (n + 255) / 256;
    const float from_hbm = (float)k * n + (float)m * k + 2.0f * m * n, hbm = from_hbm / 5.44e6f, hbm_pairs = from_hbm / 6.26e6f;
    Plan best = {};
    float least = 1e30f;
    static const int widths[] = {16, 32, 48, 64, 96, 128, 192, 256};
    for (int nt : widths) {
        if (nt > 16 && nt >= m + 32) break;
        const int room = nt <= 32 ? 3 : nt <= 128 ? 2 : 1;            // blocks an SM holds
        const int tiles = (int)std::min<int64_t>((int64_t)((m + nt - 1) / nt) * n128, 1 << 27);
        for (int split = 1; split <= I8_MAX_SPLIT && (split == 1 || slices >= 2 * split); split *= 2) {
            const int ctas = tiles * split, steps = (slices + split - 1) / split;
            const int spread = blocks_at_once(split, 1), rounds = (ctas + spread * room - 1) / (spread * room);
            const float bytes = i8_stage_bytes(nt), product = nt / 1850.0f;
            const float sm = (float)((ctas + spread - 1) / spread) * steps * std::max(bytes / 91.3e3f, product);
            const float alone = (float)rounds * steps * std::max(bytes / 60.9e3f, product);
            const float t = 2.71f + std::max(hbm, std::max(sm, alone)) + 2.79f * nt / 256 / split * rounds + (split > 1 ? 1.42f : 0.0f) + 2.28f * (rounds - 1);
            if (t < least) {
                least = t;
                best = {false, false, nt, split, (room == 3 ? 70 : room == 2 ? 104 : 200) * 1024 / i8_stage_bytes(nt)};
            }
        }
    }
    for (int nt = 32; nt <= 256 && m > 16 && (nt == 32 || nt < m + 32); nt += 32) {
        const int64_t tiles = (int64_t)((m + nt - 1) / nt) * n256;
        const float per = (float)((tiles + 73) / 74);
        const float part = nt / 256.0f;
        const float t = 3.44f + std::max(hbm_pairs, per * std::max(slices * (0.179f + 0.104f * part), 2.39f * part)) + 3.05f * part + 1.03f * (per - 1);
        if (t < least) {
            least = t;
            best = {true, false, nt, 1, std::min(I8_PAIR_STAGES, 200 * 1024 / i8_pair_stage_bytes(nt))};
        }
    }
    if (off_grid) {
        least += 4.0f + 2.0f * off_grid / 4.7e6f;
        for (int nt : {16, 32, 48, 64, 96, 128}) {
            if (nt > 16 && nt >= m + 32) break;
            const int tiles = (int)std::min<int64_t>((int64_t)((m + nt - 1) / nt) * n128, 1 << 27);
            for (int split = 1; split <= I8_MAX_SPLIT && (split == 1 || slices >= 2 * split); split *= 2) {
                const int ctas = tiles * split, steps = (slices + split - 1) / split, room = nt <= 32 ? 2 : 1;
                const int spread = blocks_at_once(split, 1), rounds = (ctas + spread * room - 1) / (spread * room);
                const float step = (room > 1 && ctas > spread ? 1.7f : 1.3f) * (I8_TN + 0.68f * nt) / 144;
                const float t = rounds * (0.56f + 3.85f * (I8_TN + nt) / 144 + (steps - 1) * step) + (split > 1 ? 1.5f : 0.0f);
                if (t < least) {
                    least = t;
                    best = {false, true, nt, split, I8_DIRECT_STAGES};
                }
            }
        }
    }
    return best;
}

// ---- operands that TMA cannot read in place -----------------------------------------------------------------------
// Rows that start off the 16-byte grid are copied to rows that start on it: a pass over those bytes, on every call (what it
// takes: at make_plan).  A thread makes 16 bytes of the copy from the two grid cells that hold them, of which it reads only
// those that hold bytes of the row.
inline __host__ __device__ int64_t up16(int64_t x) { return (x + 15) / 16 * 16; }

struct Rows {
    const int8_t* src;
    int8_t* dst;
    int64_t pitch, rows, len;
};

__global__ void __launch_bounds__(256) k_int8_align(const Rows first, const Rows second) {
    vi::await_inputs();
    const bool is_second = blockIdx.y == 1;
    const Rows r = is_second ? second : first;
    const int64_t per = up16(r.len) / 16, total = r.rows * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per, c = (i - row * per) * 16;
        const uintptr_t at = (uintptr_t)(r.src + row * r.pitch + c), end = at - c + r.len;
        const uint4* cell = (const uint4*)(at & ~(uintptr_t)15);
        const uint4 none = {0, 0, 0, 0};
        const uint4 a = __ldg(cell), b = (uintptr_t)(cell + 1) < end && (at & 15) ? __ldg(cell + 1) : none;
        reinterpret_cast<uint4*>(r.dst)[i] = shifted(a, b, (int)(at & 15));
    }
}

inline bool in_place(const void* p, int64_t pitch) { return ((uintptr_t)p) % 16 == 0 && pitch % 16 == 0; }
inline int64_t b_rows(int64_t k, int64_t n, bool by_channel) { return by_channel ? n : k; }
inline int64_t b_len(int64_t k, int64_t n, bool by_channel) { return by_channel ? k : n; }

// Copies those of the operands that need it to `room` and points p at the copies.
int align_rows(Product& p, int8_t* room, cudaStream_t st) {
    Rows todo[2];
    int n = 0;
    if (!in_place(p.A, p.lda)) {
        todo[n++] = {p.A, room, p.lda, p.m, p.k};
        p.A = room;
        p.lda = up16(p.k);
        room += p.m * p.lda;
    }
    if (!in_place(p.B, p.ldb)) {
        const int64_t rows = b_rows(p.k, p.n, p.by_channel), len = b_len(p.k, p.n, p.by_channel);
        todo[n++] = {p.B, room, p.ldb, rows, len};
        p.B = room;
        p.ldb = up16(len);
    }
    if (n == 0) return VI_OK;
    const int64_t cells0 = todo[0].rows * (up16(todo[0].len) / 16), cells1 = n > 1 ? todo[1].rows * (up16(todo[1].len) / 16) : 0;
    const int64_t want = ((cells0 > cells1 ? cells0 : cells1) + 255) / 256;
    return vi::launch_early("k_int8_align", k_int8_align, dim3((unsigned)(want < 148 * 32 ? want : 148 * 32), (unsigned)n), dim3(256), 0, 1, true, st, todo[0], todo[n - 1]);
}

int64_t copy_bytes(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb, bool nk, int64_t m, int64_t k, int64_t n) {
    if (m == 1) lda = 16;                                            // a single row has no next one
    if (b_rows(k, n, nk) == 1) ldb = 16;
    return (in_place(A, lda) ? 0 : m * up16(k)) + (in_place(B, ldb) ? 0 : b_rows(k, n, nk) * up16(b_len(k, n, nk)));
}

}  // namespace

extern "C" int64_t vi_int8_matmul_scratch_bytes(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb, int b_by_channel, int64_t m, int64_t k, int64_t n) {
    if (m <= 0 || k <= 0 || n <= 0 || m > I8_MAX_MN || n > I8_MAX_MN || k > I8_MAX_K) return 0;
    const int64_t copies = copy_bytes(A, lda, B, ldb, b_by_channel != 0, m, k, n);
    return copies && make_plan((int)m, (int)k, (int)n, copies).direct ? 0 : copies;
}

extern "C" int vi_int8_matmul(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb, int b_by_channel, const float* sa, const float* sb,
                              void* C, int out_type, int64_t ldc, int64_t m, int64_t k, int64_t n, void* scratch, int64_t scratch_bytes,
                              void* stream) {
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
    VI_REQUIRE(m <= I8_MAX_MN && n <= I8_MAX_MN, "int8_matmul: m and n are limited to 2^31 - 256");
    cudaStream_t st = (cudaStream_t)stream;
    if (m == 1) ldc = n;
    const bool nk = b_by_channel != 0;
    if (m == 1) lda = up16(k);
    if (b_rows(k, n, nk) == 1) ldb = up16(b_len(k, n, nk));
    VI_REQUIRE(k == 0 || (lda >= k && ldb >= b_len(k, n, nk)), "int8_matmul: operand rows overlap");
    VI_REQUIRE(lda < (int64_t(1) << 40) && ldb < (int64_t(1) << 40), "int8_matmul: rows too far apart");
    const int64_t copies = k ? copy_bytes(A, lda, B, ldb, nk, m, k, n) : 0;
    const Plan plan = k ? make_plan((int)m, (int)k, (int)n, copies) : Plan{};
    const int64_t need = plan.direct ? 0 : copies;
    if (need && (scratch == nullptr || scratch_bytes < need))
        return vi::fail(VI_ERR_SCRATCH, "int8_matmul: scratch of at least %lld bytes required (see vi_int8_matmul_scratch_bytes)", (long long)need);
    VI_REQUIRE(!need || ((uintptr_t)scratch) % 16 == 0, "int8_matmul: scratch must be 16-byte aligned");
    Product p = {A, B, lda, ldb, nk, sa, sb, C, ldc, m, k, n};
    if (need) {
        const int rc = align_rows(p, (int8_t*)scratch, st);
        if (rc) return rc;
    }
    switch (out_type) {
        case VI_F32: return launch_product<float>(p, plan, st);
        case VI_F16: return launch_product<__half>(p, plan, st);
        case VI_BF16: return launch_product<__nv_bfloat16>(p, plan, st);
        case VI_I32: return launch_product<int32_t>(p, plan, st);
        default: return launch_product<uint64_t>(p, plan, st);
    }
}

// The device is waited for first: the legacy default stream, on which the copy runs, does not wait for non-blocking streams.  Read
// and cleared in one step, so that a code that a product of another host thread records meanwhile is kept for the next call.
extern "C" int vi_int8_matmul_status(int* code) {
    VI_REQUIRE(code, "int8_matmul_status: null pointer");
    static std::mutex one;              // g_i8_taken is this call's until it is read
    std::lock_guard<std::mutex> lock(one);
    VI_CUDA(cudaDeviceSynchronize());
    k_int8_take_status<<<1, 1>>>();
    const int rc = vi::check_launch("k_int8_take_status");
    if (rc) return rc;
    VI_CUDA(cudaMemcpyFromSymbol(code, g_i8_taken, sizeof(int)));
    return VI_OK;
}

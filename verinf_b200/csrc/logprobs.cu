// What a row of logits says about the token that was given: its log probability, the entropy of the row, and the likeliest
// tokens.
//
// With c = log2(e) / T and a_j = (x_j - max) c:  S = sum 2^a_j, logprob = ln 2 (a_t - log2 S), entropy = ln 2 (log2 S -
// (sum 2^a_j a_j) / S), alternatives in the order of x (ties to the lowest index).  One pass: a thread keeps the maximum m of
// its entries, s = sum 2^a and w = sum 2^a a against that maximum, and rescales s and w when the maximum grows; two such
// triples join in the same way.  The sums are in fp32; a thread adds vocab / 128 terms or fewer
// (vocab / 64 of a row of 1024 packs or less), two by two.
//
// Alternatives without a second pass: a thread's packs (the entries of one 16-byte load) fall into four shares, and it keeps
// the largest entry of each share and the pack that first reached it.  The threads form 64 groups (32 for up to 16 alternatives:
// 4096 x 32000 bf16 with 5 57.0 -> 55.7 us), each with the best (value, pack) of its shares as key; a pack belongs to one share,
// so keys are distinct.  An entry that is among the `top` best lies in a share whose own key is at least the top-th largest group
// key: were it smaller, the `top` entries behind those keys would all come before it.  Only those shares, a few hundred entries
// of a row, are read again (from L2), what is not below the key is collected and ranked by counting.
//
// Bound by HBM where rows are many: 4096 x 32000 bf16 without a list 49 us, 5 us of start and then 6.0 TB/s; the list's instructions
// come on top.  Few rows are latency: a thread's rounds of loads (64 x 202045 fp16 in clusters of four: 25 packs a thread in seven
// rounds with one round ahead, 13.3 us, without a list 10.3), the joins of a block and of a cluster.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "../../include/verinf_b200.h"
#include "common.cuh"
#include "f32x2.cuh"
#include "launch.cuh"
#include "packs.cuh"
#include "umma.cuh"

namespace {

using namespace vf2;

constexpr int LP_MAX_TOP = 32, LP_GROUPS = 64, LP_CANDIDATES = 1024, LP_UNROLL = 4, LP_MAX_SPLIT = 8;
constexpr float LP_LOW = -3.402823466e38f;       // least finite value: a maximum starts here, so that -inf - max is -inf and not NaN
constexpr float LP_FAR = 1048576.0f;             // maxima of |m c| below 2^20 take the short form of a
constexpr float LP_CLAMP = -1.2676506e30f;       // -2^100: beside such a maximum (|m| < 2^40, as T <= 10^6) as good as -inf: 2^a = 0

// order of floats as unsigned numbers; -0 counts as 0
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
// larger value first, then the lower index
__device__ __forceinline__ uint64_t make_key(float x, uint32_t index) { return ((uint64_t)ordered(x) << 32) | (0xFFFFFFFFu - index); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {       // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// The entries of a 16-byte load: two at a time as fp32, the largest of them, -inf replaced by LP_CLAMP on demand.
template <typename T> struct Entries;
template <> struct Entries<float> {
    static constexpr int N = 4;
    using Raw = uint32_t;
    static constexpr uint32_t NOTHING = 0xFF800000u;       // a word of -inf
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ void two(const uint4& q, int i, float& a, float& b) {
        a = __uint_as_float(i ? q.z : q.x);
        b = __uint_as_float(i ? q.w : q.y);
    }
    static __device__ __forceinline__ float largest(const uint4& q) {
        return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    }
    static __device__ __forceinline__ void clamp_packed(uint4&) {}
    static __device__ __forceinline__ float clamp_one(float v) { return max_nan(v, LP_CLAMP); }
};
__device__ __forceinline__ uint32_t word(const uint4& q, int i) { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }
template <> struct Entries<__half> {
    static constexpr int N = 8;
    using Raw = uint16_t;
    static constexpr uint32_t NOTHING = 0xFC00FC00u;
    static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ __half2 as2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
    static __device__ __forceinline__ void two(const uint4& q, int i, float& a, float& b) {
        const float2 f = __half22float2(as2(word(q, i)));
        a = f.x;
        b = f.y;
    }
    static __device__ __forceinline__ float largest(const uint4& q) {
        const __half2 m = __hmax2(__hmax2(as2(q.x), as2(q.y)), __hmax2(as2(q.z), as2(q.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ void clamp_packed(uint4&) {}                                          // -2^100 is no fp16 number
    static __device__ __forceinline__ float clamp_one(float v) { return max_nan(v, LP_CLAMP); }
};
template <> struct Entries<__nv_bfloat16> {
    static constexpr int N = 8;
    using Raw = uint16_t;
    static constexpr uint32_t NOTHING = 0xFF80FF80u;
    static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat162 as2(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
    static __device__ __forceinline__ void two(const uint4& q, int i, float& a, float& b) {
        const uint32_t w = word(q, i);
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xFFFF0000u);
    }
    static __device__ __forceinline__ float largest(const uint4& q) {
        const __nv_bfloat162 m = __hmax2(__hmax2(as2(q.x), as2(q.y)), __hmax2(as2(q.z), as2(q.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ uint32_t clamp2(uint32_t w) {
        const __nv_bfloat162 low = __halves2bfloat162(__ushort_as_bfloat16(0xF180u), __ushort_as_bfloat16(0xF180u));     // -2^100
        const __nv_bfloat162 r = __hmax2_nan(as2(w), low);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ void clamp_packed(uint4& q) { q = {clamp2(q.x), clamp2(q.y), clamp2(q.z), clamp2(q.w)}; }
    static __device__ __forceinline__ float clamp_one(float v) { return v; }
};

struct Stat { float m, s, w; };      // max, sum 2^a, sum 2^a a

// a of an entry against a maximum.  Short form: x c - m c with one rounded m c, the same for all entries of a maximum, so that
// its rounding, at most 2^-4 where |m c| < 2^20, cancels between a_t and log2 S.  Elsewhere the difference comes first.
__device__ __forceinline__ bool is_near(float m, float c) { return fabsf(__fmul_rn(m, c)) < LP_FAR; }
__device__ __forceinline__ float arg_of(float x, float m, float c) { return is_near(m, c) ? __fmaf_rn(x, c, -__fmul_rn(m, c)) : (x - m) * c; }
// ln p of an entry.  Where the product with c could overflow though the difference over T does not, the difference comes first, of
// halves, which does not overflow either (a half that is not exact, of a subnormal number, has |m| >= 2^20 / c > 0.7 or an x
// below LP_CLAMP beside it, and does not count); no rounding makes a probability larger than one.
__device__ __forceinline__ float log_p(float x, const Stat& all, float c, float inv_t, float log_s) {
    const float ln2 = 0.6931471805599453f;
    const float v = is_near(all.m, c) && x > LP_CLAMP ? (arg_of(x, all.m, c) - log_s) * ln2 : (0.5f * x - 0.5f * all.m) * (2.0f * inv_t) - log_s * ln2;
    return fminf(v, 0.0f);
}
// what a grows by when the maximum goes from `from` to `to`: the rounded m c is the reference of a short form, the exact one of
// the others
__device__ __forceinline__ float shift_of(float from, float to, float c) {
    if (from == to) return 0.0f;
    const float mf = __fmul_rn(from, c), mt = __fmul_rn(to, c);
    if (is_near(from, c)) return is_near(to, c) ? mf - mt : __fmaf_rn(-to, c, mf);
    return is_near(to, c) ? __fmaf_rn(from, c, -mt) : (from - to) * c;
}
// the sums of a maximum, against a larger one
__device__ __forceinline__ void raise(Stat& t, float to, float c) {
    const float d = shift_of(t.m, to, c), f = ex2(d);
    t.w = f > 0.0f ? (t.w + t.s * d) * f : 0.0f;       // a vanishing side may have d = -inf: 0 * -inf stays out of the sum
    t.s *= f;
    t.m = to;
}

__device__ __forceinline__ float most_of(const float (&v)[LP_UNROLL]) {
    static_assert(LP_UNROLL == 4, "four shares");
    return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
}

// A row to a block, or, with split > 1, to a cluster of blocks that each take a share of its packs.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) k_token_logprobs(const T* __restrict__ logits, int64_t stride, int64_t vocab, const int64_t* __restrict__ tokens,
                                                               int top, float c, float inv_t, int split, float* __restrict__ logprob, float* __restrict__ entropy,
                                                               float* __restrict__ top_logprob, int64_t* __restrict__ top_token) {
    using E = Entries<T>;
    constexpr int N = E::N, WARPS = NT / 32;
    __shared__ Stat stats[WARPS];
    __shared__ __align__(16) uint64_t group[LP_GROUPS];
    __shared__ __align__(16) uint64_t cand[LP_CANDIDATES];
    __shared__ uint16_t flagged[LP_UNROLL * NT];
    __shared__ uint64_t best[LP_MAX_TOP];
    __shared__ uint64_t lists[LP_MAX_SPLIT][LP_MAX_TOP];
    __shared__ uint64_t limit;
    __shared__ int n_cand, n_flag;
    __shared__ Stat total;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)blockIdx.x % split;
    const int64_t row = blockIdx.x / (unsigned)split;
    const T* x = logits + row * stride;
    const int groups = top <= LP_GROUPS / 4 ? LP_GROUPS / 2 : LP_GROUPS, in_group = NT / groups;
    vi::await_inputs();
    const vpk::Row<typename E::Raw> packs(x, vocab);
    const int64_t p0 = packs.count * rank / split, p1 = packs.count * (rank + 1) / split;

    Stat st = {LP_LOW, 0.0f, 0.0f};
    // The packs of a thread fall into LP_UNROLL shares: the largest entry of each, and the first pack that reached it.
    float mine[LP_UNROLL];
    uint32_t mine_pack[LP_UNROLL];
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) { mine[u] = -CUDART_INF_F; mine_pack[u] = 0; }
    const int64_t inner1 = p1 < packs.whole1 ? p1 : packs.whole1;
    auto fetch = [&](uint4 (&q)[LP_UNROLL], int64_t base) {
        if (base >= packs.whole0 && base + (LP_UNROLL - 1) * NT < inner1) {
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u) q[u] = __ldg(packs.packs + base + u * NT);
        } else {                                  // packs beyond the share count as -inf
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u) {
                const int64_t p = base + u * NT;
                q[u] = {E::NOTHING, E::NOTHING, E::NOTHING, E::NOTHING};
                if (p < p1) q[u] = packs.load(p, E::NOTHING);
            }
        }
    };
    uint4 next[LP_UNROLL];
    fetch(next, p0 + tid);
    for (int64_t base = p0 + tid; base < p1; base += LP_UNROLL * NT) {
        uint4 q[LP_UNROLL];
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) q[u] = next[u];
        if (base + LP_UNROLL * NT < p1) fetch(next, base + LP_UNROLL * NT);
        float most = st.m;
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) {
            const float big = E::largest(q[u]);
            if (big > mine[u]) { mine[u] = big; mine_pack[u] = (uint32_t)(base + u * NT); }
            most = fmaxf(most, big);
        }
        if (most > st.m) raise(st, most, c);
        // with no entry above the least finite value yet, only a NaN or a row of such values would leave a trace
        const bool nothing = st.m == LP_LOW && most_of(mine) == -CUDART_INF_F;
        if (is_near(st.m, c) || nothing) {
            const float mc = nothing ? 0.0f : __fmul_rn(st.m, c);
            const uint64_t cc = pack2(c, c), neg = pack2(-mc, -mc);
            uint64_t s2 = pack2(st.s, 0.0f), w2 = pack2(st.w, 0.0f);
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u) {
                E::clamp_packed(q[u]);
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    float v0, v1, a0, a1;
                    E::two(q[u], i, v0, v1);
                    const uint64_t a2 = fma2(pack2(E::clamp_one(v0), E::clamp_one(v1)), cc, neg);
                    unpack2(a2, a0, a1);
                    const uint64_t f2 = pack2(ex2(a0), ex2(a1));
                    s2 = add2(s2, f2);
                    w2 = fma2(f2, a2, w2);
                }
            }
            float lo, hi;
            unpack2(s2, lo, hi);
            st.s = lo + hi;
            unpack2(w2, lo, hi);
            st.w = lo + hi;
        } else {
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u) {
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    float v[2];
                    E::two(q[u], i, v[0], v[1]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float a = (v[e] - st.m) * c, f = ex2(a);
                        st.s += f;
                        st.w += f * fmaxf(a, LP_LOW);           // a = -inf has f = 0
                    }
                }
            }
        }
    }
    vi::release_next();
    // the warp's sums against the warp's maximum
    {
        const float m = unordered(__reduce_max_sync(~0u, ordered(st.m)));
        raise(st, m, c);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            st.s += __shfl_xor_sync(~0u, st.s, o);
            st.w += __shfl_xor_sync(~0u, st.w, o);
        }
        if (lane == 0) stats[warp] = st;
    }
    uint64_t key[LP_UNROLL];
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) key[u] = mine[u] > -CUDART_INF_F ? make_key(mine[u], mine_pack[u]) : 0;      // 0: nothing finite here
    if (top) {
        uint64_t k = key[0];
#pragma unroll
        for (int u = 1; u < LP_UNROLL; ++u) k = key[u] > k ? key[u] : k;
        for (int o = 1; o < in_group; o <<= 1) {
            const uint64_t b = __shfl_xor_sync(~0u, k, o);
            k = b > k ? b : k;
        }
        if (tid % in_group == 0) group[tid / in_group] = k ? k : (uint64_t)(tid / in_group);      // distinct, and below every key
    }
    if (tid == 0) { n_cand = 0; n_flag = 0; }
    if (tid < LP_MAX_TOP) best[tid] = 0;
    __syncthreads();
    if (warp == 0) {
        Stat t = lane < WARPS ? stats[lane] : Stat{LP_LOW, 0.0f, 0.0f};
        const float m = unordered(__reduce_max_sync(~0u, ordered(t.m)));
        raise(t, m, c);
#pragma unroll
        for (int o = WARPS / 2; o; o >>= 1) {
            t.s += __shfl_xor_sync(~0u, t.s, o);
            t.w += __shfl_xor_sync(~0u, t.w, o);
        }
        if (lane == 0) total = t;
    }
    if (top && tid >= NT - groups) {             // rank among the groups
        const uint64_t k = group[tid - (NT - groups)];
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < groups; i += 2) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&group[i]);
            above += (o.x > k) + (o.y > k);
        }
        if (above == top - 1) limit = k;
    }
    __syncthreads();
    if (top) {
        const uint64_t lim = limit < LP_GROUPS ? 0 : limit;       // fewer groups than `top` have a key: every entry counts
        const float lim_value = lim ? unordered((uint32_t)(lim >> 32)) : LP_LOW;
        unsigned vote[LP_UNROLL];                 // shares that may hold some of the best
        int votes = 0;
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) {
            vote[u] = __ballot_sync(~0u, key[u] && key[u] >= lim);
            votes += __popc(vote[u]);
        }
        if (votes) {
            int at = 0;
            if (lane == 0) at = atomicAdd(&n_flag, votes);
            at = __shfl_sync(~0u, at, 0);
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u) {
                if (vote[u] >> lane & 1) flagged[at + __popc(vote[u] & ((1u << lane) - 1))] = (uint16_t)(tid + u * NT);
                at += __popc(vote[u]);
            }
        }
        __syncthreads();
        const unsigned per = (unsigned)((p1 - p0 + LP_UNROLL * NT - 1) / (LP_UNROLL * NT));
        const unsigned items = (unsigned)n_flag * per;                     // at most 4 NT shares of 2^31 / (4 NT) packs
        for (unsigned item = tid; item < items; item += NT) {              // their packs, one a thread
            const unsigned f = item / per, j = item - f * per;
            const int64_t p = p0 + flagged[f] + (int64_t)j * (LP_UNROLL * NT);
            if (p >= p1) continue;
            const uint4 q = packs.load(p, E::NOTHING);
            if (!(E::largest(q) >= lim_value)) continue;
            unsigned hits = 0;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                float v0, v1;
                E::two(q, i, v0, v1);
                hits |= (v0 >= lim_value ? 1u << (2 * i) : 0u) | (v1 >= lim_value ? 2u << (2 * i) : 0u);
            }
            while (hits) {
                const int64_t i = packs.first(p) + __ffs(hits) - 1;
                hits &= hits - 1;
                const float v = E::one(x + i);
                if (make_key(v, (uint32_t)p) >= lim) {                     // the same order as that of the group keys: value, then pack
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < LP_CANDIDATES) cand[at] = make_key(v, (uint32_t)i);
                }
            }
        }
        __syncthreads();
        const int nc = n_cand;
        if (nc <= LP_CANDIDATES) {
            for (int i = tid; i < nc; i += NT) {
                const uint64_t k = cand[i];
                int above = 0, j = 0;
#pragma unroll 4
                for (; j + 1 < nc; j += 2) {
                    const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&cand[j]);
                    above += (o.x > k) + (o.y > k);
                }
                if (j < nc) above += cand[j] > k;
                if (above < top) best[above] = k;
            }
        } else {
            // Shares made so that a few threads hold most of the large entries: one pass over the share for each alternative.
            const int64_t i0 = packs.first(p0) < 0 ? 0 : packs.first(p0), i1 = packs.first(p1) < vocab ? packs.first(p1) : vocab;
            uint64_t below = ~0ull;
            for (int j = 0; j < top && below; ++j) {
                uint64_t k = 0;
                for (int64_t i = i0 + tid; i < i1; i += NT) {
                    const float v = E::one(x + i);
                    const uint64_t kk = v > -CUDART_INF_F ? make_key(v, (uint32_t)i) : 0;
                    if (kk < below && kk > k) k = kk;
                }
                if (tid == 0) limit = 0;
                __syncthreads();
                atomicMax((unsigned long long*)&limit, (unsigned long long)k);
                __syncthreads();
                below = limit;
                if (tid == 0) best[j] = below;
                __syncthreads();
            }
        }
        __syncthreads();
    }
    Stat all = total;
    if (split > 1) {                              // the first block joins the cluster's sums and lists
        vumma::cluster_sync();
        if (rank == 0) {
            const uint32_t total_at = vumma::smem_u32(&total), best_at = vumma::smem_u32(best);
            Stat t = {LP_LOW, 0.0f, 0.0f};
            if (lane < split) {
                t.m = __uint_as_float(vumma::cluster_ld(total_at, lane));
                t.s = __uint_as_float(vumma::cluster_ld(total_at + 4, lane));
                t.w = __uint_as_float(vumma::cluster_ld(total_at + 8, lane));
            }
            const float m = unordered(__reduce_max_sync(~0u, ordered(t.m)));
            raise(t, m, c);
#pragma unroll
            for (int o = LP_MAX_SPLIT / 2; o; o >>= 1) {
                t.s += __shfl_xor_sync(~0u, t.s, o);
                t.w += __shfl_xor_sync(~0u, t.w, o);
            }
            all = {__shfl_sync(~0u, t.m, 0), __shfl_sync(~0u, t.s, 0), __shfl_sync(~0u, t.w, 0)};
            if (top) {
                static_assert(NT == 64 || NT == 128 || NT == 256, "a warp for each list of a cluster of NT / 32 blocks at most");
                uint64_t k = 0;
                if (warp < split) {
                    k = vumma::cluster_ld(best_at + 8 * lane, warp) | (uint64_t)vumma::cluster_ld(best_at + 8 * lane + 4, warp) << 32;
                    lists[warp][lane] = k;
                }
                __syncthreads();
                if (tid < LP_MAX_TOP) best[tid] = 0;
                __syncthreads();
                if (k) {                          // falling lists: how many of each come before this key
                    int above = lane;
                    for (int b = 0; b < split; ++b) {
                        if (b == warp) continue;
                        int n = 0;
#pragma unroll
                        for (int h = LP_MAX_TOP / 2; h; h >>= 1)
                            if (lists[b][n + h - 1] > k) n += h;
                        if (n == LP_MAX_TOP - 1 && lists[b][n] > k) ++n;
                        above += n;
                    }
                    if (above < top) best[above] = k;
                }
                __syncthreads();
            }
        }
        vumma::cluster_sync();                    // no block leaves while its sums and list are read
        if (rank != 0) return;
    }
    const bool bad = !(all.s <= CUDART_MAX_NORMAL_F), empty = all.s == 0.0f;       // NaN: an entry is NaN or +inf
    const float log_s = log2f(all.s);
    if (tid < top) {
        const uint64_t k = bad || empty ? 0 : best[tid];
        top_token[row * top + tid] = k ? (int64_t)(0xFFFFFFFFu - (uint32_t)k) : -1;
        top_logprob[row * top + tid] = bad ? CUDART_NAN_F : k ? log_p(unordered((uint32_t)(k >> 32)), all, c, inv_t, log_s) : -CUDART_INF_F;
    }
    if (tid == NT - 1) {
        const int64_t t = tokens[row];
        entropy[row] = bad ? CUDART_NAN_F : empty ? 0.0f : fmaxf((log_s - all.w / all.s) * 0.6931471805599453f, 0.0f);
        float lp = 0.0f;
        if (t >= vocab) lp = CUDART_NAN_F;
        else if (t >= 0) lp = bad ? CUDART_NAN_F : empty ? -CUDART_INF_F : log_p(E::one(x + t), all, c, inv_t, log_s);
        logprob[row] = lp;
    }
}

struct Plan { int threads, split; };      // split <= threads / 32

template <typename T, int NT>
int launch(const void* logits, int64_t rows, int64_t vocab, int64_t stride, const int64_t* tokens, int top, float c, float inv_t, float* logprob,
           float* entropy, float* top_logprob, int64_t* top_token, int split, cudaStream_t st) {
    // Clusters that are placed beside the blocks of the kernel before lie unevenly on the SMs: 64 x 202045 in clusters of four, called
    // one after the other, 17.6 us when set up early, 14.6 us when not.
    return vi::launch_early("k_token_logprobs", k_token_logprobs<T, NT>, dim3((unsigned)(rows * split)), dim3(NT), 0, split, split == 1, st, (const T*)logits, stride, vocab,
                            tokens, top, c, inv_t, split, logprob, entropy, top_logprob, top_token);
}

template <typename T>
int launch(const void* logits, int64_t rows, int64_t vocab, int64_t stride, const int64_t* tokens, int top, float c, float inv_t, float* logprob,
           float* entropy, float* top_logprob, int64_t* top_token, const Plan& plan, cudaStream_t st) {
    auto go = plan.threads == 64 ? launch<T, 64> : plan.threads == 128 ? launch<T, 128> : launch<T, 256>;
    return go(logits, rows, vocab, stride, tokens, top, c, inv_t, logprob, entropy, top_logprob, top_token, plan.split, st);
}

// Many rows: small blocks, whose ends (sums, list) hide behind other blocks' loads; 128 threads, for rows of up to 1024 packs
// 64 (us with 64 / 128 / 256 threads and 20 alternatives: 4096 x 32000 bf16 87 / 61 / 71, 4096 x 4000 20 / 24 / 42, 1000 x
// 32000 24 / 19 / 22).  Few rows: 256 threads, and while that gives no more than two blocks an SM, long rows go to clusters,
// down to 2000 packs a block (1 x 32000 fp32 on 1 / 2 / 4 / 8 blocks 7.6 / 7.2 / 6.8 / 7.2, 8 x 128000 bf16 14 / 11 / 8.7 /
// 8.3, 64 x 202048 fp16 23 / 17 / 14 / 16, 300 x 32000 bf16 11 / 16 / 22).
Plan make_plan(int64_t rows, int64_t packs) {
    if (rows >= 512) return {packs <= 1024 ? 64 : 128, 1};
    Plan p = {256, 1};
    while (p.split < LP_MAX_SPLIT && rows * p.split * 2 <= 2 * 148 && packs > p.split * 4000) p.split *= 2;
    return p;
}

}  // namespace

extern "C" int vi_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t stride, const int64_t* tokens, int top,
                                 double temperature, float* logprob, float* entropy, float* top_logprob, int64_t* top_token, void* stream) {
    VI_REQUIRE(dtype == VI_F32 || dtype == VI_F16 || dtype == VI_BF16, "token_logprobs: dtype must be VI_F32, VI_F16 or VI_BF16");
    VI_REQUIRE(rows >= 0 && vocab >= 1, "token_logprobs: rows must not be negative, vocab at least 1");
    VI_REQUIRE(rows <= 0x7FFFFFFF && vocab <= 0x7FFFFFFF, "token_logprobs: rows and vocab are limited to 2^31 - 1");
    VI_REQUIRE(top >= 0 && top <= LP_MAX_TOP, "token_logprobs: top must be 0 .. 32");
    VI_REQUIRE(temperature >= 1e-6 && temperature <= 1e6, "token_logprobs: temperature must be between 1e-6 and 1e6");
    if (rows == 0) return VI_OK;
    VI_REQUIRE(logits && tokens && logprob && entropy && (top == 0 || (top_logprob && top_token)), "token_logprobs: null pointer");
    VI_REQUIRE(((uintptr_t)logits) % (dtype == VI_F32 ? 4 : 2) == 0, "token_logprobs: logits are not aligned to their type");
    VI_REQUIRE(((uintptr_t)tokens | (uintptr_t)top_token) % 8 == 0 && ((uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_logprob) % 4 == 0,
               "token_logprobs: misaligned tokens or outputs");
    VI_REQUIRE(rows == 1 || stride >= 0, "token_logprobs: negative stride");
    cudaStream_t st = (cudaStream_t)stream;
    const float c = (float)(1.4426950408889634 / temperature), inv_t = (float)(1.0 / temperature);
    const Plan plan = make_plan(rows, vocab / (dtype == VI_F32 ? 4 : 8));
    if (dtype == VI_F32) return launch<float>(logits, rows, vocab, stride, tokens, top, c, inv_t, logprob, entropy, top_logprob, top_token, plan, st);
    if (dtype == VI_F16) return launch<__half>(logits, rows, vocab, stride, tokens, top, c, inv_t, logprob, entropy, top_logprob, top_token, plan, st);
    return launch<__nv_bfloat16>(logits, rows, vocab, stride, tokens, top, c, inv_t, logprob, entropy, top_logprob, top_token, plan, st);
}

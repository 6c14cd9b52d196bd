// What a row of logits says about the token that was given: its log probability, the entropy of the row, and the likeliest
// tokens.
//
// z_j = (x_j - max) / T, Z = sum e^z_j:  logprob = z_t - log Z,  entropy = log Z - (sum e^z_j z_j) / Z, alternatives in the
// order of x (ties to the lowest index).  One pass: a thread keeps the maximum m of its entries, s = sum e^((x - m) / T) and
// w = sum e^((x - m) / T) (x - m), and rescales s and w when its maximum grows; two such triples join in the same way.
//
// Alternatives without a second pass: each thread also keeps which pack (consecutive entries that one load brings) first
// reached its maximum.  The threads form 64 groups, each with the best (value, pack) of its threads as key; a pack belongs to
// one thread, so keys are distinct.  An entry that is among the `top` best lies in a thread whose own key is at least the
// top-th largest group key: were it smaller, the `top` entries behind those keys would all come before it.  Only those
// threads' entries, a handful, are read again (from L2), those not below the key are collected and ranked by counting.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "../../include/verinf_b200.h"
#include "common.cuh"

namespace {

constexpr int LP_MAX_TOP = 32, LP_GROUPS = 64, LP_CANDIDATES = 1024;
constexpr float LP_LOW = -3.402823466e38f;       // least finite value: a maximum starts here, so that -inf - max is -inf and not NaN

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// order of floats as unsigned numbers; -0 counts as 0
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
// larger value first, then the lower index
__device__ __forceinline__ uint64_t make_key(float x, uint32_t index) { return ((uint64_t)ordered(x) << 32) | (0xFFFFFFFFu - index); }

struct Stat { float m, s, w; };      // max, sum e^d, sum e^d d (d = x - m, not yet divided by T)

// 2^((x - m) c) with c = log2(e) / T
__device__ __forceinline__ float expo(float d, float c) { return exp2f(d * c); }

__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float c) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m - r.m, db = b.m - r.m, ea = expo(da, c), eb = expo(db, c);
    // an empty or vanishing side has e = 0; its difference may be -inf, and 0 * -inf must stay out of the sum
    r.s = a.s * ea + b.s * eb;
    r.w = (ea > 0.0f ? (a.w + a.s * da) * ea : 0.0f) + (eb > 0.0f ? (b.w + b.s * db) * eb : 0.0f);
    return r;
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

template <typename T, int VEC, int NT>
__global__ void __launch_bounds__(NT) k_token_logprobs(const T* __restrict__ logits, int64_t stride, int64_t vocab, const int64_t* __restrict__ tokens,
                                                       int top, float inv_t, float* __restrict__ logprob, float* __restrict__ entropy,
                                                       float* __restrict__ top_logprob, int64_t* __restrict__ top_token) {
    __shared__ Stat stats[NT / 32];
    __shared__ uint64_t group[LP_GROUPS];
    __shared__ uint64_t cand[LP_CANDIDATES];
    __shared__ uint64_t best[LP_MAX_TOP];
    __shared__ uint64_t limit;
    __shared__ int flagged[NT];
    __shared__ int n_cand, n_flag;
    __shared__ Stat total;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x;
    const T* x = logits + row * stride;
    const float c = 1.4426950408889634f * inv_t;
    const int64_t npack = (vocab + VEC - 1) / VEC;
    auto entry = [&](int64_t i) { return as_float(x[i]); };

    Stat st = {LP_LOW, 0.0f, 0.0f};
    float mine = -CUDART_INF_F;          // largest entry of this thread, and the first pack that reached it
    uint32_t mine_pack = 0;
    for (int64_t p = tid; p < npack; p += NT) {
        float v[VEC];
        if (p * VEC + VEC <= vocab) {
            const Pack<T, VEC> q = reinterpret_cast<const Pack<T, VEC>*>(x)[p];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = as_float(q.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = p * VEC + e < vocab ? entry(p * VEC + e) : -CUDART_INF_F;
        }
        float big = v[0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) big = fmaxf(big, v[e]);
        if (big > mine) { mine = big; mine_pack = (uint32_t)p; }
        if (big > st.m) {
            const float d = st.m - big, f = expo(d, c);
            st.w = f > 0.0f ? (st.w + st.s * d) * f : 0.0f;
            st.s *= f;
            st.m = big;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = v[e] - st.m, f = expo(d, c);
            st.s += f;
            st.w += f * fmaxf(d, LP_LOW);           // d = -inf has f = 0
        }
    }
    // sums of the block
    for (int o = 16; o; o >>= 1) {
        Stat b = {__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o), __shfl_xor_sync(~0u, st.w, o)};
        st = join(st, b, c);
    }
    if (lane == 0) stats[warp] = st;
    uint64_t key = mine > -CUDART_INF_F ? make_key(mine, mine_pack) : 0;      // 0: nothing finite here
    if (tid < LP_GROUPS) group[tid] = 0;
    if (tid == 0) { n_cand = 0; n_flag = 0; }
    __syncthreads();
    if (top) atomicMax((unsigned long long*)&group[tid % LP_GROUPS], (unsigned long long)key);
    if (warp == 0) {
        st = lane < NT / 32 ? stats[lane] : Stat{LP_LOW, 0.0f, 0.0f};
        for (int o = 16; o; o >>= 1) {
            Stat b = {__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o), __shfl_xor_sync(~0u, st.w, o)};
            st = join(st, b, c);
        }
        if (lane == 0) {
            total = st;
            const int64_t t = tokens[row];
            const bool bad = !(st.s <= CUDART_MAX_NORMAL_F), empty = st.s == 0.0f;      // NaN: an entry is NaN or +inf
            const float nan = CUDART_NAN_F, log_z = logf(st.s);
            entropy[row] = bad ? nan : empty ? 0.0f : log_z - inv_t * (st.w / st.s);
            float lp = 0.0f;
            if (t >= vocab) lp = nan;
            else if (t >= 0) lp = bad ? nan : empty ? -CUDART_INF_F : (entry(t) - st.m) * inv_t - log_z;
            logprob[row] = lp;
        }
    }
    if (!top) return;
    __syncthreads();
    const Stat all = total;
    const bool none = !(all.s <= CUDART_MAX_NORMAL_F) || all.s == 0.0f;
    if (!none) {
        if (tid < LP_GROUPS) {              // rank among the groups; a group without a key counts by its number
            const uint64_t k0 = group[tid];
            int rank = 0;
            for (int g = 0; g < LP_GROUPS; ++g) rank += group[g] > k0 || (group[g] == k0 && g < tid);
            if (rank == top - 1) limit = k0;
        }
        __syncthreads();
        const uint64_t lim = limit;
        if (key && key >= lim) flagged[atomicAdd(&n_flag, 1)] = tid;
        __syncthreads();
        const int nf = n_flag;
        for (int f = warp; f < nf; f += NT / 32) {
            for (int64_t p = flagged[f] + (int64_t)lane * NT; p < npack; p += 32 * (int64_t)NT) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int64_t i = p * VEC + e;
                    if (i >= vocab) break;
                    const float v = entry(i);
                    // the same order as that of the group keys: value, then pack
                    if (v > -CUDART_INF_F && make_key(v, (uint32_t)p) >= lim) {
                        const int at = atomicAdd(&n_cand, 1);
                        if (at < LP_CANDIDATES) cand[at] = make_key(v, (uint32_t)i);
                    }
                }
            }
        }
        __syncthreads();
        int nc = n_cand;
        if (tid < LP_MAX_TOP) best[tid] = 0;
        __syncthreads();
        if (nc <= LP_CANDIDATES) {
            for (int i = tid; i < nc; i += NT) {
                const uint64_t k0 = cand[i];
                int rank = 0;
                for (int j = 0; j < nc; ++j) rank += cand[j] > k0;
                if (rank < top) best[rank] = k0;
            }
        } else {
            // Rows made so that a few threads hold most of the large entries: one pass over the row for each alternative.
            uint64_t below = ~0ull;
            for (int j = 0; j < top && below; ++j) {
                uint64_t k0 = 0;
                for (int64_t i = tid; i < vocab; i += NT) {
                    const float v = entry(i);
                    const uint64_t kk = v > -CUDART_INF_F ? make_key(v, (uint32_t)i) : 0;
                    if (kk < below && kk > k0) k0 = kk;
                }
                if (tid == 0) limit = 0;
                __syncthreads();
                atomicMax((unsigned long long*)&limit, (unsigned long long)k0);
                __syncthreads();
                below = limit;
                if (tid == 0) best[j] = below;
                __syncthreads();
            }
        }
        __syncthreads();
    }
    if (tid < top) {
        const uint64_t k0 = none ? 0 : best[tid];
        const int64_t i = 0xFFFFFFFFu - (uint32_t)k0;
        const bool bad = !(all.s <= CUDART_MAX_NORMAL_F);
        top_token[row * top + tid] = k0 ? i : -1;
        top_logprob[row * top + tid] = bad ? CUDART_NAN_F : k0 ? (entry(i) - all.m) * inv_t - logf(all.s) : -CUDART_INF_F;
    }
}

template <typename T>
int launch(const void* logits, int64_t rows, int64_t vocab, int64_t stride, const int64_t* tokens, int top, float inv_t, float* logprob,
           float* entropy, float* top_logprob, int64_t* top_token, cudaStream_t st) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const bool wide = ((uintptr_t)logits) % 16 == 0 && (rows == 1 || (stride * (int64_t)sizeof(T)) % 16 == 0);
    const T* x = (const T*)logits;
    if (wide) k_token_logprobs<T, VEC, 256><<<(unsigned)rows, 256, 0, st>>>(x, stride, vocab, tokens, top, inv_t, logprob, entropy, top_logprob, top_token);
    else k_token_logprobs<T, 1, 256><<<(unsigned)rows, 256, 0, st>>>(x, stride, vocab, tokens, top, inv_t, logprob, entropy, top_logprob, top_token);
    return vi::check_launch("k_token_logprobs");
}

}  // namespace

extern "C" int vi_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t stride, const int64_t* tokens, int top,
                                 float temperature, float* logprob, float* entropy, float* top_logprob, int64_t* top_token, void* stream) {
    VI_REQUIRE(dtype == VI_F32 || dtype == VI_F16 || dtype == VI_BF16, "token_logprobs: dtype must be VI_F32, VI_F16 or VI_BF16");
    VI_REQUIRE(rows >= 0 && vocab >= 1, "token_logprobs: rows must not be negative, vocab at least 1");
    VI_REQUIRE(rows <= 0x7FFFFFFF && vocab <= 0x7FFFFFFF, "token_logprobs: rows and vocab are limited to 2^31 - 1");
    VI_REQUIRE(top >= 0 && top <= LP_MAX_TOP, "token_logprobs: top must be 0 .. 32");
    VI_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, "token_logprobs: temperature must be between 1e-6 and 1e6");
    if (rows == 0) return VI_OK;
    VI_REQUIRE(logits && tokens && logprob && entropy && (top == 0 || (top_logprob && top_token)), "token_logprobs: null pointer");
    VI_REQUIRE(((uintptr_t)logits) % (dtype == VI_F32 ? 4 : 2) == 0, "token_logprobs: logits are not aligned to their type");
    VI_REQUIRE(((uintptr_t)tokens | (uintptr_t)top_token) % 8 == 0 && ((uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_logprob) % 4 == 0,
               "token_logprobs: misaligned tokens or outputs");
    VI_REQUIRE(rows == 1 || stride >= 0, "token_logprobs: negative stride");
    cudaStream_t st = (cudaStream_t)stream;
    const float inv_t = 1.0f / temperature;
    if (dtype == VI_F32) return launch<float>(logits, rows, vocab, stride, tokens, top, inv_t, logprob, entropy, top_logprob, top_token, st);
    if (dtype == VI_F16) return launch<__half>(logits, rows, vocab, stride, tokens, top, inv_t, logprob, entropy, top_logprob, top_token, st);
    return launch<__nv_bfloat16>(logits, rows, vocab, stride, tokens, top, inv_t, logprob, entropy, top_logprob, top_token, st);
}

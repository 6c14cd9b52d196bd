// Rows that start anywhere, read as packs: 16-byte loads on the 16-byte grid.  Pack p of a row whose first entry is `head`
// entries behind the grid holds the entries p N - head .. p N - head + N - 1; those before whole0 or from whole1 on are shared
// with what lies around the row and are put together from the row's entries alone.
#pragma once
#include <cstdint>

namespace vpk {

// entries of size sizeof(Raw) from `first` on; places outside [0, len) keep what `fill` has there
template <typename Raw>
__device__ __noinline__ uint4 edge_pack(const Raw* x, int64_t first, int64_t len, uint32_t fill) {
    constexpr int IN_WORD = 4 / (int)sizeof(Raw);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = fill;
#pragma unroll
        for (int e = 0; e < IN_WORD; ++e) {
            const int64_t at = first + i * IN_WORD + e;
            if (at >= 0 && at < len) {
                const uint32_t keep = IN_WORD == 1 ? 0u : e ? 0x0000FFFFu : 0xFFFF0000u;
                w[i] = (w[i] & keep) | (uint32_t)x[at] << (16 * e);
            }
        }
    }
    return {w[0], w[1], w[2], w[3]};
}

template <typename Raw>
struct Row {
    static constexpr int N = 16 / (int)sizeof(Raw);
    const Raw* x;
    const uint4* packs;
    int64_t len;
    int head;
    int64_t count, whole0, whole1;      // packs, and those of the row alone: [whole0, whole1)
    __device__ __forceinline__ Row(const void* at, int64_t len_) : x((const Raw*)at), len(len_) {
        head = (int)(((uintptr_t)at & 15) / sizeof(Raw));
        packs = reinterpret_cast<const uint4*>((uintptr_t)at & ~(uintptr_t)15);
        count = (len + head + N - 1) / N;
        whole0 = head ? 1 : 0;
        whole1 = (len + head) / N;
    }
    __device__ __forceinline__ bool whole(int64_t p) const { return p >= whole0 && p < whole1; }
    __device__ __forceinline__ int64_t first(int64_t p) const { return p * N - head; }
    __device__ __forceinline__ uint4 load(int64_t p, uint32_t fill) const { return whole(p) ? __ldg(packs + p) : edge_pack(x, first(p), len, fill); }
};

}  // namespace vpk

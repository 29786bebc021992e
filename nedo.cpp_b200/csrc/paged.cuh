// paged.cuh -- device views of the paged KV cache and of a ragged batch over it
// (nedo_gpu_kv_cache / nedo_gpu_kv_batch in include/nedo_gpu.h), shared by the
// append, attention and page-selection kernels.
//
// Everything these kernels index with comes from device memory that the host
// cannot check (lengths, page ids), so every value is range-checked here before
// it is used: a bad one sets kErrArgument in the device status word and its
// sequence or page is left out.
#pragma once

#include "common.cuh"
#include "launch.h"

namespace nedo_gpu {

constexpr uint32_t kNone = 0xFFFFFFFFu;

struct PagedSeq {
    uint32_t t0;   // first token row
    uint32_t n;    // token rows (0: none, or the descriptor's values are out of range)
    uint32_t kv;   // tokens in the cache, the n new ones included
    // position of token row t0 + i; negative for the rows of a sequence with fewer
    // cached tokens than rows (padding: they see nothing and write nothing)
    __device__ __forceinline__ int pos(uint32_t i) const { return static_cast<int>(kv) - static_cast<int>(n - i); }
};

__device__ __forceinline__ void flag_argument(DeviceStatus* st) {
    if (st != nullptr) atomicOr(&st->flags, kErrArgument);
}

__device__ __forceinline__ PagedSeq load_seq(const PagedBatch& b, uint32_t s, DeviceStatus* st) {
    const uint32_t a = b.q_start[s], z = b.q_start[s + 1], kv = b.kv_len[s];
    if (a > z || z > b.tokens || z - a > b.max_q_len || kv > b.max_kv_len) {
        flag_argument(st);
        return PagedSeq{0u, 0u, 0u};
    }
    return PagedSeq{a, z - a, kv};
}

// The sequence that holds token row t (the last one starting at or before it), or
// kNone for a row behind the last sequence or before the first.
__device__ __forceinline__ uint32_t seq_of_token(const PagedBatch& b, uint32_t t) {
    // one row per sequence, as in decoding: no search
    if (t < b.seqs && b.q_start[t] == t && b.q_start[t + 1u] == t + 1u) return t;
    uint32_t lo = 0, hi = b.seqs + 1u;  // first index in [0, seqs] whose start is above t
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (b.q_start[mid] > t) hi = mid;
        else lo = mid + 1u;
    }
    return lo == 0u || lo > b.seqs ? kNone : lo - 1u;
}

// Page id of logical page `i` of sequence s, or kNone (flagged) when the id is
// not a page of the cache.
__device__ __forceinline__ uint32_t load_page(const PagedBatch& b, const PagedKv& kv, uint32_t s, uint32_t i,
                                              DeviceStatus* st) {
    const uint32_t p = b.table[static_cast<size_t>(s) * b.max_pages + i];
    if (p >= kv.num_pages) {
        flag_argument(st);
        return kNone;
    }
    return p;
}

// First key position that a query at position p sees (window 0: no limit).
__device__ __forceinline__ uint32_t first_key(int p, uint32_t window) {
    return window != 0u && p >= static_cast<int>(window) ? static_cast<uint32_t>(p) + 1u - window : 0u;
}

__device__ __forceinline__ float kv_float(float v) { return v; }
__device__ __forceinline__ float kv_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T to_kv(float v);
template <>
__device__ __forceinline__ float to_kv<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half to_kv<__half>(float v) { return __float2half_rn(v); }

}  // namespace nedo_gpu

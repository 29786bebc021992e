// paged_q4.cuh -- pages of a Q4_0 cache: blocks of 32 channels of a token, 4-bit numbers n in
// 0..15 and an fp16 scale d for the values d (n - 8).  A page holds, for one KV head, the numbers of
// all its tokens, [page_size][head_dim / 8] words, and behind them the scales,
// [head_dim / 32][page_size]: as many bytes as GGUF's 18-byte blocks, but every copy of 16 tokens is
// whole 16-byte pieces.  In a word of channels 8 w .. 8 w + 7 the even ones are the low half's four
// numbers and the odd ones the high half's, so that one mask takes two neighbouring channels to the
// halves of an fp16 pair.
//
// Scales that the append writes have eight significant bits: n - 8 has three and a sign (and -8), so
// d (n - 8) is an fp16 number, and the attention over a Q4_0 cache is that over an F16 cache with
// these values.  Other scales give the product rounded to fp16.
#pragma once

#include "paged.cuh"

namespace nedo_gpu {

// Bytes of a page of one KV head, and where its scales begin.
__host__ __device__ __forceinline__ uint32_t q4_scales_at(const PagedKv& kv) { return kv.page_size * (kv.head_dim / 2u); }
__host__ __device__ __forceinline__ uint32_t q4_head_bytes(const PagedKv& kv) {
    return kv.page_size * (kv.head_dim / 32u) * 18u;
}

// The four pairs of a word as n - 8: channels (0, 1), (2, 3), (4, 5), (6, 7) of its eight.  The number
// goes into the low bits of 1024, or above them as 16 n, from where a sum or a product and a sum,
// exact, take it; the shift serves two pairs.
__device__ __forceinline__ void q4_pairs(uint32_t w, __half2 (&n)[4]) {
    const __half2 one = __halves2half2(__ushort_as_half(0xE408), __ushort_as_half(0xE408));       // -1032
    const __half2 sixteenth = __halves2half2(__ushort_as_half(0x2C00), __ushort_as_half(0x2C00));  // 1/16
    const __half2 high = __halves2half2(__ushort_as_half(0xD480), __ushort_as_half(0xD480));      // -72
    auto half2 = [](uint32_t x) { return *reinterpret_cast<__half2*>(&x); };
    const uint32_t v = w >> 8;
    n[0] = __hadd2(half2(lop_and_or(w, 0x000F000Fu, 0x64006400u)), one);
    n[1] = __hfma2(half2(lop_and_or(w, 0x00F000F0u, 0x64006400u)), sixteenth, high);
    n[2] = __hadd2(half2(lop_and_or(v, 0x000F000Fu, 0x64006400u)), one);
    n[3] = __hfma2(half2(lop_and_or(v, 0x00F000F0u, 0x64006400u)), sixteenth, high);
}

// The scale of channel d of a token in slot `slot` of a page and head at `at`.
__device__ __forceinline__ __half q4_scale(const PagedKv& kv, const uint8_t* at, uint32_t slot, uint32_t d) {
    return reinterpret_cast<const __half*>(at + q4_scales_at(kv))[(d >> 5) * kv.page_size + slot];
}

// Channel d of a token in slot `slot` of a page and head at `at`.
__device__ __forceinline__ float q4_value(const PagedKv& kv, const uint8_t* at, uint32_t slot, uint32_t d) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(at + slot * (kv.head_dim / 2u) + (d >> 3) * 4u);
    const int n = static_cast<int>(w >> ((d & 1u) * 16u + ((d >> 1) & 3u) * 4u) & 15u) - 8;
    return __half2float(__hmul(q4_scale(kv, at, slot, d), __int2half_rn(n)));
}

}  // namespace nedo_gpu

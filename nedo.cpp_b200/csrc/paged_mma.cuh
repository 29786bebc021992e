// paged_mma.cuh -- fp16 tensor-core pieces of the attention kernels: asynchronous
// copies, fragment loads, the split of an fp32 factor into two fp16 halves.
#pragma once

#include "common.cuh"

namespace nedo_gpu {

constexpr float kUp = 14.f;  // exponent by which the softmax weights are taken up before they are split

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// A pair of numbers as two fp16 halves each, x = hi + 2^-11 lo.  Below 2^15, as the kernels scale
// them, they keep 22 bits down to 2^-14, and 2^-36 below (a low half that is not taken up would leave
// 2^-25, which is what an unscaled softmax weight of 2^-39 is: not nothing next to a large value).
constexpr int kLowBits = 11;
constexpr float kLowDown = 1.f / (1 << kLowBits);
__device__ __forceinline__ void split(float2 x, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __float22half2_rn(x);
    const float2 f = __half22float2(h), up = make_float2(1 << kLowBits, 1 << kLowBits);
    *hi = pack(h);
    *lo = pack(__float22half2_rn(__fmul2_rn(__fadd2_rn(x, make_float2(-f.x, -f.y)), up)));
}
__device__ __forceinline__ void split(float x, float y, uint32_t* hi, uint32_t* lo) { split(make_float2(x, y), hi, lo); }
// Sums from low halves, on which those from high halves can go.
__device__ __forceinline__ void low_down(float (&c)[4]) {
    const float2 d = make_float2(kLowDown, kLowDown);
    const float2 x = __fmul2_rn(make_float2(c[0], c[1]), d), y = __fmul2_rn(make_float2(c[2], c[3]), d);
    c[0] = x.x;
    c[1] = x.y;
    c[2] = y.x;
    c[3] = y.y;
}

// The power of two that takes a row's largest magnitude to [2^13, 2^14), where the low
// half of its fp16 split is a normal number (0 for zero, infinite and NaN rows).
__device__ __forceinline__ int up_exponent(float big) {
    return big > 0.f && big < INFINITY ? min(126, 13 + 127 - static_cast<int>(__float_as_uint(big) >> 23)) : 0;
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }  // -126 <= e <= 127

// 2^x; results below 2^-126 are zero.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace nedo_gpu

// kv_append.cuh -- what the append kernels share (kv_append.cu: F16 and F32 caches, kv_append4.cu:
// Q4_0 caches): the rotation in 32 bits.
#pragma once

#include "paged.cuh"

namespace nedo_gpu {

// Cosine and sine of position p's rotation.
__device__ __forceinline__ float2 rotation(int p, double turns) {
    double turn = static_cast<double>(p) * turns;
    turn -= rint(turn);
    // what the fraction loses in 32 bits turns the result by the rest of the angle
    const float f = static_cast<float>(turn), rest = static_cast<float>((turn - f) * 6.283185307179586);
    float c, s;
    sincospif(2.f * f, &s, &c);
    return make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
}
__device__ __forceinline__ void rotate4(float4& x, float4& y, const float2* c) {
    const float4 u = x, w = y;
    x = make_float4(u.x * c[0].x - w.x * c[0].y, u.y * c[1].x - w.y * c[1].y, u.z * c[2].x - w.z * c[2].y,
                    u.w * c[3].x - w.w * c[3].y);
    y = make_float4(u.x * c[0].y + w.x * c[0].x, u.y * c[1].y + w.y * c[1].x, u.z * c[2].y + w.z * c[2].x,
                    u.w * c[3].y + w.w * c[3].x);
}
__device__ __forceinline__ float4 min4(const float4& a, const float4& b) {
    return make_float4(fminf(a.x, b.x), fminf(a.y, b.y), fminf(a.z, b.z), fminf(a.w, b.w));
}
__device__ __forceinline__ float4 max4(const float4& a, const float4& b) {
    return make_float4(fmaxf(a.x, b.x), fmaxf(a.y, b.y), fmaxf(a.z, b.z), fmaxf(a.w, b.w));
}

cudaError_t launch_kv_append4(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* qkv, double theta,
                              float* q_out, DeviceStatus* st, cudaStream_t stream);

}  // namespace nedo_gpu

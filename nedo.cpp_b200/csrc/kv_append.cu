// kv_append.cu -- the new tokens' keys and values into a paged cache, with the
// position rotation of queries and keys applied on the way (the RoPE and
// cache-write steps of src/model.cpp:218-225 and src/kernels.cpp:93-105, for a
// ragged batch over pages).
//
// Token row t of sequence s stands at position p = kv_len[s] - (q_start[s+1] - t).
// Channel pair (i, i + hd/2) of a query or key head turns by p * theta^(-2i/hd).
// The angle is formed in 64 bits, as a fraction of a turn: p * frequency loses
// nothing that matters at any position (32 bits are 1e-3 of a turn off at position
// 10^5), and the sine and cosine of the remaining fraction are taken in 32 bits.
#include "paged.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kAppendThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(PagedKv kv, PagedBatch b, uint32_t heads,
                                                                   const float* __restrict__ qkv, bool rotate, double log2_theta,
                                                                   float* __restrict__ q_out, DeviceStatus* st) {
    __shared__ float2 cs[128];
    const uint32_t t = blockIdx.x;
    const uint32_t s = seq_of_token(b, t);
    if (s == kNone) return;
    const PagedSeq sq = load_seq(b, s, st);
    if (sq.n == 0u) return;
    const int p = sq.pos(t - sq.t0);
    if (p < 0) return;
    const uint32_t page = load_page(b, kv, s, static_cast<uint32_t>(p) >> kv.page_shift, st);
    if (page == kNone) return;
    const uint32_t hd = kv.head_dim, half = hd / 2u;
    for (uint32_t i = threadIdx.x; i < half; i += kAppendThreads) {
        float2 c = make_float2(1.f, 0.f);
        if (rotate) {
            double turn = static_cast<double>(p) * exp2(-2.0 * i / hd * log2_theta) * 0.15915494309189535;
            turn -= rint(turn);
            sincospif(2.f * static_cast<float>(turn), &c.y, &c.x);
        }
        cs[i] = c;
    }
    __syncthreads();
    const float* row = qkv + static_cast<size_t>(t) * (heads + 2u * kv.kv_heads) * hd;
    const uint32_t slot = static_cast<uint32_t>(p) & (kv.page_size - 1u);
    for (uint32_t i = threadIdx.x; i < (heads + kv.kv_heads) * half; i += kAppendThreads) {
        const uint32_t h = i / half, d = i - h * half;
        const float x = row[h * hd + d], y = row[h * hd + d + half];
        const float2 c = cs[d];
        const float x1 = x * c.x - y * c.y, y1 = x * c.y + y * c.x;
        if (h < heads) {
            float* o = q_out + (static_cast<size_t>(t) * heads + h) * hd + d;
            o[0] = x1;
            o[half] = y1;
        } else {
            T* o = static_cast<T*>(kv.k) +
                   ((static_cast<size_t>(page) * kv.kv_heads + (h - heads)) * kv.page_size + slot) * hd + d;
            o[0] = to_kv<T>(x1);
            o[half] = to_kv<T>(y1);
        }
    }
    for (uint32_t i = threadIdx.x; i < kv.kv_heads * hd; i += kAppendThreads) {
        const uint32_t h = i / hd, d = i - h * hd;
        static_cast<T*>(kv.v)[((static_cast<size_t>(page) * kv.kv_heads + h) * kv.page_size + slot) * hd + d] =
            to_kv<T>(row[(heads + kv.kv_heads) * hd + i]);
    }
}

// Channel-wise minimum and maximum of a page's stored keys, per KV head: one CTA
// for each page that this call writes and each KV head.  A page whose first slot
// is written begins anew.  fminf / fmaxf leave NaN keys out.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) kv_bounds_kernel(PagedKv kv, PagedBatch b, uint32_t segs) {
    const uint32_t h = blockIdx.x % kv.kv_heads, i = blockIdx.x / kv.kv_heads, s = i / segs, seg = i % segs;
    const PagedSeq sq = load_seq(b, s, nullptr);
    const uint32_t fresh = sq.n < sq.kv ? sq.n : sq.kv;  // rows that are tokens
    if (fresh == 0u) return;
    const uint32_t begin = sq.kv - fresh, lp = (begin >> kv.page_shift) + seg;
    const uint32_t first = lp << kv.page_shift;
    if (first >= sq.kv) return;
    const uint32_t page = load_page(b, kv, s, lp, nullptr);
    if (page == kNone) return;
    const uint32_t j0 = first < begin ? begin - first : 0u;
    const uint32_t j1 = sq.kv - first < kv.page_size ? sq.kv - first : kv.page_size;
    const uint32_t hd = kv.head_dim;
    const T* k = static_cast<const T*>(kv.k) + (static_cast<size_t>(page) * kv.kv_heads + h) * kv.page_size * hd;
    T* bo = static_cast<T*>(kv.bounds) + (static_cast<size_t>(page) * kv.kv_heads + h) * 2u * hd;
    for (uint32_t d = threadIdx.x; d < hd; d += kAppendThreads) {
        float lo = j0 == 0u ? INFINITY : kv_float(bo[d]), hi = j0 == 0u ? -INFINITY : kv_float(bo[hd + d]);
        for (uint32_t j = j0; j < j1; ++j) {
            const float v = kv_float(k[static_cast<size_t>(j) * hd + d]);
            lo = fminf(lo, v);
            hi = fmaxf(hi, v);
        }
        bo[d] = to_kv<T>(lo);
        bo[hd + d] = to_kv<T>(hi);
    }
}

template <typename T>
cudaError_t append(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* qkv, bool rotate,
                   double log2_theta, float* q_out, DeviceStatus* st, cudaStream_t stream) {
    kv_append_kernel<T><<<b.tokens, kAppendThreads, 0, stream>>>(kv, b, heads, qkv, rotate, log2_theta, q_out, st);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || kv.bounds == nullptr) return e;
    const uint32_t segs = (b.max_q_len + kv.page_size - 2u) / kv.page_size + 1u;
    kv_bounds_kernel<T><<<b.seqs * segs * kv.kv_heads, kAppendThreads, 0, stream>>>(kv, b, segs);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_append(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* qkv, double theta,
                             float* q_out, DeviceStatus* st, cudaStream_t stream) {
    const bool rotate = theta > 0.0;
    const double l = rotate ? log2(theta) : 0.0;
    return kv.type == kF16 ? append<__half>(kv, b, heads, qkv, rotate, l, q_out, st, stream)
                           : append<float>(kv, b, heads, qkv, rotate, l, q_out, st, stream);
}

}  // namespace nedo_gpu

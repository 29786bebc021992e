// block_select.cu -- which pages of the cache a query token looks at: for each
// token and KV head, the page that holds the token itself and the picks - 1 others
// whose key bounds allow the largest scores.
//
//   score_b = sum_d (hi_bd * sum_g max(q_gd, 0) + lo_bd * sum_g min(q_gd, 0))
//
// over the KV head's query heads g bounds sum_g q_g.k from above for every key k
// of page b.  The sums are in 64 bits, so that the order of two pages is that of
// their scores and not of rounding; equal scores: the lower page first; NaN below
// every number.
#include "paged.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kThreads = 256;

// Order-preserving 64-bit key of a score (never 0; 0 marks "not there").
__device__ __forceinline__ uint64_t score_key(double v) {
    if (v == 0.0) v = 0.0;  // one key for both zeros
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
    if (v != v) return 1ull;
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) block_select_kernel(PagedKv kv, PagedBatch b, uint32_t heads,
                                                                const float* __restrict__ q, uint32_t picks,
                                                                uint32_t* __restrict__ blocks, DeviceStatus* st) {
    extern __shared__ __align__(16) uint64_t key[];
    __shared__ double up[256], down[256];
    __shared__ uint32_t hist[256];
    __shared__ uint32_t sh_bin, sh_left, sh_count[2][kThreads / 32], sh_base[2];
    const uint32_t t = blockIdx.x / kv.kv_heads, kh = blockIdx.x % kv.kv_heads, tid = threadIdx.x;
    const uint32_t warp = tid >> 5, lane = tid & 31u, hd = kv.head_dim, group = heads / kv.kv_heads;
    const uint32_t s = seq_of_token(b, t);
    if (s == kNone) return;
    const PagedSeq sq = load_seq(b, s, st);
    if (sq.n == 0u) return;
    const int p = sq.pos(t - sq.t0);
    uint32_t* out = blocks + (static_cast<size_t>(t) * kv.kv_heads + kh) * picks;
    const uint32_t n = p < 0 ? 0u : (static_cast<uint32_t>(p) >> kv.page_shift) + 1u;  // pages the token sees
    if (n <= picks) {  // all of them
        for (uint32_t i = tid; i < picks; i += kThreads) out[i] = i < n ? i : kNone;
        return;
    }
    for (uint32_t d = tid; d < hd; d += kThreads) {
        double u = 0.0, w = 0.0;
        for (uint32_t g = 0; g < group; ++g) {
            const double x = q[(static_cast<size_t>(t) * heads + kh * group + g) * hd + d];
            if (x < 0.0) w += x;
            else u += x;  // NaN too
        }
        up[d] = u;
        down[d] = w;
    }
    __syncthreads();
    for (uint32_t i = warp; i < n; i += kThreads / 32u) {
        uint64_t k = ~0ull;  // the token's own page
        if (i + 1u < n) {
            const uint32_t page = load_page(b, kv, s, i, st);
            double v = 0.0;
            if (page != kNone) {
                const T* lo = static_cast<const T*>(kv.bounds) + (static_cast<size_t>(page) * kv.kv_heads + kh) * 2u * hd;
                for (uint32_t d = lane; d < hd; d += 32u)
                    v += up[d] * static_cast<double>(kv_float(lo[hd + d])) + down[d] * static_cast<double>(kv_float(lo[d]));
            }
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
            k = page != kNone ? score_key(v) : 0ull;
        }
        if (lane == 0) key[i] = k;
    }
    __syncthreads();
    // the picks-th largest key, eight bits at a time
    uint64_t prefix = 0;
    uint32_t left = picks;  // still to be found among the keys that share `prefix`
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (uint32_t i = tid; i < 256u; i += kThreads) hist[i] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += kThreads)
            if (shift == 56 || (key[i] >> (shift + 8)) == (prefix >> (shift + 8)))
                atomicAdd(&hist[(key[i] >> shift) & 255u], 1u);
        __syncthreads();
        if (tid == 0) {
            uint32_t sum = 0, bin = 255;
            for (;; --bin) {
                if (sum + hist[bin] >= left || bin == 0u) break;
                sum += hist[bin];
            }
            sh_bin = bin;
            sh_left = left - sum;
        }
        __syncthreads();
        prefix |= static_cast<uint64_t>(sh_bin) << shift;
        left = sh_left;
        __syncthreads();
    }
    // in page order: the keys above it, and the first `left` that equal it
    if (tid < 2u) sh_base[tid] = 0;
    __syncthreads();
    for (uint32_t i0 = 0; i0 < n; i0 += kThreads) {
        const uint64_t k = i0 + tid < n ? key[i0 + tid] : 0ull;
        const bool in = i0 + tid < n, above = in && k > prefix, same = in && k == prefix;
        const uint32_t ma = __ballot_sync(0xFFFFFFFFu, above), ms = __ballot_sync(0xFFFFFFFFu, same);
        if (lane == 0) {
            sh_count[0][warp] = __popc(ma);
            sh_count[1][warp] = __popc(ms);
        }
        __syncthreads();
        uint32_t ca = sh_base[0], cs = sh_base[1];
        for (uint32_t w = 0; w < warp; ++w) {
            ca += sh_count[0][w];
            cs += sh_count[1][w];
        }
        const uint32_t below = (1u << lane) - 1u;
        ca += __popc(ma & below);
        cs += __popc(ms & below);
        const uint32_t at = ca + min(cs, left);
        if (above || (same && cs < left)) out[at] = i0 + tid;
        __syncthreads();
        if (tid == 0) {
            for (uint32_t w = 0; w < kThreads / 32u; ++w) {
                sh_base[0] += sh_count[0][w];
                sh_base[1] += sh_count[1][w];
            }
        }
        __syncthreads();
    }
}

}  // namespace

cudaError_t launch_block_select(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* q, uint32_t picks,
                                uint32_t* blocks, DeviceStatus* st, cudaStream_t stream) {
    const size_t smem = ((static_cast<size_t>(b.max_kv_len) + kv.page_size - 1u) >> kv.page_shift) * sizeof(uint64_t) + 16u;
    auto* kernel = kv.type == kF16 ? block_select_kernel<__half> : block_select_kernel<float>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    kernel<<<b.tokens * kv.kv_heads, kThreads, smem, stream>>>(kv, b, heads, q, picks, blocks, st);
    return cudaGetLastError();
}

}  // namespace nedo_gpu

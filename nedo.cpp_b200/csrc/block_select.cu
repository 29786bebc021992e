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
//
// Bound by reading the pages' bounds (4 hd bytes of an F16 cache per page and KV head).
// A cluster of CTAs takes one token and KV head, its warps eight pages at a time with all
// their loads in flight; the halves of a page's bounds lie next to each other, so a lane
// takes 16 bytes of them with its own factors in registers.  The bounds go into 64 bits by
// moving their bits (value * 2^-1008, or 2^-896 from fp32, exact down to the subnormals)
// instead of by the conversion unit.  The scores' order-preserving keys go to the first CTA's
// shared memory, which finds the threshold eight bits at a time below the bits that all keys
// share and writes the pages above it in order.
#include <algorithm>

#include "paged.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32u;
constexpr uint32_t kGroup = 8;  // pages a warp scores at once

// Order-preserving 64-bit key of a score: 0 is kept for "no page", NaN is 1.
__device__ __forceinline__ uint64_t score_key(double v) {
    if (v == 0.0) v = 0.0;  // one key for both zeros
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
    if (v != v) return 1ull;
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A 64-bit store at `addr` of the first CTA's shared memory.
__device__ __forceinline__ void store_first(uint32_t addr, uint64_t v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(addr));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(v) : "memory");
}

// The values of a 16-byte piece of the bounds, times 2^-1008 (fp16) or 2^-896 (fp32).
// An infinity or NaN comes out as a number: the caller looks for those first.
template <typename T>
struct Piece;
template <>
struct Piece<__half> {
    static constexpr uint32_t kCount = 8;
    static __device__ __forceinline__ double value(const uint4& x, uint32_t i) {
        const uint32_t w = i < 2u ? x.x : i < 4u ? x.y : i < 6u ? x.z : x.w;
        // sign to bit 31, exponent and mantissa to bits 24..10 of the upper word
        const int up = static_cast<int>((i & 1u) ? w : w << 16) >> 6;
        return __hiloint2double(static_cast<int>(static_cast<uint32_t>(up) & 0x81FFFC00u), 0);
    }
    static __device__ __forceinline__ double exact(const uint4& x, uint32_t i) {  // any value
        const uint32_t w = i < 2u ? x.x : i < 4u ? x.y : i < 6u ? x.z : x.w;
        return static_cast<double>(half_bits_to_float((i & 1u) ? w >> 16 : w)) * __hiloint2double(15 << 20, 0);
    }
    // nonzero in kOdd: an infinity or NaN among them (the exponent's carry)
    static constexpr uint32_t kOdd = 0x80008000u;
    static __device__ __forceinline__ uint32_t odd(const uint4& x) {
        auto carry = [](uint32_t w) { return (w & 0x7C007C00u) + 0x04000400u; };
        return carry(x.x) | carry(x.y) | carry(x.z) | carry(x.w);
    }
};
template <>
struct Piece<float> {
    static constexpr uint32_t kCount = 4;
    static __device__ __forceinline__ double value(const uint4& x, uint32_t i) {
        const uint32_t u = i == 0u ? x.x : i == 1u ? x.y : i == 2u ? x.z : x.w;
        return __hiloint2double(static_cast<int>((u & 0x80000000u) | ((u & 0x7FFFFFFFu) >> 3)), static_cast<int>(u << 29));
    }
    static __device__ __forceinline__ double exact(const uint4& x, uint32_t i) {
        const uint32_t u = i == 0u ? x.x : i == 1u ? x.y : i == 2u ? x.z : x.w;
        return static_cast<double>(__uint_as_float(u)) * __hiloint2double(127 << 20, 0);
    }
    static constexpr uint32_t kOdd = 0x80000000u;
    static __device__ __forceinline__ uint32_t odd(const uint4& x) {
        auto carry = [](uint32_t u) { return (u & 0x7F800000u) + 0x00800000u; };
        return carry(x.x) | carry(x.y) | carry(x.z) | carry(x.w);
    }
};

__device__ __forceinline__ double exchange(double a, double b, bool up, uint32_t mask) {
    const double keep = up ? b : a, send = up ? a : b;
    return keep + __shfl_xor_sync(0xFFFFFFFFu, send, mask);
}

// Inclusive sum over the CTA's threads, in thread order (and the CTA's total).
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t* total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    for (uint32_t o = 1; o < 32u; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += x;
    }
    __syncthreads();
    if (lane == 31u) warp_sums[warp] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    *total = all;
    return v + before;
}

// PIECES: 16-byte pieces of a page's bounds per lane.
template <typename T, uint32_t PIECES>
__global__ void __launch_bounds__(kThreads) block_select_kernel(PagedKv kv, PagedBatch b, uint32_t heads,
                                                                const float* __restrict__ q, uint32_t picks,
                                                                uint32_t* __restrict__ blocks, uint32_t cluster,
                                                                DeviceStatus* st) {
    using P = Piece<T>;
    extern __shared__ __align__(16) uint64_t key[];
    __shared__ uint32_t hist[256], warp_sums[kWarps], found[2];
    __shared__ uint64_t masks[2][kWarps];
    const uint32_t unit = blockIdx.x / cluster, rank = cluster_rank();
    const uint32_t t = unit / kv.kv_heads, kh = unit % kv.kv_heads, tid = threadIdx.x;
    const uint32_t warp = tid >> 5, lane = tid & 31u, hd = kv.head_dim, group = heads / kv.kv_heads;
    const uint32_t s = seq_of_token(b, t);
    if (s == kNone) return;
    const PagedSeq sq = load_seq(b, s, st);
    if (sq.n == 0u) return;
    const int p = sq.pos(t - sq.t0);
    uint32_t* out = blocks + (static_cast<size_t>(t) * kv.kv_heads + kh) * picks;
    const uint32_t n = p < 0 ? 0u : (static_cast<uint32_t>(p) >> kv.page_shift) + 1u;  // pages the token sees
    if (n <= picks) {  // all of them
        if (rank == 0u)
            for (uint32_t i = tid; i < picks; i += kThreads) out[i] = i < n ? i : kNone;
        return;
    }
    cluster_arrive();  // the first CTA runs before anything is stored into its memory
    // this lane's factors: of its pieces of the bounds (lowest values first, then highest)
    const uint32_t half_pieces = hd / P::kCount;
    double f[PIECES][P::kCount];
#pragma unroll
    for (uint32_t i = 0; i < PIECES; ++i) {
        const uint32_t piece = lane + 32u * i;
#pragma unroll
        for (uint32_t e = 0; e < P::kCount; ++e) {
            double x = 0.0;
            if (piece < 2u * half_pieces) {
                const bool high = piece >= half_pieces;
                const uint32_t d = (high ? piece - half_pieces : piece) * P::kCount + e;
                for (uint32_t g = 0; g < group; ++g) {
                    const double y = q[(static_cast<size_t>(t) * heads + kh * group + g) * hd + d];
                    if (!(y < 0.0) == high) x += y;  // NaN to the highest
                }
            }
            f[i][e] = x * __hiloint2double((1023 + 512) << 20, 0);
        }
    }
    // the n - 1 pages in front of the token's own one, whose page is always taken
    const uint32_t others = n - 1u, stride = cluster * kWarps * kGroup;
    const uint4* bounds = static_cast<const uint4*>(kv.bounds);
    auto look_up = [&](uint32_t i0) {
        return lane < kGroup && i0 + lane < others ? load_page(b, kv, s, i0 + lane, st) : kNone;
    };
    uint4 x[kGroup][PIECES], ahead[kGroup][PIECES];
    auto fetch = [&](uint32_t of) {  // of: the group's page ids, one per lane
#pragma unroll
        for (uint32_t j = 0; j < kGroup; ++j) {
            const uint32_t page = __shfl_sync(0xFFFFFFFFu, of, j);
#pragma unroll
            for (uint32_t i = 0; i < PIECES; ++i) {
                ahead[j][i] = make_uint4(0u, 0u, 0u, 0u);
                if (page != kNone && lane + 32u * i < 2u * half_pieces)
                    ahead[j][i] = __ldg(bounds + (static_cast<size_t>(page) * kv.kv_heads + kh) * 2u * half_pieces + lane + 32u * i);
            }
        }
    };
    // with one piece per lane there are registers for the next group's loads to be in flight
    // while this one is added up
    constexpr bool kAhead = PIECES == 1u;
    uint32_t i0 = (rank * kWarps + warp) * kGroup;
    uint32_t next = look_up(i0), pages = kNone, after = look_up(i0 + stride);
    if (kAhead) fetch(next);
    bool waited = false;
    for (; i0 < others; i0 += stride) {
        if (!kAhead) fetch(next);
#pragma unroll
        for (uint32_t j = 0; j < kGroup; ++j)
#pragma unroll
            for (uint32_t i = 0; i < PIECES; ++i) x[j][i] = ahead[j][i];
        pages = next;
        next = after;
        if (kAhead && i0 + stride < others) fetch(next);
        after = look_up(i0 + 2u * stride);
        double v[kGroup];
        uint32_t odd = 0u;
#pragma unroll
        for (uint32_t j = 0; j < kGroup; ++j) {
            v[j] = 0.0;
#pragma unroll
            for (uint32_t i = 0; i < PIECES; ++i) {
                odd |= P::odd(x[j][i]);
#pragma unroll
                for (uint32_t e = 0; e < P::kCount; ++e) v[j] = fma(P::value(x[j][i], e), f[i][e], v[j]);
            }
        }
        if (__any_sync(0xFFFFFFFFu, (odd & P::kOdd) != 0u)) {  // infinities and NaN
#pragma unroll
            for (uint32_t j = 0; j < kGroup; ++j) {
                v[j] = 0.0;
#pragma unroll
                for (uint32_t i = 0; i < PIECES; ++i)
                    if (lane + 32u * i < 2u * half_pieces)
#pragma unroll
                        for (uint32_t e = 0; e < P::kCount; ++e) v[j] = fma(P::exact(x[j][i], e), f[i][e], v[j]);
            }
        }
        double w[4], y[2];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) w[j] = exchange(v[j], v[j + 4], lane & 16u, 16u);
        y[0] = exchange(w[0], w[2], lane & 8u, 8u);
        y[1] = exchange(w[1], w[3], lane & 8u, 8u);
        double z = exchange(y[0], y[1], lane & 4u, 4u);  // page lane / 4
        z += __shfl_xor_sync(0xFFFFFFFFu, z, 2);
        z += __shfl_xor_sync(0xFFFFFFFFu, z, 1);
        const uint32_t mine = __shfl_sync(0xFFFFFFFFu, pages, lane >> 2);
        if (!waited) {
            cluster_wait();
            waited = true;
        }
        if ((lane & 3u) == 0u && i0 + (lane >> 2) < others) {
            const uint64_t k = mine != kNone ? score_key(z) : 0ull;
            store_first(smem_addr(key + i0 + (lane >> 2)), k);
        }
        __syncwarp();
    }
    if (!waited) cluster_wait();
    cluster_arrive();
    if (rank != 0u) return;
    cluster_wait();
    // the (picks - 1)-th largest key: the bits that all keys share, then eight bits at a time
    uint32_t left = picks - 1u, total;  // still to be found among the keys that share `prefix`
    uint64_t prefix = 0;                // in the bits above `shift`
    int shift = 64;
    if (left != 0u) {
        uint64_t any = 0, every = ~0ull;
        for (uint32_t i = tid; i < others; i += kThreads) {
            any |= key[i];
            every &= key[i];
        }
        for (int o = 16; o > 0; o >>= 1) {
            any |= __shfl_xor_sync(0xFFFFFFFFu, any, o);
            every &= __shfl_xor_sync(0xFFFFFFFFu, every, o);
        }
        if (lane == 0u) {
            masks[0][warp] = any;
            masks[1][warp] = every;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
            any |= masks[0][w];
            every &= masks[1][w];
        }
        shift = 64 - __clzll(static_cast<long long>(any ^ every));  // all keys share the bits from here up
        prefix = shift < 64 ? any >> shift << shift : 0ull;
        bool done = shift == 0;  // all keys are the same
        while (!done) {
            const int next = max(0, shift - 8);
            const uint32_t mask = (1u << (shift - next)) - 1u;
            hist[tid] = 0u;
            __syncthreads();
            for (uint32_t i = tid; i < others; i += kThreads) {
                const uint64_t k = key[i];
                if (shift == 64 || (k >> shift) == (prefix >> shift))
                    atomicAdd(&hist[static_cast<uint32_t>(k >> next) & mask], 1u);
            }
            __syncthreads();
            const uint32_t mine = hist[255u - tid];  // bins from the top
            const uint32_t upto = block_scan(mine, warp_sums, &total);
            if (upto >= left && upto - mine < left) {
                found[0] = 255u - tid;
                found[1] = left - (upto - mine);
            }
            __syncthreads();
            prefix |= static_cast<uint64_t>(found[0]) << next;
            left = found[1];
            shift = next;
            done = shift == 0 || hist[found[0]] == left;  // the whole bin is taken
            __syncthreads();
        }
    }
    // in page order: the keys above the threshold's bits, and the first `left` that share them
    const uint32_t run = (others + kThreads - 1u) / kThreads, a0 = min(others, tid * run), a1 = min(others, a0 + run);
    const uint64_t floor_key = shift < 64 ? prefix >> shift : 0ull;
    auto rank_of = [&](uint64_t k) -> uint32_t {  // 2 above, 1 the same, 0 below
        if (picks == 1u) return 0u;
        if (shift == 64) return 1u;
        const uint64_t x = k >> shift;
        return x > floor_key ? 2u : x == floor_key ? 1u : 0u;
    };
    uint32_t count = 0;  // above in the low half, the same in the high half (at most 16384 each)
    for (uint32_t i = a0; i < a1; ++i) {
        const uint32_t c = rank_of(key[i]);
        count += c == 2u ? 1u : c == 1u ? 0x10000u : 0u;
    }
    const uint32_t before = block_scan(count, warp_sums, &total) - count;
    uint32_t above = before & 0xFFFFu, same = before >> 16;
    for (uint32_t i = a0; i < a1; ++i) {
        const uint32_t c = rank_of(key[i]);
        if (c == 2u || (c == 1u && same < left)) out[above + min(same, left)] = i;
        above += c == 2u;
        same += c == 1u;
    }
    if (tid == 0u) out[picks - 1u] = n - 1u;  // the token's own page
}

template <typename T, uint32_t PIECES>
cudaError_t launch(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* q, uint32_t picks,
                   uint32_t* blocks, DeviceStatus* st, cudaStream_t stream) {
    const uint32_t pages = (b.max_kv_len + kv.page_size - 1u) >> kv.page_shift;
    const size_t smem = static_cast<size_t>(pages) * sizeof(uint64_t) + 16u;
    cudaError_t e = cudaFuncSetAttribute(block_select_kernel<T, PIECES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    // CTAs per token and KV head: enough for two to an SM, each with pages for its warps (48
    // tokens x 4 heads x up to 1024 pages: 51 us with one, 47 with two, 50 with four, 67 with eight)
    const uint64_t units = static_cast<uint64_t>(b.tokens) * kv.kv_heads;
    uint32_t cluster = 1;
    while (cluster < 8u && units * cluster < 2u * 148u && pages > cluster * kWarps * kGroup) cluster *= 2u;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<uint32_t>(units * cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, block_select_kernel<T, PIECES>, kv, b, heads, q, picks, blocks, cluster, st);
}

}  // namespace

cudaError_t launch_block_select(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* q, uint32_t picks,
                                uint32_t* blocks, DeviceStatus* st, cudaStream_t stream) {
    const uint32_t pieces = 2u * kv.head_dim * (kv.type == kF16 ? 2u : 4u) / 16u;  // of a page's bounds
    if (kv.type == kF16)
        return pieces <= 32u ? launch<__half, 1>(kv, b, heads, q, picks, blocks, st, stream)
                             : launch<__half, 2>(kv, b, heads, q, picks, blocks, st, stream);
    return pieces <= 32u   ? launch<float, 1>(kv, b, heads, q, picks, blocks, st, stream)
           : pieces <= 64u ? launch<float, 2>(kv, b, heads, q, picks, blocks, st, stream)
                           : launch<float, 4>(kv, b, heads, q, picks, blocks, st, stream);
}

}  // namespace nedo_gpu

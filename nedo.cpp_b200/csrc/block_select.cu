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
// Bound by reading the pages' bounds (4 hd bytes of an F16 cache per page and KV head).  A
// cluster of CTAs takes one token and KV head, its warps eight pages at a time with the next
// eight pages' loads in flight; the halves of a page's bounds lie next to each other, so a
// lane takes 16 bytes of them with its own factors in registers.
//
// The scores are first formed in 32 bits, with a bound on what that can be off: every sum of
// n terms is n + 13 roundings (in the factors, the products, the sums along a lane and across
// the warp) of at most 2^-24 sum |factor| max |bound|.  Their order-preserving keys go to the
// first CTA's shared memory, which finds the (picks - 1)-th largest, eight bits at a time
// below the bits that all keys share.  Pages further above it than twice the bound are taken,
// pages further below are not, and only those between, if not all of them fit, are scored
// again in 64 bits.  Where there are too many of those (many equal pages) or the bounds are
// not finite, all pages are scored in 64 bits by that CTA.
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
// A store, and a maximum, at `addr` of the first CTA's shared memory.
__device__ __forceinline__ void store_first(uint32_t addr, uint32_t v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(addr));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
__device__ __forceinline__ void max_first(uint32_t addr, uint32_t v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(addr));
    asm volatile("red.shared::cluster.max.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}

// A 16-byte piece of the bounds: its values, and the largest magnitude among them and `top`
// as non-negative bits that order NaN above infinity above all numbers.
template <typename T>
struct Piece;
template <>
struct Piece<__half> {
    static constexpr uint32_t kCount = 8;
    static __device__ __forceinline__ float2 pair(const uint4& x, uint32_t i) {  // values 2 i, 2 i + 1
        const uint32_t w = i == 0u ? x.x : i == 1u ? x.y : i == 2u ? x.z : x.w;
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
    static __device__ __forceinline__ void magnitude(const uint4& x, uint32_t* top) {
        *top = __vmaxu2(__vmaxu2(*top, __vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu)),
                        __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
    }
    static __device__ __forceinline__ float largest(uint32_t top) {
        return half_bits_to_float(max(top & 0xFFFFu, top >> 16));
    }
};
template <>
struct Piece<float> {
    static constexpr uint32_t kCount = 4;
    static __device__ __forceinline__ float2 pair(const uint4& x, uint32_t i) {
        return i == 0u ? make_float2(__uint_as_float(x.x), __uint_as_float(x.y))
                       : make_float2(__uint_as_float(x.z), __uint_as_float(x.w));
    }
    static __device__ __forceinline__ void magnitude(const uint4& x, uint32_t* top) {
        *top = max(max(*top, max(x.x & 0x7FFFFFFFu, x.y & 0x7FFFFFFFu)), max(x.z & 0x7FFFFFFFu, x.w & 0x7FFFFFFFu));
    }
    static __device__ __forceinline__ float largest(uint32_t top) { return __uint_as_float(top); }
};

template <typename V>
__device__ __forceinline__ V exchange(V a, V b, bool up, uint32_t mask) {
    const V keep = up ? b : a, send = up ? a : b;
    return keep + __shfl_xor_sync(0xFFFFFFFFu, send, mask);
}

// Order-preserving 32-bit key of a finite number, and back.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __float_as_uint(v);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7FFFFFFFu : ~k); }

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

// The `left`-th largest of key[0..n) (one CTA), to `shift` bits: *prefix holds its bits from
// `shift` up, and the first return value how many of the keys that share them are to be taken.
// Stops early where the keys that share them are all taken, unless the key is wanted whole.
template <typename K>
__device__ uint32_t find_largest(const K* key, uint32_t n, uint32_t left, bool whole, K* prefix_out, int* shift_out,
                                 uint32_t* hist, uint32_t* warp_sums, uint32_t* found, K (*masks)[kWarps]) {
    constexpr int kBits = 8 * sizeof(K);
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    K any = 0, every = ~static_cast<K>(0);
    for (uint32_t i = tid; i < n; i += kThreads) {
        any |= key[i];
        every &= key[i];
    }
    for (int o = 16; o > 0; o >>= 1) {
        any |= __shfl_xor_sync(0xFFFFFFFFu, any, o);
        every &= __shfl_xor_sync(0xFFFFFFFFu, every, o);
    }
    __syncthreads();
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
    const uint64_t differ = any ^ every;
    int shift = differ ? 64 - __clzll(static_cast<long long>(differ)) : 0;  // all keys share the bits from here up
    K prefix = shift < kBits ? any >> shift << shift : 0;
    bool done = shift == 0;  // all keys are the same
    while (!done) {
        const int next = max(0, shift - 8);
        const uint32_t mask = (1u << (shift - next)) - 1u;
        uint32_t total;
        hist[tid] = 0u;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += kThreads) {
            const K k = key[i];
            if (shift == kBits || (k >> shift) == (prefix >> shift))
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
        prefix |= static_cast<K>(found[0]) << next;
        left = found[1];
        shift = next;
        done = shift == 0 || (!whole && hist[found[0]] == left);
        __syncthreads();
    }
    *prefix_out = prefix;
    *shift_out = shift;
    return left;
}

// PIECES: 16-byte pieces of a page's bounds per lane.
template <typename T, uint32_t PIECES>
__global__ void __launch_bounds__(kThreads) block_select_kernel(PagedKv kv, PagedBatch b, uint32_t heads,
                                                                const float* __restrict__ q, uint32_t picks,
                                                                uint32_t* __restrict__ blocks, uint32_t cluster,
                                                                DeviceStatus* st) {
    using P = Piece<T>;
    extern __shared__ __align__(16) uint64_t key64[];
    uint32_t* const key = reinterpret_cast<uint32_t*>(key64);
    __shared__ uint32_t hist[256], warp_sums[kWarps], found[2], top_bits, cand[256], cands;
    __shared__ uint64_t masks[2][kWarps], cand_key[256];
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
    if (n <= picks || picks == 1u) {  // all of them, or its own only
        if (rank == 0u)
            for (uint32_t i = tid; i < picks; i += kThreads) out[i] = picks == 1u && n != 0u ? n - 1u : i < n ? i : kNone;
        return;
    }
    if (tid == 0u) {
        top_bits = 0u;
        cands = 0u;
    }
    cluster_arrive();  // the first CTA runs, and has set these, before anything is stored into its memory
    // this lane's factors: of its pieces of the bounds (lowest values first, then highest)
    const uint32_t half_pieces = hd / P::kCount;
    const float* qh = q + (static_cast<size_t>(t) * heads + kh * group) * hd;
    float f[PIECES][P::kCount], size = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < PIECES; ++i) {
#pragma unroll
        for (uint32_t e = 0; e < P::kCount; ++e) f[i][e] = 0.f;
        const uint32_t piece = lane + 32u * i;
        if (piece < 2u * half_pieces) {
            const bool high = piece >= half_pieces;
            const float* src = qh + (high ? piece - half_pieces : piece) * P::kCount;
            for (uint32_t g = 0; g < group; ++g)
#pragma unroll
                for (uint32_t e = 0; e < P::kCount; e += 4u) {
                    const float4 y = *reinterpret_cast<const float4*>(src + static_cast<size_t>(g) * hd + e);
                    const float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (uint32_t u = 0; u < 4u; ++u)
                        if (!(v[u] < 0.f) == high) f[i][e + u] += v[u];  // NaN to the highest
                }
        }
#pragma unroll
        for (uint32_t e = 0; e < P::kCount; ++e) size += fabsf(f[i][e]);
    }
    size = warp_sum(size);
    // the n - 1 pages in front of the token's own one, whose page is always taken
    const uint32_t others = n - 1u, stride = cluster * kWarps * kGroup;
    const uint4* bounds = static_cast<const uint4*>(kv.bounds);
    auto look_up = [&](uint32_t i0) {
        return lane < kGroup && i0 + lane < others ? load_page(b, kv, s, i0 + lane, st) : kNone;
    };
    // with one piece per lane there are registers for the next group's loads to be in flight
    // while this one is added up
    constexpr bool kAhead = PIECES == 1u;
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
    uint32_t i0 = (rank * kWarps + warp) * kGroup;
    uint32_t next = look_up(i0), pages = kNone, after = look_up(i0 + stride), top = 0u;
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
        float v[kGroup];
#pragma unroll
        for (uint32_t j = 0; j < kGroup; ++j) {
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (uint32_t i = 0; i < PIECES; ++i) {
                P::magnitude(x[j][i], &top);
#pragma unroll
                for (uint32_t e = 0; e < P::kCount / 2u; ++e)
                    sum = ffma2(P::pair(x[j][i], e), make_float2(f[i][2u * e], f[i][2u * e + 1u]), sum);
            }
            v[j] = sum.x + sum.y;
        }
        float w[4], y[2];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) w[j] = exchange(v[j], v[j + 4], lane & 16u, 16u);
        y[0] = exchange(w[0], w[2], lane & 8u, 8u);
        y[1] = exchange(w[1], w[3], lane & 8u, 8u);
        float z = exchange(y[0], y[1], lane & 4u, 4u);  // page lane / 4
        z += __shfl_xor_sync(0xFFFFFFFFu, z, 2);
        z += __shfl_xor_sync(0xFFFFFFFFu, z, 1);
        const uint32_t mine = __shfl_sync(0xFFFFFFFFu, pages, lane >> 2);
        if (!waited) {
            cluster_wait();
            waited = true;
        }
        // a page that is none: below all others
        if ((lane & 3u) == 0u && i0 + (lane >> 2) < others)
            store_first(smem_addr(key + i0 + (lane >> 2)), mine != kNone ? key_of(z == 0.f ? 0.f : z) : 0u);
        __syncwarp();
    }
    if (!waited) cluster_wait();
    // the largest magnitude of all bounds, as a number's bits
    const uint32_t largest = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(P::largest(top)));
    if (lane == 0u) max_first(smem_addr(&top_bits), largest);
    cluster_arrive();
    if (rank != 0u) return;
    cluster_wait();

    // a page's score in 64 bits, by one warp
    auto exact_key = [&](uint32_t i) -> uint64_t {
        const uint32_t page = load_page(b, kv, s, i, st);
        if (page == kNone) return 0ull;
        const T* lo = static_cast<const T*>(kv.bounds) + (static_cast<size_t>(page) * kv.kv_heads + kh) * 2u * hd;
        double z = 0.0;
        for (uint32_t d = lane; d < hd; d += 32u) {
            double up = 0.0, down = 0.0;
            for (uint32_t g = 0; g < group; ++g) {
                const double y = qh[static_cast<size_t>(g) * hd + d];
                if (y < 0.0) down += y;
                else up += y;
            }
            z += up * static_cast<double>(kv_float(lo[hd + d])) + down * static_cast<double>(kv_float(lo[d]));
        }
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
        return score_key(z);
    };

    const uint32_t want = picks - 1u;
    // what a score can be off, rounded up (nothing where all of them are zero)
    const float most = size * __uint_as_float(top_bits) * 1.01f;
    const float off = most == 0.f ? 0.f : (PIECES * P::kCount + group + 13u) * 6.0e-8f * most + 1e-37f;
    uint32_t prefix = 0, total, sure = 0, left = 0;
    int shift = 0;
    bool all64 = !(most < INFINITY);
    float above = 0.f, below = 0.f;
    if (!all64) {
        left = find_largest<uint32_t>(key, others, want, true, &prefix, &shift, hist, warp_sums, found,
                                      reinterpret_cast<uint32_t(*)[kWarps]>(masks));
        if (off > 0.f && prefix != 0u) {
            // the pages that 32 bits leave open
            above = number_of(prefix) + 2.f * off;
            below = number_of(prefix) - 2.f * off;
            above += fabsf(above) * 2.4e-7f;  // these sums round too
            below -= fabsf(below) * 2.4e-7f;
            uint32_t taken = 0;
            for (uint32_t i = tid; i < others; i += kThreads) {
                const uint32_t k = key[i];
                if (k == 0u) continue;
                const float z = number_of(k);
                if (z > above) {
                    ++taken;
                } else if (z >= below) {
                    const uint32_t c = atomicAdd(&cands, 1u);
                    if (c < 256u) cand[c] = i;
                }
            }
            block_scan(taken, warp_sums, &sure);
            __syncthreads();
            left = want - sure;
            all64 = cands > 256u;
            if (!all64 && cands > left) {
                const uint32_t count = cands;
                for (uint32_t c = warp; c < count; c += kWarps) {
                    const uint64_t k = exact_key(cand[c]);
                    if (lane == 0u) cand_key[c] = k;
                }
                __syncthreads();
                // those that `left` others beat are not taken
                if (tid < count) {
                    const uint64_t mine = cand_key[tid];
                    const uint32_t at = cand[tid];
                    uint32_t better = 0;
                    for (uint32_t c = 0; c < count; ++c)
                        better += cand_key[c] > mine || (cand_key[c] == mine && cand[c] < at);
                    if (better >= left) key[at] = 0u;
                }
                __syncthreads();
            }
        }
    }
    uint64_t prefix64 = 0;
    if (all64) {
        for (uint32_t i = warp; i < others; i += kWarps) {
            const uint64_t k = exact_key(i);
            if (lane == 0u) key64[i] = k;
        }
        __syncthreads();
        left = find_largest<uint64_t>(key64, others, want, false, &prefix64, &shift, hist, warp_sums, found, masks);
    }
    // in page order: the pages that are taken for certain (2), and the first `left` of those that
    // share the threshold (1)
    const bool bounded = !all64 && off > 0.f && prefix != 0u;
    auto rank_of = [&](uint32_t i) -> uint32_t {
        if (all64) {
            if (shift == 64) return 1u;
            const uint64_t x = key64[i] >> shift, y = prefix64 >> shift;
            return x > y ? 2u : x == y ? 1u : 0u;
        }
        const uint32_t k = key[i];
        if (bounded) return k != 0u && number_of(k) >= below ? 2u : 0u;
        return k > prefix ? 2u : k == prefix ? 1u : 0u;
    };
    const uint32_t run = (others + kThreads - 1u) / kThreads, a0 = min(others, tid * run), a1 = min(others, a0 + run);
    uint32_t count = 0;  // taken in the low half, sharing in the high half (at most 16384 each)
    for (uint32_t i = a0; i < a1; ++i) {
        const uint32_t c = rank_of(i);
        count += c == 2u ? 1u : c == 1u ? 0x10000u : 0u;
    }
    const uint32_t before = block_scan(count, warp_sums, &total) - count;
    uint32_t in = before & 0xFFFFu, same = before >> 16;
    for (uint32_t i = a0; i < a1; ++i) {
        const uint32_t c = rank_of(i);
        if (c == 2u || (c == 1u && same < left)) out[in + min(same, left)] = i;
        in += c == 2u;
        same += c == 1u;
    }
    if (tid == 0u) out[want] = n - 1u;  // the token's own page
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

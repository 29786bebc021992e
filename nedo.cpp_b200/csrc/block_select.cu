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
// cluster of CTAs takes one token and KV head, its warps eight pages at a time through a ring of
// their own (cp.async, two stages); the halves of a page's bounds lie next to each
// other, so a lane takes 16 bytes of them, its own copy, with its own factors in registers.
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
#include "paged_mma.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kThreads = 128;
constexpr uint32_t kWarps = kThreads / 32u;
constexpr uint32_t kGroup = 8;  // pages a warp scores at once
constexpr uint32_t kOpen = 64;  // pages that are scored again in 64 bits at most

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
// A store, and a maximum, union and intersection of bits, at `addr` of the first CTA's shared
// memory.
__device__ __forceinline__ uint32_t first_cta(uint32_t addr) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(addr));
    return remote;
}
__device__ __forceinline__ void store_first(uint32_t remote, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
__device__ __forceinline__ void max_first(uint32_t remote, uint32_t v) {
    asm volatile("red.shared::cluster.max.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
__device__ __forceinline__ void or_first(uint32_t remote, uint32_t v) {
    asm volatile("red.shared::cluster.or.b32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
__device__ __forceinline__ void and_first(uint32_t remote, uint32_t v) {
    asm volatile("red.shared::cluster.and.b32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
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

// The `left`-th largest of key[0..n) (one CTA): its bits from *shift up, in *prefix, and how
// many of the keys that share them are still to be taken (returned).  All keys share the bits
// outside `differ`; *prefix comes with those.  Stops where at most `few` keys share the bits.
template <typename K>
__device__ uint32_t find_largest(const K* key, uint32_t n, uint32_t left, uint32_t few, uint64_t differ, K* prefix, int* shift,
                                 uint32_t* hist, uint32_t* warp_sums, uint32_t* found) {
    constexpr int kBits = 8 * sizeof(K);
    const uint32_t tid = threadIdx.x;
    int at = differ ? 64 - __clzll(static_cast<long long>(differ)) : 0;
    K bits = at < kBits ? *prefix >> at << at : 0;
    bool done = at == 0 || n <= few;
    while (!done) {
        const int next = max(0, at - 8);
        const uint32_t mask = (1u << (at - next)) - 1u;
        uint32_t total;
        hist[2u * tid] = hist[2u * tid + 1u] = 0u;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += kThreads) {
            const K k = key[i];
            if (at == kBits || (k >> at) == (bits >> at)) atomicAdd(&hist[static_cast<uint32_t>(k >> next) & mask], 1u);
        }
        __syncthreads();
        const uint32_t high = hist[255u - 2u * tid], low = hist[254u - 2u * tid];  // two bins, from the top
        const uint32_t upto = block_scan(high + low, warp_sums, &total), before = upto - high - low;
        if (upto >= left && before < left) {
            const bool first = before + high >= left;
            found[0] = 255u - 2u * tid - (first ? 0u : 1u);
            found[1] = left - before - (first ? 0u : high);
            found[2] = first ? high : low;
        }
        __syncthreads();
        bits |= static_cast<K>(found[0]) << next;
        left = found[1];
        at = next;
        done = at == 0 || found[2] <= few;
        __syncthreads();
    }
    *prefix = bits;
    *shift = at;
    return left;
}

constexpr uint32_t kStages = 2;  // three run no faster: fewer CTAs fit (48 tokens x 4 heads: 26.2 us with two, 27.2 with three)

// PIECES: 16-byte pieces of a page's bounds per lane.  Dynamic shared memory: key_words words of
// 32 bits for the keys, then the warps' rings.  Keys of 64 bits lie over both: they are formed
// when the rings are done with.
template <typename T, uint32_t PIECES>
__global__ void __launch_bounds__(kThreads) block_select_kernel(PagedKv kv, PagedBatch b, uint32_t heads,
                                                                const float* __restrict__ q, uint32_t picks,
                                                                uint32_t* __restrict__ blocks, uint32_t cluster,
                                                                uint32_t key_words, DeviceStatus* st) {
    using P = Piece<T>;

    extern __shared__ __align__(16) uint64_t key64[];
    uint32_t* const key = reinterpret_cast<uint32_t*>(key64);
    __shared__ uint32_t hist[256], warp_sums[kWarps], found[3], top_bits, any_bits, all_bits, cand[kOpen], cands;
    __shared__ uint64_t cand_key[kOpen], masks[2][kWarps];
    __shared__ double factor[2][256];
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
        top_bits = any_bits = cands = 0u;
        all_bits = 0xFFFFFFFFu;
    }
    cluster_arrive();  // the first CTA runs, and has set these, before anything is stored into its memory
    // the n - 1 pages in front of the token's own one, whose page is always taken
    const uint32_t others = n - 1u, stride = cluster * kWarps * kGroup;
    const uint32_t half_pieces = hd / P::kCount;
    const uint4* bounds = static_cast<const uint4*>(kv.bounds);
    // group k of this warp: pages i0 + k * stride .. + 7.  Lane 8 g + j holds the id of page j of
    // group 4 m + g (now) and of group 4 m + 4 + g (then).
    const uint32_t i0 = (rank * kWarps + warp) * kGroup, ng = i0 < others ? (others - i0 + stride - 1u) / stride : 0u;
    auto look_up = [&](uint32_t m) {
        const uint32_t k = 4u * m + (lane >> 3), i = i0 + k * stride + (lane & 7u);
        return k < ng && i < others ? load_page(b, kv, s, i, st) : kNone;
    };
    uint4* const ring = reinterpret_cast<uint4*>(key + key_words) + warp * kStages * kGroup * PIECES * 32u;
    uint32_t now = look_up(0), then = look_up(1), top = 0u;
    auto fetch = [&](uint32_t k, uint32_t m) {
        if (k < ng) {
            const uint32_t ids = k >> 2 == m ? now : then;
#pragma unroll
            for (uint32_t j = 0; j < kGroup; ++j) {
                const uint32_t page = __shfl_sync(0xFFFFFFFFu, ids, (k & 3u) * 8u + j);
#pragma unroll
                for (uint32_t i = 0; i < PIECES; ++i) {
                    const bool there = page != kNone && lane + 32u * i < 2u * half_pieces;
                    const size_t at = (static_cast<size_t>(there ? page : 0u) * kv.kv_heads + kh) * 2u * half_pieces +
                                      (there ? lane + 32u * i : 0u);
                    cp_async16(smem_addr(ring + (((k % kStages) * kGroup + j) * PIECES + i) * 32u + lane), bounds + at,
                               there ? 16u : 0u);
                }
            }
        }
        cp_commit();
    };
#pragma unroll
    for (uint32_t k = 0; k + 1u < kStages; ++k) fetch(k, 0u);
    // this lane's factors: of its pieces of the bounds (lowest values first, then highest)
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
#pragma unroll 4
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
    const uint32_t key_addr = first_cta(smem_addr(key));
    uint32_t any = 0u, every = 0xFFFFFFFFu;
    bool waited = false;
    for (uint32_t k = 0; k < ng; ++k) {
        const uint32_t first = i0 + k * stride, pages = __shfl_sync(0xFFFFFFFFu, now, (k & 3u) * 8u + (lane >> 2));
        fetch(k + kStages - 1u, k >> 2);
        if ((k & 3u) == 3u) {
            now = then;
            then = look_up((k >> 2) + 2u);
        }
        cp_wait<kStages - 1>();
        float v[kGroup];
#pragma unroll
        for (uint32_t j = 0; j < kGroup; ++j) {
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (uint32_t i = 0; i < PIECES; ++i) {
                const uint4 x = ring[(((k % kStages) * kGroup + j) * PIECES + i) * 32u + lane];  // this lane's own copy
                P::magnitude(x, &top);
#pragma unroll
                for (uint32_t e = 0; e < P::kCount / 2u; ++e)
                    sum = ffma2(P::pair(x, e), make_float2(f[i][2u * e], f[i][2u * e + 1u]), sum);
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
        if (!waited) {
            cluster_wait();
            waited = true;
        }
        if ((lane & 3u) == 0u && first + (lane >> 2) < others) {
            const uint32_t x = pages != kNone ? key_of(z == 0.f ? 0.f : z) : 0u;  // a page that is none: below all others
            store_first(key_addr + 4u * (first + (lane >> 2)), x);
            any |= x;
            every &= x;
        }
        __syncwarp();
    }
    if (!waited) cluster_wait();
    // the largest magnitude of all bounds, as a number's bits, and the bits of the keys
    const uint32_t largest = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(P::largest(top)));
    any = __reduce_or_sync(0xFFFFFFFFu, any);
    every = __reduce_and_sync(0xFFFFFFFFu, every);
    if (lane == 0u) {
        max_first(first_cta(smem_addr(&top_bits)), largest);
        or_first(first_cta(smem_addr(&any_bits)), any);
        and_first(first_cta(smem_addr(&all_bits)), every);
    }
    cluster_arrive();
    if (rank != 0u) return;
    cluster_wait();

    // a page's score in 64 bits, by one warp, from the factors in shared memory
    auto factors = [&]() {
        for (uint32_t d = tid; d < hd; d += kThreads) {
            double up = 0.0, down = 0.0;
#pragma unroll 4
            for (uint32_t g = 0; g < group; ++g) {
                const double y = qh[static_cast<size_t>(g) * hd + d];
                if (y < 0.0) down += y;
                else up += y;
            }
            factor[0][d] = down;
            factor[1][d] = up;
        }
        __syncthreads();
    };
    auto exact_key = [&](uint32_t i) -> uint64_t {
        const uint32_t page = load_page(b, kv, s, i, st);
        if (page == kNone) return 0ull;
        const T* lo = static_cast<const T*>(kv.bounds) + (static_cast<size_t>(page) * kv.kv_heads + kh) * 2u * hd;
        double z = 0.0;
#pragma unroll 4
        for (uint32_t d = lane; d < hd; d += 32u)
            z += factor[1][d] * static_cast<double>(kv_float(lo[hd + d])) + factor[0][d] * static_cast<double>(kv_float(lo[d]));
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
        return score_key(z);
    };

    const uint32_t want = picks - 1u;
    // what a score can be off, rounded up (nothing where all of them are zero, not only too small for 32 bits)
    const float most = size * __uint_as_float(top_bits) * 1.01f;
    const bool zero = most == 0.f && (size == 0.f || top_bits == 0u);
    const float off = zero ? 0.f : (PIECES * P::kCount + group + 13u) * 6.0e-8f * most + 1e-37f;
    // a thread's share of the pages, in order
    const uint32_t run = (others + kThreads - 1u) / kThreads, a0 = min(others, tid * run), a1 = min(others, a0 + run);
    uint32_t total;
    if (most < INFINITY && off > 0.f) {
        uint32_t prefix = any_bits;
        int shift;
        find_largest<uint32_t>(key, others, want, 1u, any_bits ^ all_bits, &prefix, &shift, hist,
                                                     warp_sums, found);
        // the threshold lies between these; pages above are taken, below not, the others are open
        const uint32_t high = prefix | (shift < 32 ? (1u << shift) - 1u : 0xFFFFFFFFu);
        if (prefix != 0u && high < 0xFF800000u) {
            float above = number_of(high) + 2.f * off, below = number_of(prefix) - 2.f * off;
            above += fabsf(above) * 2.4e-7f;  // these sums round too
            below -= fabsf(below) * 2.4e-7f;
            uint32_t taken = 0, which = 0;  // which: of the thread's first 32 pages
            for (uint32_t i = a0; i < a1; ++i) {
                const float z = number_of(key[i]);
                if (z > above) {
                    ++taken;
                    if (i - a0 < 32u) which |= 1u << (i - a0);
                } else if (z >= below) {
                    const uint32_t c = atomicAdd(&cands, 1u);
                    if (c < kOpen) cand[c] = i;
                }
            }
            const uint32_t before = block_scan(taken, warp_sums, &total) - taken;
            __syncthreads();
            const uint32_t left = want - total, count = cands;
            if (count <= kOpen) {
                if (count > left) {
                    factors();
                    for (uint32_t c = warp; c < count; c += kWarps) {
                        const uint64_t k = exact_key(cand[c]);
                        if (lane == 0u) cand_key[c] = k;
                    }
                    __syncthreads();
                    // those that `left` others beat are not taken
                    uint32_t better = 0;
                    if (tid < count)
                        for (uint32_t c = 0; c < count; ++c)
                            better += cand_key[c] > cand_key[tid] || (cand_key[c] == cand_key[tid] && cand[c] < cand[tid]);
                    __syncthreads();
                    if (tid < count && better >= left) cand[tid] = kNone;
                    __syncthreads();
                }
                // in page order: a page comes behind the taken ones in front of it
                uint32_t in = before;
                auto put = [&](uint32_t i) {
                    uint32_t open = 0;
                    for (uint32_t c = 0; c < count; ++c) open += cand[c] < i;
                    out[in + open] = i;
                    ++in;
                };
                for (uint32_t m = which; m != 0u; m &= m - 1u) put(a0 + __ffs(m) - 1u);
                for (uint32_t i = a0 + 32u; i < a1; ++i)
                    if (number_of(key[i]) > above) put(i);
                // an open page that is taken: its thread counts the certain ones in front of it
                for (uint32_t c = 0; c < count; ++c) {
                    const uint32_t i = cand[c];
                    if (i == kNone || i < a0 || i >= a1) continue;
                    uint32_t at = before;
                    for (uint32_t k = a0; k < i; ++k) at += number_of(key[k]) > above;
                    for (uint32_t k = 0; k < count; ++k) at += cand[k] < i;
                    out[at] = i;
                }
                if (tid == 0u) out[want] = n - 1u;  // the token's own page
                return;
            }
        }
    }
    if (zero && all_bits == any_bits) {  // all scores are zero: the first pages
        for (uint32_t i = tid; i < picks; i += kThreads) out[i] = i < want ? i : n - 1u;
        return;
    }
    // all scores in 64 bits
    factors();
    for (uint32_t i = warp; i < others; i += kWarps) {
        const uint64_t k = exact_key(i);
        __syncwarp();
        if (lane == 0u) key64[i] = k;
    }
    __syncthreads();
    uint64_t any64 = 0, every64 = ~0ull;
    for (uint32_t i = tid; i < others; i += kThreads) {
        any64 |= key64[i];
        every64 &= key64[i];
    }
    for (int o = 16; o > 0; o >>= 1) {
        any64 |= __shfl_xor_sync(0xFFFFFFFFu, any64, o);
        every64 &= __shfl_xor_sync(0xFFFFFFFFu, every64, o);
    }
    if (lane == 0u) {
        masks[0][warp] = any64;
        masks[1][warp] = every64;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        any64 |= masks[0][w];
        every64 &= masks[1][w];
    }
    uint64_t prefix = any64;
    int shift;
    const uint32_t left = find_largest<uint64_t>(key64, others, want, 0u, any64 ^ every64, &prefix, &shift, hist, warp_sums, found);
    // in page order: the keys above it, and the first `left` of those that equal it
    uint32_t count = 0;  // above in the low half, equal in the high half (at most 16384 each)
    for (uint32_t i = a0; i < a1; ++i) count += key64[i] > prefix ? 1u : key64[i] == prefix ? 0x10000u : 0u;
    const uint32_t before = block_scan(count, warp_sums, &total) - count;
    uint32_t in = before & 0xFFFFu, same = before >> 16;
    for (uint32_t i = a0; i < a1; ++i) {
        const bool above = key64[i] > prefix, equal = key64[i] == prefix;
        if (above || (equal && same < left)) out[in + min(same, left)] = i;
        in += above;
        same += equal;
    }
    if (tid == 0u) out[want] = n - 1u;  // the token's own page
}

template <typename T, uint32_t PIECES>
cudaError_t launch(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* q, uint32_t picks,
                   uint32_t* blocks, DeviceStatus* st, cudaStream_t stream) {
    const uint32_t pages = (b.max_kv_len + kv.page_size - 1u) >> kv.page_shift;
    const uint32_t key_words = (pages + 3u) & ~3u;
    auto bytes = [](uint32_t words) {
        return std::max(words * sizeof(uint64_t), words * sizeof(uint32_t) + kWarps * kStages * kGroup * PIECES * 512u);
    };
    const size_t smem = bytes(key_words);
    // the limit is the process's: the same for every call, or one host thread's call could lower it
    // between another's limit and launch
    cudaError_t e = cudaFuncSetAttribute(block_select_kernel<T, PIECES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(bytes(kMaxSelectPages)));
    if (e != cudaSuccess) return e;
    // CTAs per token and KV head: as many as run at once on 148 SMs, with pages for every warp
    const uint64_t units = static_cast<uint64_t>(b.tokens) * kv.kv_heads;
    const uint64_t at_once = 148u * (224u * 1024u / (smem + 8192u));
    uint32_t cluster = 1;
    while (cluster < 8u && units * (cluster + 1u) <= at_once && pages > cluster * kWarps * kGroup) ++cluster;
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
    return cudaLaunchKernelEx(&cfg, block_select_kernel<T, PIECES>, kv, b, heads, q, picks, blocks, cluster,
                              key_words, st);
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

// verify_drafts.cu -- drafted tokens of a batch of sequences against the target's probabilities, and
// the token that follows those that are taken (speculative sampling; the sampling step of
// src/model.cpp:31-53 for several tokens at a time).
//
// Row i of a sequence has the logits behind its i-th draft, p_i = softmax(logits_i / T).  Draft x_i is
// taken where u_i q_i(x_i) < p_i(x_i), up to the first that is not; the next token is drawn from what
// is left of its row, max(p - q, 0), or from p of the last row where all were taken: the first token
// at which the running sum passes u times the whole.  Without draft probabilities q is 1 at the
// draft.  T = 0: a draft is taken where it is the first largest logit, and that is the next token.
//
// Two launches.  The first reads all logits, bound by that: a CTA takes a part of a row and leaves its
// largest logit and the sum of 2^((l - m) log2(e) / T), in 32 bits (T = 0: the largest one's place, which
// a thread looks for at the end, among the 16 that it remembers: 19 us for 288 rows of 64000, 22 with a key
// carried along).  The second, a cluster of CTAs per
// sequence, adds the parts and decides: a draft whose two sides differ by more than 2^-14, which is twice what they
// can be off (kOff), is decided, any other is looked at again with the row summed in 64 bits.  Then
// the one row that the next token comes from is read again, from L2, in 64 bits: a token
// of a large vocabulary can be 10^-6 of the whole, and u falls on the border of two in 32 bits
// every so often.  Every warp has a share of the tokens in order; the CTA of the warp whose share holds the
// border goes through that once more, a run of tokens to a thread.
//
// What bounds it: 32 sequences of four drafts with their probabilities over 128000 tokens 46 us, of which
// the first launch 15 (82 MB: 13 at the rate of a copy); then 5.5 us for the row's sum, 10 for that of what
// the draft's probabilities leave and 3 for the search.  Those are latency: six warps to a scheduler, which issue in
// 42 % of its cycles (the 64-bit pipe is busy for 20), wait for loads, for the result before and for
// the cluster's other CTAs in about equal parts; the second sum has a row of probabilities to load from memory, with
// two quads of a lane on their way, and forms the first one's exponentials again.  (Four CTAs to a cluster: 61 us; a
// table for every lane, or the probabilities brought into L2 during the first sum: the same.)  One sequence over
// 64000 tokens 16 us: two launches, and some 25,000 cycles of the second.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace nedo_gpu {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32u;
constexpr uint32_t kMaxCtas = 8;       // of a cluster
constexpr uint32_t kNone = 0xFFFFFFFFu;

// NaN counts as minus infinity, infinity as the largest number.
__device__ __forceinline__ float counted(float l) { return fminf(fmaxf(l, -INFINITY), 3.402823466e38f); }

struct VerifyArgs {
    VerifyDrafts v;
    float rate;          // log2(e) / T
    double inv_t;
    uint32_t chunk;      // logits per part, a multiple of 1024
    uint32_t parts;      // of a row
    float2* stats;       // [rows][parts]: (largest, sum); T = 0: the largest's key
    uint32_t* accepted;
    uint32_t* ids;
    DeviceStatus* st;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Larger is later: the logit's order, then the lower index.
__device__ __forceinline__ uint64_t pick_key(float l, uint32_t i) {
    const uint32_t u = l == 0.f ? 0u : __float_as_uint(l);  // (one key for both zeros)
    return static_cast<uint64_t>((u >> 31) ? ~u : (u | 0x80000000u)) << 32 | (~i);
}

// A row, which begins `shift` elements behind a 16-byte border, as quads: quad x holds its elements
// 4 x - shift and on.  Those in front of it, and behind its `n` elements, count as `none`.
struct Row {
    const float* first;
    uint32_t shift, n, whole0, wholes;  // quads [whole0, whole0 + wholes) are the row's alone
    __device__ __forceinline__ Row(const float* base, size_t at, uint32_t vocab)
        : first(base + at), shift(static_cast<uint32_t>(at & 3u)), n(vocab) {
        whole0 = shift != 0u;
        const uint32_t end = (n + shift) / 4u;
        wholes = end > whole0 ? end - whole0 : 0u;
    }
    __device__ __forceinline__ uint32_t quads() const { return (n + shift + 3u) / 4u; }
    __device__ __forceinline__ float4 load(uint32_t x, float none) const {
        const float* at = first + (static_cast<int64_t>(x) * 4 - shift);
        if (x - whole0 < wholes) return __ldcs(reinterpret_cast<const float4*>(at));
        float v[4];
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) {
            v[e] = none;
            if (4u * x + e >= shift && 4u * x + e - shift < n) v[e] = __ldg(at + e);
        }
        return make_float4(v[0], v[1], v[2], v[3]);
    }
};

// 16 of them, kThreads quads apart, up to quad `end`.
__device__ __forceinline__ void load_sixteen(const Row& row, uint32_t x, uint32_t end, float (&v)[16]) {
    float4 q[4];
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u) {
        q[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (x + u * kThreads < end) q[u] = row.load(x + u * kThreads, -INFINITY);
    }
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u) {
        v[4 * u] = q[u].x;
        v[4 * u + 1] = q[u].y;
        v[4 * u + 2] = q[u].z;
        v[4 * u + 3] = q[u].w;
    }
}

template <bool GREEDY>
__global__ void __launch_bounds__(kThreads, 8) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
    __shared__ float2 sums[kWarps];
    __shared__ uint32_t first;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    asm volatile("griddepcontrol.launch_dependents;");
    const Row row(a.v.logits, static_cast<size_t>(r) * a.v.vocab, a.v.vocab);
    // (quads, so that no part reads another's)
    const uint32_t x0 = part * (a.chunk / 4u), x1 = part + 1u == a.parts ? row.quads() : x0 + a.chunk / 4u;
    float m = -INFINITY, s = 0.f;
    uint32_t at = x0;  // the first sixteen with m
    auto add = [&](const float(&v)[16]) {
        float top = v[0];
#pragma unroll
        for (uint32_t e = 1; e < 16u; ++e) top = fmaxf(top, v[e]);
        if (top > m) {
            s *= exp2_fast((m - top) * a.rate);
            m = top;
        }
        if (m > -INFINITY) {  // the sixteen by halves: four roundings and one of the running sum
            float w[16];
#pragma unroll
            for (uint32_t e = 0; e < 16u; ++e) w[e] = exp2_fast((v[e] - m) * a.rate);
#pragma unroll
            for (uint32_t n = 8; n != 0u; n /= 2u)
#pragma unroll
                for (uint32_t e = 0; e < n; ++e) w[e] = w[2u * e] + w[2u * e + 1u];
            s += w[0];
        }
    };
    for (uint32_t x = x0 + tid; x < x1; x += 4u * kThreads) {
        float v[16];
        load_sixteen(row, x, x1, v);
        if constexpr (GREEDY) {
            float top = v[0];
#pragma unroll
            for (uint32_t e = 1; e < 16u; ++e) top = fmaxf(top, v[e]);
            top = counted(top);
            if (top > m) {
                m = top;
                at = x;
            }
        } else {
            add(v);
        }
    }
    if (!GREEDY && s != s) {  // NaN, or infinite logits: once more, with what they count as
        m = -INFINITY;
        s = 0.f;
        for (uint32_t x = x0 + tid; x < x1; x += 4u * kThreads) {
            float v[16];
            load_sixteen(row, x, x1, v);
#pragma unroll
            for (uint32_t e = 0; e < 16u; ++e) v[e] = counted(v[e]);
            add(v);
        }
    }
    float top = m;
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if constexpr (!GREEDY) s = warp_sum(m > -INFINITY ? s * exp2_fast((m - top) * a.rate) : 0.f);
    if (lane == 0u) sums[warp] = make_float2(top, s);
    if (GREEDY && tid == 0u) first = kNone;
    __syncthreads();
    top = -INFINITY;
    for (uint32_t w = 0; w < kWarps; ++w) top = fmaxf(top, sums[w].x);
    if constexpr (GREEDY) {
        // who has the largest looks for it once more
        if (m == top && m > -INFINITY) {
            float v[16];
            load_sixteen(row, at, x1, v);
            uint32_t i = kNone;
#pragma unroll
            for (uint32_t e = 16; e-- > 0u;)
                if (counted(v[e]) == m) i = 4u * (at + (e >> 2) * kThreads) + (e & 3u) - row.shift;
            atomicMin(&first, i);
        }
        __syncthreads();
        if (tid == 0u) reinterpret_cast<uint64_t*>(a.stats)[blockIdx.x] = first == kNone ? 0u : pick_key(top, first);
    } else if (tid == 0u) {
        s = 0.f;
        for (uint32_t w = 0; w < kWarps; ++w)
            if (sums[w].x > -INFINITY) s += sums[w].y * exp2_fast((sums[w].x - top) * a.rate);
        a.stats[blockIdx.x] = make_float2(top, s);
    }
}

// The sequence's rows, or false (flagged).
__device__ __forceinline__ bool load_rows(const VerifyArgs& a, uint32_t s, uint32_t* first, uint32_t* n) {
    const uint32_t b = a.v.row_start[s], e = a.v.row_start[s + 1u];
    if (b > e || e > a.v.rows || e - b > a.v.max_rows) {
        if (threadIdx.x == 0u && a.st != nullptr) atomicOr(&a.st->flags, kErrArgument);
        return false;
    }
    *first = b;
    *n = e - b;
    return true;
}
__device__ __forceinline__ void write_ids(const VerifyArgs& a, uint32_t s, uint32_t t0, uint32_t n, const uint32_t* drafts,
                                          uint32_t taken, uint32_t next) {
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) a.ids[t0 + i] = i < taken ? drafts[i] : i == taken ? next : kNone;
    if (threadIdx.x == 0u) a.accepted[s] = taken;
}

__global__ void __launch_bounds__(kThreads) verify_greedy_kernel(const __grid_constant__ VerifyArgs a) {
    static_assert(kVerifyMaxRows <= kThreads, "a thread to a row");
    __shared__ uint32_t pick[kVerifyMaxRows], drafts[kVerifyMaxRows], end;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, s = blockIdx.x;
    uint32_t t0, n;
    const bool ok = load_rows(a, s, &t0, &n);
    if (tid == 0u) end = n - 1u;
    const bool mine = ok && tid + 1u < n;  // (inputs, while the first kernel runs)
    const uint32_t x = mine ? a.v.draft_ids[t0 + tid] : 0u;
    if (mine) drafts[tid] = x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!ok) return;
    if (n == 0u) {
        if (tid == 0u) a.accepted[s] = 0u;
        return;
    }
    for (uint32_t i = warp; i < n; i += kWarps) {
        const uint64_t* keys = reinterpret_cast<const uint64_t*>(a.stats) + static_cast<size_t>(t0 + i) * a.parts;
        uint64_t best = 0;
        for (uint32_t c = lane; c < a.parts; c += 32u) best = keys[c] > best ? keys[c] : best;
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t k = __shfl_xor_sync(0xFFFFFFFFu, static_cast<unsigned long long>(best), o);
            best = k > best ? k : best;
        }
        if (lane == 0u) pick[i] = best == 0u ? kNone : ~static_cast<uint32_t>(best);
    }
    __syncthreads();
    if (mine) {
        if (x >= a.v.vocab && a.st != nullptr) atomicOr(&a.st->flags, kErrArgument);
        if (x >= a.v.vocab || pick[tid] != x) atomicMin(&end, tid);
    }
    __syncthreads();
    write_ids(a, s, t0, n, drafts, end, pick[end]);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// 2^(d scale / 32) for d <= 0, by table (Tang's method): with d scale = 32 j + i + f, |f| <= 1/2, it is 2^j times
// 2^(i/32), from the table, times the Taylor series of e^(f ln 2 / 32), whose sixth power is below 3 10^-15.
// d scale no less than -32 * 1018.
__device__ __forceinline__ double exp64(double d, double scale, const double* table) {
    const double up = fma(d, scale, 6755399441055744.0);  // 1.5 2^52 rounds to a whole number
    const double f = fma(d, scale, 6755399441055744.0 - up);
    constexpr double c = 0.021660849392498290195;  // ln 2 / 32
    double p = fma(f, c * c * c * c * c / 120.0, c * c * c * c / 24.0);
    p = fma(f, p, c * c * c / 6.0);
    p = fma(f, p, c * c / 2.0);
    p = fma(f, p, c);
    p = fma(f, p, 1.0);
    const int k = __double2loint(up);
    const double e = p * table[k & 31];
    return __hiloint2double(__double2hiint(e) + ((k & ~31) << 15), __double2loint(e));
}

// What the tokens of a row weigh, in 64 bits.
struct Weights {
    const double* table;  // 2^(i/32), i < 32
    Row logits, probs;    // probs, where `cut`: taken off
    uint32_t without;     // a token without weight
    bool cut;
    float least;          // logits below it, whose weight is under 2^-500 of the largest, count as without
    float m;              // the largest
    double scale, inv_z;  // scale: 32 log2(e) / T
    template <bool CUT>
    __device__ __forceinline__ double of(float l, float q, uint32_t i) const {
        // (NaN becomes the least, infinity the largest)
        double e = exp64(static_cast<double>(fminf(fmaxf(l, least), m)) - static_cast<double>(m), scale, table);
        if constexpr (CUT) e = fma(e, inv_z, -static_cast<double>(fmaxf(q, 0.f)));
        return l >= least && (CUT ? __double2hiint(e) > 0 : i != without) ? e : 0.0;
    }
    __device__ __forceinline__ double at(uint32_t i) const {
        return cut ? of<true>(__ldg(logits.first + i), __ldg(probs.first + i), i) : of<false>(__ldg(logits.first + i), 0.f, i);
    }
};

// One warp: the sum over quads [x0, x1) of the row.
template <bool CUT>
__device__ __noinline__ double share_sum(const Weights& weights, uint32_t x0, uint32_t x1) {
    constexpr uint32_t kAtOnce = CUT ? 2 : 4;  // quads on their way
    const Weights w = weights;
    const uint32_t lane = threadIdx.x & 31u;
    double sum = 0.0;
    for (uint32_t x = x0 + lane; x < x1; x += 32u * kAtOnce) {
        float4 l[kAtOnce], q[kAtOnce];
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u) {
            l[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            q[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (x + 32u * u < x1) {
                l[u] = w.logits.load(x + 32u * u, -INFINITY);
                if (CUT) q[u] = w.probs.load(x + 32u * u, 0.f);
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u) {
            const uint32_t i = 4u * (x + 32u * u) - w.logits.shift;
            sum += (w.of<CUT>(l[u].x, q[u].x, i) + w.of<CUT>(l[u].y, q[u].y, i + 1u)) +
                   (w.of<CUT>(l[u].z, q[u].z, i + 2u) + w.of<CUT>(l[u].w, q[u].w, i + 3u));
        }
    }
    return warp_sum64(sum);
}
__device__ __forceinline__ double share_of(const Weights& w, uint32_t x0, uint32_t x1) {
    return w.cut ? share_sum<true>(w, x0, x1) : share_sum<false>(w, x0, x1);
}

constexpr uint32_t kSampleThreads = 512, kSampleWarps = kSampleThreads / 32u;
struct VerifyShared {
    double table[32];
    float row_m[kVerifyMaxRows];
    double row_z[kVerifyMaxRows];
    uint32_t drafts[kVerifyMaxRows];
    double warps[2][kSampleWarps], ctas[2][kMaxCtas];  // sums of the warps of this CTA, of all CTAs (two, taken in turns)
    uint32_t stop, last;
};
// Into the same place of CTA `rank` of the cluster.
__device__ __forceinline__ void store_cluster(double* p, uint32_t rank, double v) {
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
// Of n shares in order the first whose running sum passes `border`, or the last with any weight; `run`: the
// sum in front of the first, then of the one found.
__device__ __forceinline__ uint32_t owner_of(const double* shares, uint32_t n, double border, double* run) {
    uint32_t k = kNone;
    double up = *run;
    for (uint32_t i = 0; i < n; ++i) {
        const double x = shares[i];
        if (x > 0.0) {
            k = i;
            *run = up;
            if (up + x > border) break;
        }
        up += x;
    }
    return k;
}

// The whole cluster of a sequence.
__global__ void __launch_bounds__(kSampleThreads, 2) verify_sample_kernel(const __grid_constant__ VerifyArgs a, uint32_t ctas) {
    __shared__ VerifyShared sm;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, s = blockIdx.x / ctas, rank = cluster_rank();
    uint32_t t0, n;
    const bool ok = load_rows(a, s, &t0, &n);
    cluster_arrive();
    if (warp == 0u) sm.table[lane] = exp2(lane / 32.0);
    // what the inputs say of the thread's row's draft, while the first kernel runs
    static_assert(kVerifyMaxRows <= kSampleThreads, "a thread to a row");
    const bool mine = ok && tid + 1u < n;
    const uint32_t x = mine ? a.v.draft_ids[t0 + tid] : 0u;
    float logit = -INFINITY, u = 0.f, q = 1.f;
    if (mine) {
        sm.drafts[tid] = x;
        u = a.v.accept_u[t0 + tid];
        const size_t at = static_cast<size_t>(t0 + tid) * a.v.vocab + x;
        if (x < a.v.vocab) {
            logit = counted(a.v.logits[at]);
            if (a.v.draft_probs != nullptr) q = fmaxf(a.v.draft_probs[at], 0.f);
        }
    }
    const float sample_u = a.v.sample_u[s];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    cluster_wait();  // (no CTA writes into another before that one runs)
    if (!ok) return;
    if (n == 0u) {
        if (tid == 0u && rank == 0u) a.accepted[s] = 0u;
        return;
    }
    // the rows' parts
    for (uint32_t i = warp; i < n; i += kSampleWarps) {
        const float2* part = a.stats + static_cast<size_t>(t0 + i) * a.parts;
        float m = -INFINITY;
        for (uint32_t c = lane; c < a.parts; c += 32u) m = fmaxf(m, part[c].x);
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        double z = 0.0;  // (a lane can have many)
        for (uint32_t c = lane; c < a.parts; c += 32u)
            if (part[c].x > -INFINITY) z += static_cast<double>(part[c].y) * exp2_fast((part[c].x - m) * a.rate);
        z = warp_sum64(z);
        if (lane == 0u) {
            sm.row_m[i] = m;
            sm.row_z[i] = z;
        }
    }
    auto weights_of = [&](uint32_t i) {
        const size_t at = static_cast<size_t>(t0 + i) * a.v.vocab;
        const float m = sm.row_m[i];
        return Weights{sm.table, Row(a.v.logits, at, a.v.vocab), Row(a.v.draft_probs, at, a.v.vocab), kNone, false,
                       fmaxf(m - 500.f / a.rate, -3.402823466e38f), m, 32.0 * 1.4426950408889634074 * a.inv_t, 1.0};
    };
    // the quads of a row that warp k of all takes
    auto begin_of = [&](const Weights& w, uint32_t k) {
        const uint32_t quads = w.logits.quads(), each = (quads + ctas * kSampleWarps - 1u) / (ctas * kSampleWarps);
        return min(quads, k * each);
    };
    uint32_t turn = 0;
    // a row's sum, the same in every thread of the cluster: every CTA's goes to all of them
    auto total = [&](const Weights& w) {
        turn ^= 1u;
        const uint32_t k = rank * kSampleWarps + warp;
        const double sum = share_of(w, begin_of(w, k), begin_of(w, k + 1u));
        if (lane == 0u) sm.warps[turn][warp] = sum;
        __syncthreads();
        if (warp == 0u) {
            const double all = warp_sum64(lane < kSampleWarps ? sm.warps[turn][lane] : 0.0);
            if (lane < ctas) store_cluster(&sm.ctas[turn][rank], lane, all);
        }
        cluster_sync();
        double all = 0.0;
        for (uint32_t c = 0; c < ctas; ++c) all += sm.ctas[turn][c];
        return all;
    };
    // the first draft that is not taken (n - 1: all are)
    uint32_t taken = 0;
    while (true) {
        if (tid == 0u) sm.stop = 2u * (n - 1u);
        __syncthreads();
        if (mine && tid >= taken) {
            uint32_t what = 2u * tid + 1u;  // not taken
            if (x >= a.v.vocab) {
                if (a.st != nullptr) atomicOr(&a.st->flags, kErrArgument);
            } else {
                const float m = sm.row_m[tid], e = m > -INFINITY ? exp2_fast((logit - m) * a.rate) : 0.f;
                const double left = static_cast<double>(u) * q * sm.row_z[tid], right = e;
                // In units of 2^-24 the row's sum is off by no more than 298: a weight by 4 (the exponential) and its
                // exponent's three roundings, 2.1 a bit, of which those that weigh have log2(vocab) in the mean, 31 at
                // most; a thread's sum by 4 in the sixteen and 6 in each of up to kLongest / 4096 + 1 steps; a warp's by
                // 10, a CTA's by 13, a row's by 4, each brought to the largest on the way.  The draft's weight, of up
                // to 100 bits, is off by 212.
                constexpr double kOff = 1024.0 / (1 << 24);
                if (m == -INFINITY || left > right * (1.0 + kOff) + 1e-30) what = 2u * tid + 1u;
                else if (left < right * (1.0 - kOff) - 1e-30) what = kNone;
                else what = 2u * tid;  // open
            }
            if (what != kNone) atomicMin(&sm.stop, what);
        }
        __syncthreads();
        const uint32_t stop = sm.stop;
        taken = stop >> 1;
        if (taken == n - 1u || (stop & 1u)) break;
        // the row in 64 bits
        const Weights w = weights_of(taken);
        const double z = total(w);
        const uint32_t token = sm.drafts[taken];
        const double p = a.v.draft_probs != nullptr ? fmax(static_cast<double>(a.v.draft_probs[static_cast<size_t>(t0 + taken) * a.v.vocab + token]), 0.0) : 1.0;
        if (!(static_cast<double>(a.v.accept_u[t0 + taken]) * p < w.at(token) / z)) break;
        ++taken;
        if (taken == n - 1u) break;
    }
    // the next token
    const bool cut = taken + 1u < n;
    Weights w = weights_of(taken);
    double all = 0.0;
    if (cut && sm.row_m[taken] > -INFINITY) {
        if (a.v.draft_probs != nullptr) {
            w.inv_z = 1.0 / total(w);
            w.cut = true;
        } else {
            w.without = sm.drafts[taken];
        }
        all = total(w);
        if (!(all > 0.0)) {  // nothing left: from p itself
            w.cut = false;
            w.without = kNone;
        }
    }
    if (!(all > 0.0) && sm.row_m[taken] > -INFINITY) all = total(w);
    if (!(all > 0.0)) {
        if (rank == 0u) write_ids(a, s, t0, n, sm.drafts, taken, kNone);
        return;
    }
    // the CTA and the warp whose share holds the border; the CTA goes through that once more, a run of
    // tokens to a thread
    const double border = static_cast<double>(sample_u) * all;
    double run = 0.0;
    if (owner_of(sm.ctas[turn], ctas, border, &run) != rank) return;  // (nobody reads what is here any more)
    const uint32_t owner = rank * kSampleWarps + owner_of(sm.warps[turn], kSampleWarps, border, &run);
    const uint32_t shift = w.logits.shift, from = max(4u * begin_of(w, owner), shift) - shift;
    const uint32_t to = min(4u * begin_of(w, owner + 1u) - shift, a.v.vocab), each = (to - from + kSampleThreads - 1u) / kSampleThreads;
    const uint32_t i0 = min(to, from + tid * each), i1 = min(to, i0 + each);
    if (tid == 0u) {
        sm.stop = kNone;
        sm.last = 0u;
    }
    double sum = 0.0;
    uint32_t last = 0;
    for (uint32_t i = i0; i < i1; ++i) {
        const double e = w.at(i);
        sum += e;
        if (e > 0.0) last = i;
    }
    double pre = sum;
#pragma unroll
    for (uint32_t o = 1; o < 32u; o <<= 1) {
        const double up = __shfl_up_sync(0xFFFFFFFFu, pre, o);
        if (lane >= o) pre += up;
    }
    turn ^= 1u;
    if (lane == 31u) sm.warps[turn][warp] = pre;
    __syncthreads();
    for (uint32_t k = 0; k < warp; ++k) run += sm.warps[turn][k];
    if (sum > 0.0) {
        atomicMax(&sm.last, last);
        if (run + pre > border) {
            run += pre - sum;
            uint32_t hit = last;
            for (uint32_t i = i0; i < i1; ++i) {
                const double e = w.at(i);
                run += e;
                if (e > 0.0 && run > border) {
                    hit = i;
                    break;
                }
            }
            atomicMin(&sm.stop, hit);
        }
    }
    __syncthreads();
    write_ids(a, s, t0, n, sm.drafts, taken, sm.stop != kNone ? sm.stop : sm.last);
}

// CTAs of a sequence's cluster: all that run at once for few sequences, but no warp with less than four
// loads of a lane.
uint32_t sample_ctas(const VerifyDrafts& v) {
    const uint32_t work = (v.vocab + 8191u) / 8192u;
    uint32_t c = 1;
    while (c < kMaxCtas && c < work && static_cast<uint64_t>(v.seqs) * c < 148u) c *= 2u;
    return c;
}

// Parts of a row: as many CTAs as run at once, but no part smaller than two loads of a thread, nor longer than the
// bound on its sum allows for.
constexpr uint32_t kLongest = 32u * 16u * kThreads;
uint32_t parts_of(const VerifyDrafts& v, uint32_t* chunk) {
    constexpr uint32_t kRound = 4u * kThreads;
    const uint64_t most = (static_cast<uint64_t>(v.vocab) + 2u * kRound - 1u) / (2u * kRound);
    const uint64_t want = std::min<uint64_t>(most, std::max<uint64_t>(1u, 8u * 148u / v.rows));
    const uint64_t each = (v.vocab + want - 1u) / want;
    *chunk = static_cast<uint32_t>(std::min<uint64_t>((each + kRound - 1u) / kRound * kRound, kLongest));
    return static_cast<uint32_t>((static_cast<uint64_t>(v.vocab) + *chunk - 1u) / *chunk);
}

}  // namespace

uint64_t verify_drafts_workspace(const VerifyDrafts& v) {
    uint32_t chunk;
    return static_cast<uint64_t>(v.rows) * parts_of(v, &chunk) * sizeof(float2);
}

cudaError_t launch_verify_drafts(const VerifyDrafts& v, float temperature, uint32_t* accepted, uint32_t* ids, void* workspace,
                                 DeviceStatus* st, cudaStream_t stream) {
    VerifyArgs a = {};
    a.v = v;
    a.rate = temperature > 0.f ? static_cast<float>(1.4426950408889634 / temperature) : 0.f;
    a.inv_t = temperature > 0.f ? 1.0 / temperature : 0.0;
    a.parts = parts_of(v, &a.chunk);
    a.stats = static_cast<float2*>(workspace);
    a.accepted = accepted;
    a.ids = ids;
    a.st = st;
    const uint64_t grid = static_cast<uint64_t>(v.rows) * a.parts;
    if (grid > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    if (temperature > 0.f) verify_stats_kernel<false><<<static_cast<uint32_t>(grid), kThreads, 0, stream>>>(a);
    else verify_stats_kernel<true><<<static_cast<uint32_t>(grid), kThreads, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const uint32_t ctas = temperature > 0.f ? sample_ctas(v) : 1u;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(v.seqs * ctas);
    cfg.blockDim = dim3(temperature > 0.f ? kSampleThreads : kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = temperature > 0.f ? 2 : 1;
    if (temperature > 0.f) return cudaLaunchKernelEx(&cfg, verify_sample_kernel, a, ctas);
    return cudaLaunchKernelEx(&cfg, verify_greedy_kernel, a);
}

}  // namespace nedo_gpu

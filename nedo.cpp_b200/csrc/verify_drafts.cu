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
// largest logit and the sum of 2^((l - m) log2(e) / T), in 32 bits.  The second, a cluster of CTAs per
// sequence, adds the parts and decides: with the sums within 2^-14 (17 + 17 roundings of an exponent
// of up to 17 that carries weight, those of up to 2^7 additions, 2^-22 of the exponential), a draft
// whose two sides differ by more is decided, any other is looked at again with the row summed in 64
// bits.  Then the one row that the next token comes from is read again, from L2, in 64 bits: a token
// of a large vocabulary can be 10^-6 of the whole, and u falls on the border of two in 32 bits
// every so often.  Every warp has a part of the tokens in order; the warp whose part holds the border
// goes through it once more.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace nedo_gpu {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32u;
constexpr uint32_t kMaxCtas = 8;       // of a cluster
constexpr uint32_t kStep = kThreads * 16u;  // logits that a CTA has on their way at once
constexpr uint32_t kNone = 0xFFFFFFFFu;

// NaN counts as minus infinity, infinity as the largest number.
__device__ __forceinline__ float counted(float l) { return fminf(fmaxf(l, -INFINITY), 3.402823466e38f); }

struct VerifyArgs {
    VerifyDrafts v;
    float rate;          // log2(e) / T
    double inv_t;
    uint32_t chunk;      // logits per part, a multiple of kStep
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

// Four numbers of a row from its element 4 x - shift on (those before the row's first and behind its
// last count as minus infinity): the row begins `shift` elements behind a 16-byte border.
__device__ __forceinline__ float4 load_quad(const float* row, uint32_t shift, uint32_t x, uint32_t from, uint32_t to) {
    const int64_t i = static_cast<int64_t>(4u) * x - shift;
    if (i >= static_cast<int64_t>(from) && i + 4 <= static_cast<int64_t>(to)) return __ldg(reinterpret_cast<const float4*>(row + i));
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = -INFINITY;
        if (i + e >= static_cast<int64_t>(from) && i + e < static_cast<int64_t>(to)) v[e] = __ldg(row + i + e);
    }
    return make_float4(v[0], v[1], v[2], v[3]);
}

template <bool GREEDY>
__global__ void __launch_bounds__(kThreads) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
    __shared__ float2 sums[kWarps];
    __shared__ uint64_t keys[kWarps];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    asm volatile("griddepcontrol.launch_dependents;");
    const size_t at = static_cast<size_t>(r) * a.v.vocab;
    const float* row = a.v.logits + at;
    const uint32_t shift = static_cast<uint32_t>(at & 3u);
    const uint32_t from = part * a.chunk, to = min(a.v.vocab, from + a.chunk);
    // (the parts' borders are 16-byte borders but for the shift: both sides read the quad on it)
    const uint32_t x0 = (from + shift) / 4u, x1 = (to + shift + 3u) / 4u;
    float m = -INFINITY, s = 0.f;
    uint64_t key = 0;
    for (uint32_t x = x0 + tid; x < x1; x += 4u * kThreads) {
        float4 q[4];
#pragma unroll
        for (uint32_t u = 0; u < 4u; ++u) {
            q[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (x + u * kThreads < x1) q[u] = load_quad(row, shift, x + u * kThreads, from, to);
        }
        float v[16], top = -INFINITY;
#pragma unroll
        for (uint32_t u = 0; u < 4u; ++u) {
            v[4 * u] = counted(q[u].x);
            v[4 * u + 1] = counted(q[u].y);
            v[4 * u + 2] = counted(q[u].z);
            v[4 * u + 3] = counted(q[u].w);
        }
        if constexpr (GREEDY) {
#pragma unroll
            for (uint32_t e = 0; e < 16u; ++e) {
                // (in ascending order: the first of equal ones stays)
                const uint32_t i = 4u * (x + (e >> 2) * kThreads) + (e & 3u) - shift;
                if (v[e] > m) {
                    m = v[e];
                    key = pick_key(v[e], i);
                }
            }
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 16u; ++e) top = fmaxf(top, v[e]);
            if (top > m) {
                s *= exp2_fast((m - top) * a.rate);
                m = top;
            }
            if (m > -INFINITY)
#pragma unroll
                for (uint32_t e = 0; e < 16u; ++e) s += exp2_fast((v[e] - m) * a.rate);
        }
    }
    if constexpr (GREEDY) {
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t k = __shfl_xor_sync(0xFFFFFFFFu, static_cast<unsigned long long>(key), o);
            key = k > key ? k : key;
        }
        if (lane == 0u) keys[warp] = key;
    } else {
        float top = m;
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        s = warp_sum(m > -INFINITY ? s * exp2_fast((m - top) * a.rate) : 0.f);
        if (lane == 0u) sums[warp] = make_float2(top, s);
    }
    __syncthreads();
    if (tid != 0u) return;
    if constexpr (GREEDY) {
        key = 0;
        for (uint32_t w = 0; w < kWarps; ++w) key = keys[w] > key ? keys[w] : key;
        reinterpret_cast<uint64_t*>(a.stats)[blockIdx.x] = key;
    } else {
        float top = -INFINITY;
        for (uint32_t w = 0; w < kWarps; ++w) top = fmaxf(top, sums[w].x);
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
__device__ __forceinline__ void write_ids(const VerifyArgs& a, uint32_t s, uint32_t t0, uint32_t n, uint32_t taken, uint32_t next) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads)
        a.ids[t0 + i] = i < taken ? a.v.draft_ids[t0 + i] : i == taken ? next : kNone;
    if (threadIdx.x == 0u) a.accepted[s] = taken;
}

__global__ void __launch_bounds__(kThreads) verify_greedy_kernel(const __grid_constant__ VerifyArgs a) {
    __shared__ uint32_t pick[kVerifyMaxRows], end;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, s = blockIdx.x;
    uint32_t t0, n;
    const bool ok = load_rows(a, s, &t0, &n);
    if (tid == 0u) end = n - 1u;
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
    for (uint32_t i = tid; i + 1u < n; i += kThreads) {
        const uint32_t x = a.v.draft_ids[t0 + i];
        if (x >= a.v.vocab && a.st != nullptr) atomicOr(&a.st->flags, kErrArgument);
        if (x >= a.v.vocab || pick[i] != x) atomicMin(&end, i);
    }
    __syncthreads();
    write_ids(a, s, t0, n, end, pick[end]);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ double load_cluster(const double* p, uint32_t rank) {
    uint32_t addr;
    double v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// What the tokens of a row weigh, in 64 bits.
struct Weights {
    const float* logits;
    const float* probs;  // null: nothing taken off, but from token `without`
    uint32_t without;
    float m;
    double inv_t, inv_z;
    __device__ __forceinline__ double operator()(uint32_t i) const {
        const float l = counted(__ldg(logits + i));
        double e = m > -INFINITY ? exp((static_cast<double>(l) - m) * inv_t) : 0.0;
        if (probs != nullptr) e = fmax(e * inv_z - fmax(static_cast<double>(__ldg(probs + i)), 0.0), 0.0);
        return i == without ? 0.0 : e;
    }
};

struct VerifyShared {
    float row_m[kVerifyMaxRows];
    double row_z[kVerifyMaxRows];
    double totals[2][kWarps];  // of the warps' parts (two, taken in turns)
    uint32_t stop;
};

// A row's sum, the same in every thread of the cluster, and what makes it up: lane k of every warp
// has the shares of warps k and k + 32 of the cluster and the sums up to and with them.
struct Total {
    double all, share[2], upto[2];
};
// Every warp takes tokens [begin, end); `mine`: the CTA's warps' shares.
__device__ __forceinline__ Total row_total(const Weights& w, uint32_t begin, uint32_t end, double* mine, uint32_t ctas) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    double sum = 0.0;
#pragma unroll 4
    for (uint32_t i = begin + lane; i < end; i += 32u) sum += w(i);
    sum = warp_sum64(sum);
    if (lane == 0u) mine[warp] = sum;
    cluster_sync();
    Total t;
    t.all = 0.0;
#pragma unroll
    for (uint32_t h = 0; h < 2u; ++h) {
        const uint32_t k = lane + 32u * h;
        t.share[h] = k < ctas * kWarps ? load_cluster(mine + k % kWarps, k / kWarps) : 0.0;
    }
#pragma unroll
    for (uint32_t h = 0; h < 2u; ++h) {
        double up = t.share[h];
#pragma unroll
        for (uint32_t o = 1; o < 32u; o <<= 1) {
            const double x = __shfl_up_sync(0xFFFFFFFFu, up, o);
            if (lane >= o) up += x;
        }
        t.upto[h] = t.all + up;
        t.all = __shfl_sync(0xFFFFFFFFu, t.upto[h], 31);
    }
    return t;
}

// The whole cluster of a sequence.
__global__ void __launch_bounds__(kThreads) verify_sample_kernel(const __grid_constant__ VerifyArgs a, uint32_t ctas) {
    __shared__ VerifyShared sm;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, s = blockIdx.x / ctas, rank = cluster_rank();
    uint32_t t0, n;
    const bool ok = load_rows(a, s, &t0, &n);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!ok) return;
    if (n == 0u) {
        if (tid == 0u && rank == 0u) a.accepted[s] = 0u;
        return;
    }
    // the rows' parts
    for (uint32_t i = warp; i < n; i += kWarps) {
        const float2* part = a.stats + static_cast<size_t>(t0 + i) * a.parts;
        float m = -INFINITY;
        for (uint32_t c = lane; c < a.parts; c += 32u) m = fmaxf(m, part[c].x);
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        float z = 0.f;
        for (uint32_t c = lane; c < a.parts; c += 32u)
            if (part[c].x > -INFINITY) z += part[c].y * exp2_fast((part[c].x - m) * a.rate);
        z = warp_sum(z);
        if (lane == 0u) {
            sm.row_m[i] = m;
            sm.row_z[i] = z;
        }
    }
    // this warp's tokens
    const uint32_t share = (a.v.vocab + ctas * kWarps - 1u) / (ctas * kWarps);
    const uint32_t begin = min(a.v.vocab, (rank * kWarps + warp) * share), end = min(a.v.vocab, begin + share);
    uint32_t turn = 0;
    auto total = [&](const Weights& w) {
        double* mine = sm.totals[turn];
        turn ^= 1u;
        return row_total(w, begin, end, mine, ctas);
    };
    auto weights_of = [&](uint32_t i) {
        const size_t at = static_cast<size_t>(t0 + i) * a.v.vocab;
        return Weights{a.v.logits + at, nullptr, kNone, sm.row_m[i], a.inv_t, 1.0};
    };
    // the first draft that is not taken (n - 1: all are)
    uint32_t taken = 0;
    while (true) {
        if (tid == 0u) sm.stop = 2u * (n - 1u);
        __syncthreads();
        for (uint32_t i = taken + tid; i + 1u < n; i += kThreads) {
            const uint32_t x = a.v.draft_ids[t0 + i];
            uint32_t what = 2u * i + 1u;  // not taken
            if (x >= a.v.vocab) {
                if (a.st != nullptr) atomicOr(&a.st->flags, kErrArgument);
            } else {
                const size_t at = static_cast<size_t>(t0 + i) * a.v.vocab + x;
                const float m = sm.row_m[i], e = m > -INFINITY ? exp2_fast((counted(a.v.logits[at]) - m) * a.rate) : 0.f;
                const float q = a.v.draft_probs != nullptr ? fmaxf(a.v.draft_probs[at], 0.f) : 1.f;
                const double left = static_cast<double>(a.v.accept_u[t0 + i]) * q * sm.row_z[i], right = e;
                constexpr double kOff = 1.0 / 16384.0;
                if (m == -INFINITY || left > right * (1.0 + kOff) + 1e-30) what = 2u * i + 1u;
                else if (left < right * (1.0 - kOff) - 1e-30) what = kNone;
                else what = 2u * i;  // open
            }
            if (what != kNone) {
                atomicMin(&sm.stop, what);
                break;
            }
        }
        __syncthreads();
        const uint32_t stop = sm.stop;
        taken = stop >> 1;
        if (taken == n - 1u || (stop & 1u)) break;
        // the row in 64 bits
        const Weights w = weights_of(taken);
        const double z = total(w).all;
        const uint32_t x = a.v.draft_ids[t0 + taken];
        const double q = a.v.draft_probs != nullptr ? fmax(static_cast<double>(a.v.draft_probs[static_cast<size_t>(t0 + taken) * a.v.vocab + x]), 0.0) : 1.0;
        if (!(static_cast<double>(a.v.accept_u[t0 + taken]) * q < w(x) / z)) break;
        ++taken;
        if (taken == n - 1u) break;
    }
    // the next token
    const bool cut = taken + 1u < n;
    Weights w = weights_of(taken);
    Total t;
    t.all = 0.0;
    if (cut && w.m > -INFINITY) {
        if (a.v.draft_probs != nullptr) {
            w.inv_z = 1.0 / total(w).all;
            w.probs = a.v.draft_probs + static_cast<size_t>(t0 + taken) * a.v.vocab;
        } else {
            w.without = a.v.draft_ids[t0 + taken];
        }
        t = total(w);
        if (!(t.all > 0.0)) {  // nothing left: from p itself
            w.probs = nullptr;
            w.without = kNone;
        }
    }
    if (!(t.all > 0.0) && w.m > -INFINITY) t = total(w);
    uint32_t next = kNone;
    bool mine = rank == 0u;  // the CTA that writes
    if (t.all > 0.0) {
        // the warp whose share holds the border: the first whose running sum passes it, or the last
        // with any weight
        const double border = static_cast<double>(a.v.sample_u[s]) * t.all;
        uint32_t some[2], hits[2];
#pragma unroll
        for (uint32_t h = 0; h < 2u; ++h) {
            some[h] = __ballot_sync(0xFFFFFFFFu, t.share[h] > 0.0);
            hits[h] = __ballot_sync(0xFFFFFFFFu, t.share[h] > 0.0 && t.upto[h] > border);
        }
        const bool passed = (hits[0] | hits[1]) != 0u;
        const uint32_t owner = passed ? (hits[0] != 0u ? __ffs(hits[0]) - 1u : 31u + __ffs(hits[1]))
                                      : (some[1] != 0u ? 63u - __clz(some[1]) : 31u - __clz(some[0]));
        // the running sum in front of it
        const uint32_t prev = owner == 0u ? 0u : owner - 1u;
        const double upto = __shfl_sync(0xFFFFFFFFu, prev >= 32u ? t.upto[1] : t.upto[0], prev & 31u);
        const double before = owner == 0u ? 0.0 : upto;
        mine = owner / kWarps == rank;
        if (owner == rank * kWarps + warp) {
            uint32_t last = kNone;
            double sum = before;
            for (uint32_t i0 = begin; i0 < end; i0 += 32u) {
                const double e = i0 + lane < end ? w(i0 + lane) : 0.0;
                double pre = e;
#pragma unroll
                for (uint32_t o = 1; o < 32u; o <<= 1) {
                    const double up = __shfl_up_sync(0xFFFFFFFFu, pre, o);
                    if (lane >= o) pre += up;
                }
                const uint32_t some = __ballot_sync(0xFFFFFFFFu, e > 0.0);
                if (some != 0u) last = i0 + 31u - __clz(some);
                const uint32_t hit = __ballot_sync(0xFFFFFFFFu, e > 0.0 && sum + pre > border);
                if (passed && hit != 0u) {
                    last = i0 + __ffs(hit) - 1u;
                    break;
                }
                sum += __shfl_sync(0xFFFFFFFFu, pre, 31);
            }
            if (lane == 0u) sm.stop = last;
        }
        __syncthreads();
        next = sm.stop;
    }
    if (mine) write_ids(a, s, t0, n, taken, next);
    cluster_sync();  // no CTA leaves while another still reads its sums
}

// CTAs of a sequence's cluster.
uint32_t sample_ctas(const VerifyDrafts& v) {
    const uint32_t work = (v.vocab + 4095u) / 4096u;
    uint32_t c = 1;
    while (c < kMaxCtas && c < work && static_cast<uint64_t>(v.seqs) * c < 4u * 148u) c *= 2u;
    return c;
}

// Parts of a row: as many CTAs as run at once, but no part smaller than what one has on its way.
uint32_t parts_of(const VerifyDrafts& v, uint32_t* chunk) {
    const uint64_t want = std::max<uint64_t>(1u, (8u * 148u + v.rows - 1u) / std::max(v.rows, 1u));
    const uint64_t steps = (static_cast<uint64_t>(v.vocab) + kStep - 1u) / kStep;
    const uint64_t per = (steps + want - 1u) / want;
    *chunk = static_cast<uint32_t>(std::min<uint64_t>(per * kStep, 0x40000000u));
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
    cfg.blockDim = dim3(kThreads);
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

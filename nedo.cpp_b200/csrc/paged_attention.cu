// paged_attention.cu -- softmax attention of a ragged batch of query rows over a
// paged KV cache (the attention step of src/model.cpp:226-247 for many
// sequences), dense (causal, optional sliding window, optional prefix of pages
// that all sequences share) or over a list of pages per query token and KV head.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale * log2(e) * q.k_j
//
// in one pass over the keys with a running maximum m.  Sums and statistics are in 32 bits; the
// factors that the tensor cores multiply are split in two fp16 halves, 22 bits.  A
// work item is a tile of query rows of one KV head (the heads of its group next
// to each other, so a key is read once for all of them) times a chunk of keys.
// With one chunk per row the item writes the output; otherwise it writes
// (sum_j p_j v_j, m, sum_j p_j) of its chunk, and attention_combine_kernel adds a
// row's chunks in order, so results repeat bit for bit.  The shared prefix is a
// part of its own, whose row tiles run across all sequences: its keys are read
// once for the whole batch.
#include <algorithm>

#include "paged_attention.cuh"

namespace nedo_gpu {
namespace {

// ---- adding a row's chunks ---------------------------------------------------
struct CombineArgs {
    PagedKv kv;
    PagedBatch b;
    float* out;
    const float* part_o;
    const float2* part_ml;
    uint32_t heads, window, shared_len;
    uint32_t own_chunk, own_chunks, prefix_chunk, prefix_chunks;
    uint32_t few_rows, few_chunk;        // sequences of at most few_rows rows have chunks of their own
    uint32_t own_direct, few_direct;     // written out already
    uint32_t group, heads_per_cta;
    uint32_t blocks;  // the sparse call: every slot is written
    const uint32_t* chunk_at;  // the own part's chunks follow from the lengths (null: own_chunk)
};

// One CTA per token and head (per token where most rows are done already).  The maximum over the
// row's chunks first, then in blocks of kCombineThreads chunks their weights 2^(m_i - m) into
// shared memory, and the weighted sum with head_dim / 4 threads to a chunk and as many chunks at once as the CTA holds,
// four loads in flight each; the groups' sums meet in group order.  A chunk in which the
// row sees nothing has weight sum 0 and may hold anything.  Launched so that it comes up
// while the last work items run; it waits for their sums before it reads them.
constexpr uint32_t kCombineThreads = 128;
__global__ void __launch_bounds__(kCombineThreads) attention_combine_kernel(CombineArgs a) {
    __shared__ float wt[kCombineThreads], red[kCombineThreads / 32u];
    __shared__ float4 sums[kCombineThreads];
    const size_t rows_all = static_cast<size_t>(a.b.tokens) * a.heads;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t per_token = a.heads / a.heads_per_cta;  // CTAs
    const uint32_t t = blockIdx.x / per_token;
    const uint32_t s = seq_of_token(a.b, t);
    PagedSeq sq{0u, 0u, 0u};
    if (s != kNone) sq = load_seq(a.b, s, nullptr);
    const int p = sq.n != 0u ? sq.pos(t - sq.t0) : -1;
    const bool few = sq.n * a.group <= a.few_rows;
    const uint32_t chunk = few ? a.few_chunk : a.own_chunk;
    // the row's slots: [b0, e0) of the prefix, [b1, e1) of its own keys
    uint32_t b0 = 0, e0 = 0, b1 = 0, e1 = 0;
    if (a.blocks) {
        if (p >= 0) e1 = a.own_chunks;
    } else if (p >= 0) {
        const uint32_t lo = first_key(p, a.window), hi = static_cast<uint32_t>(p) + 1u;
        if (a.prefix_chunks != 0u && lo < a.shared_len) {
            b0 = lo / a.prefix_chunk;
            e0 = (min(hi, a.shared_len) + a.prefix_chunk - 1u) / a.prefix_chunk;
        }
        if (hi > a.shared_len) {
            const uint32_t begin = own_begin(sq, a.window, a.shared_len);
            b1 = a.prefix_chunks + (max(lo, begin) - begin) / chunk;
            e1 = a.prefix_chunks + (hi - 1u - begin) / chunk + 1u;
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (a.chunk_at != nullptr && e1 != 0u) {
        const uint32_t n = *a.chunk_at, begin = own_begin(sq, a.window, a.shared_len);
        b1 = a.prefix_chunks + (max(first_key(p, a.window), begin) - begin) / n;
        e1 = a.prefix_chunks + (static_cast<uint32_t>(p) - begin) / n + 1u;
    }
    if (sq.n == 0u || (few ? a.few_direct : a.own_direct)) return;  // no row of any sequence, or done
    const uint32_t n0 = e0 - b0, n = n0 + (e1 - b1);
    for (uint32_t h = 0; h < a.heads_per_cta; ++h) {
        const size_t row = static_cast<size_t>(t) * a.heads + (blockIdx.x % per_token) * a.heads_per_cta + h;
        const float2* ml = a.part_ml + row;
        auto slot = [&](uint32_t i) -> size_t { return i < n0 ? b0 + i : b1 + (i - n0); };
        float m = -INFINITY;
        for (uint32_t i = tid; i < n; i += kCombineThreads) {
            const float2 x = ml[slot(i) * rows_all];
            if (x.y != 0.f) m = fmaxf(m, x.x);
        }
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        __syncthreads();
        if (lane == 0u) red[warp] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const uint32_t hd = a.kv.head_dim, hd4 = hd / 4u, groups = kCombineThreads / hd4;
        const uint32_t grp = tid / hd4, d = tid - grp * hd4;
        float l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t i0 = 0; i0 < n; i0 += kCombineThreads) {
            const uint32_t cnt = min(kCombineThreads, n - i0);
            __syncthreads();
            float w = -1.f;  // nothing seen there
            if (tid < cnt) {
                const float2 x = ml[slot(i0 + tid) * rows_all];
                if (x.y != 0.f) {
                    w = exp2f(x.x - m);
                    l = fmaf(x.y, w, l);
                }
            }
            wt[tid] = w;
            __syncthreads();
            if (grp < groups) {
#pragma unroll 4
                for (uint32_t i = grp; i < cnt; i += groups) {
                    const float f = wt[i];
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (f != -1.f)  // (also where the weight is nothing: an infinite value is not passed over)
                        x = *reinterpret_cast<const float4*>(a.part_o + (slot(i0 + i) * rows_all + row) * hd + 4u * d);
                    acc.x = fmaf(x.x, f, acc.x);
                    acc.y = fmaf(x.y, f, acc.y);
                    acc.z = fmaf(x.z, f, acc.z);
                    acc.w = fmaf(x.w, f, acc.w);
                }
            }
        }
        l = warp_sum(l);
        __syncthreads();
        if (lane == 0u) red[warp] = l;
        sums[tid] = acc;
        __syncthreads();
        if (tid < hd4) {
            l = (red[0] + red[1]) + (red[2] + red[3]);
            for (uint32_t k = 1; k < groups; ++k) {
                const float4 x = sums[k * hd4 + tid];
                acc.x += x.x;
                acc.y += x.y;
                acc.z += x.z;
                acc.w += x.w;
            }
            const bool none = l == 0.f;
            *reinterpret_cast<float4*>(a.out + row * hd + 4u * tid) =
                none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc.x / l, acc.y / l, acc.z / l, acc.w / l);
        }
    }
}

// Which kernel takes a part, and what its work items cost (for the plan).
enum class Kernel { kFew, kFew16, kFew32, kFew4, kFew4x8, kFew4x16, kMany, kMany64, kMany32, kTc };
struct Cost {
    uint32_t rows;       // query rows per tile
    uint32_t slots;      // work items that run at once on 148 SMs
    uint32_t max_chunk;  // keys an item can take (0: any number)
    double ns_per_key, ns_fixed;
    double least;        // share of ns_per_key that an item takes on its own
};
Cost cost_of(Kernel k, const PagedKv& kv) {
    const uint32_t hd = kv.head_dim;
    switch (k) {
        case Kernel::kFew:
        case Kernel::kFew16: {  // reads 4 hd bytes per key of the SMs' common 6.5 TB/s
            const uint32_t slots = 148u * (hd <= 64u ? 4u : hd <= 128u ? 2u : 1u);
            return {k == Kernel::kFew ? kFewRows : 2u * kFewRows, slots, 2048u, 4.0 * hd * slots / 6500.0, 4000.0, 0.45};
        }
        // 128 or 64 rows of a head above 128 through the tensor cores, an item to an SM (148 items of 128
        // rows: 79, 134, 242 and 463 us over 500, 1000, 2000 and 4000 keys; of 64: 51, 90, 163 and 310)
        case Kernel::kMany:
            return {128u, 148u, 0u, 110.0, 24000.0, 1.0};
        case Kernel::kMany64:
            return {64u, 148u, 0u, 74.0, 14000.0, 1.0};
        case Kernel::kTc:  // 128 rows through 32 MMAs per 128 keys, an item to an SM; 24,000 cycles around its tiles
            return {kTcRows, 148u, 0u, hd <= 64u ? 8.0 : 12.0, 12000.0, 1.0};
        case Kernel::kFew32: {
            const uint32_t slots = 148u * (hd <= 64u ? 4u : hd <= 128u ? 2u : 1u);
            return {kFewRows, slots, 2048u, 8.0 * hd * slots / 6500.0, 4000.0, 0.45};
        }
        case Kernel::kFew4:
        case Kernel::kFew4x8:
        case Kernel::kFew4x16: {
            // bound by its instructions (1.125 hd bytes per key): what runs at once on an SM takes 5.1, 6.0 and
            // 8.7 ns a key at 4, 8 and 16 rows of 128 channels, one alone three quarters of its share
            const uint32_t rows = k == Kernel::kFew4 ? 4u : k == Kernel::kFew4x8 ? 8u : 16u;
            const uint32_t slots = 148u * (hd > 128u ? 2u : rows == 16u ? 3u : 4u);
            const double ns = rows == 16u ? 26.0 : rows == 8u ? 24.0 : 20.5;
            return {rows, slots, 2048u, ns * hd / 128.0, rows == 16u ? 6000.0 : 4500.0, 0.75};
        }
        default:  // kMany32: three products each way
            return {many32_rows(hd), 148u, 0u, hd <= 64u ? 24.0 : 48.0, 5000.0, 1.0};
    }
}

// Keys per work item, a multiple of 64 and of the page size: of the chunkings that fill
// one, two, ... rounds of items the one with the least estimated time, the fixed cost of an
// item and the bytes of the chunks' sums counted.
// `cluster`: up to kMaxCluster chunks of a row tile can be added within a cluster, without the
// combining kernel.
// `joined`: a prefix makes the combining kernel necessary in any case.
// `causal`: share of its keys by which a sequence's first rows see fewer than its last.  Where
// items are of equal length (0) they run in whole rounds; where they are not, the long ones come
// first and the short ones even them out.
struct Chunks {
    uint32_t keys;
    double ns;  // estimated time
};
Chunks chunk_keys(uint64_t keys, uint64_t units, uint64_t sum_bytes, const PagedKv& kv, const Cost& c, bool cluster,
                  double causal = 0.0, bool joined = false) {
    const uint64_t step = std::max(64u, kv.page_size);
    keys = std::max<uint64_t>(keys, 1u);
    auto rounded = [&](uint64_t n) { return ((keys + n - 1u) / n + step - 1u) / step * step; };
    uint64_t best = 0;
    double best_ns = 0.0;
    auto consider = [&](uint64_t n) {
        uint64_t chunk = rounded(n);
        if (c.max_chunk != 0u && chunk > c.max_chunk) chunk = c.max_chunk / step * step;
        n = (keys + chunk - 1u) / chunk;
        const double rounds = static_cast<double>((units * n + c.slots - 1u) / c.slots);
        // a chunk's sums are written once and read once at about half the copy rate
        // few items do not share the memory's rate, but one alone has only its own copies in flight
        const double busy = std::min(1.0, static_cast<double>(units * n) / c.slots);
        const double item = static_cast<double>(chunk) * c.ns_per_key * std::max(busy, c.least) + c.ns_fixed;
        const double all = units * (static_cast<double>(keys) * (1.0 - 0.5 * causal) * c.ns_per_key + n * c.ns_fixed);
        const double ns = (1.0 - causal) * rounds * item + causal * std::max(item, all / c.slots) +
                          (n == 1u                          ? 0.0
                           : cluster && n <= kMaxCluster ? 1000.0
                                                         : (joined ? 0.0 : 4000.0) + static_cast<double>(n * sum_bytes) * 2.0 / 3000.0);
        if (best == 0u || ns < best_ns) {
            best = chunk;
            best_ns = ns;
        }
    };
    for (uint64_t n = 1; n <= (cluster ? kMaxCluster : 1u); ++n) consider(n);
    for (uint64_t rounds = 1; rounds <= 12u; ++rounds) {
        const uint64_t n = rounds * c.slots / units;
        if (n > 1u) consider(std::min<uint64_t>(n, (keys + step - 1u) / step));
    }
    return {static_cast<uint32_t>(best), best_ns};
}

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1u) / b; }

// Row tiles of the own part: every sequence has whole tiles.
uint64_t own_tiles(const PagedAttention& a, uint32_t rows) {
    const uint64_t group = a.heads / a.kv.kv_heads;
    return std::min<uint64_t>(a.b.tokens * group / rows + a.b.seqs, a.b.seqs * ceil_div(a.b.max_q_len * group, rows));
}

// The kernel of a part whose row tiles have up to `rows` rows.
Kernel kernel_for(const PagedKv& kv, uint64_t rows) {
    if (kv.type == kQ4_0 && rows <= kFewMax)
        return rows <= 4u ? Kernel::kFew4 : rows <= 8u || kv.head_dim > 128u ? Kernel::kFew4x8 : Kernel::kFew4x16;
    if (kv.type == kF32) return rows <= kFewMax ? Kernel::kFew32 : Kernel::kMany32;
    if (rows <= kFewRows || (rows <= kFewMax && kv.head_dim > 128u)) return Kernel::kFew;
    if (rows <= kFewMax) return Kernel::kFew16;
    return kv.head_dim <= 128u ? Kernel::kTc : Kernel::kMany;
}
Kernel low_or_not(Kernel k, bool low) { return k == Kernel::kMany && low ? Kernel::kMany64 : k; }
Kernel prefix_kernel(const PagedAttention& a) {
    return low_or_not(kernel_for(a.kv, static_cast<uint64_t>(a.b.tokens) * (a.heads / a.kv.kv_heads)), a.prefix_low);
}
Kernel own_kernel(const PagedAttention& a) {
    const uint32_t group = a.heads / a.kv.kv_heads;
    return low_or_not(kernel_for(a.kv, a.picks ? std::min(group, kFewMax) : static_cast<uint64_t>(a.b.max_q_len) * group), a.own_low);
}
// The kernel of the sequences with few rows among others with many: mostly single tokens.
Kernel few_kernel(const PagedAttention& a) { return kernel_for(a.kv, std::min(a.heads / a.kv.kv_heads, kFewMax)); }
bool takes_few4(Kernel k) { return k == Kernel::kFew4 || k == Kernel::kFew4x8 || k == Kernel::kFew4x16; }
bool takes_few(Kernel k) { return k == Kernel::kFew || k == Kernel::kFew16 || k == Kernel::kFew32 || takes_few4(k); }

// A part on its kernel: `tiles` row tiles of up to max_rows rows, times KV heads and chunks.
cudaError_t launch_part(Kernel k, const AttnArgs& a, uint64_t tiles, uint64_t max_rows, cudaStream_t stream) {
    const uint64_t items = tiles * a.kv.kv_heads * a.chunks;
    switch (k) {
        case Kernel::kFew: return launch_attention_few(a, kFewRows, items, stream);
        case Kernel::kFew16: return launch_attention_few(a, 2u * kFewRows, items, stream);
        case Kernel::kFew32: return launch_attention_few32(a, static_cast<uint32_t>(std::min<uint64_t>(max_rows, kFewRows)), items, stream);
        case Kernel::kFew4: return launch_attention_few4(a, 4u, items, stream);
        case Kernel::kFew4x8: return launch_attention_few4(a, 8u, items, stream);
        case Kernel::kFew4x16: return launch_attention_few4(a, 16u, items, stream);
        case Kernel::kMany: return launch_attention_many(a, 128u, tiles, stream);
        case Kernel::kMany64: return launch_attention_many(a, 64u, tiles, stream);
        case Kernel::kTc: return launch_attention_tc(a, tiles, stream);
        default: return launch_attention_many32(a, tiles, stream);
    }
}

}  // namespace

bool plan_paged_attention(PagedAttention* a) {
    // a part's plan with tiles of 64 rows or not, whichever should take less time
    const bool choice = a->kv.type != kF32 && a->kv.head_dim > 128u;
    auto faster = [choice](bool* low, auto plan) {
        Chunks best = plan();
        if (!choice) return best;
        *low = true;
        const Chunks at64 = plan();
        if (at64.ns < best.ns) return at64;
        *low = false;
        return plan();
    };
    const uint64_t rows = static_cast<uint64_t>(a->b.tokens) * a->heads;
    const uint64_t group = a->heads / a->kv.kv_heads, all = a->b.tokens * group;
    const uint64_t sums = rows * (a->kv.head_dim * sizeof(float) + sizeof(float2));  // bytes of one chunk of every row
    const uint64_t shared = a->picks ? 0u : static_cast<uint64_t>(a->shared_pages) << a->kv.page_shift;
    uint64_t units = 0, prefix_units = 0;
    if (shared != 0u) {
        const Chunks best = faster(&a->prefix_low, [&] {
            const Cost c = cost_of(prefix_kernel(*a), a->kv);
            prefix_units = ceil_div(all, c.rows) * a->kv.kv_heads;
            return chunk_keys(shared, prefix_units, sums, a->kv, c, false);
        });
        a->prefix_chunk = best.keys;
        a->prefix_chunks = static_cast<uint32_t>(ceil_div(shared, a->prefix_chunk));
    }
    const uint64_t most = a->picks ? static_cast<uint64_t>(a->picks) << a->kv.page_shift
                                   : (a->b.max_kv_len > shared ? a->b.max_kv_len - shared : 0u);
    uint64_t keys = most;
    // with a window the chunks begin up to 63 keys in front of it
    if (!a->picks && a->window != 0u)
        keys = std::min<uint64_t>(keys, static_cast<uint64_t>(a->window) + a->b.max_q_len - 1u + 63u);
    auto chunks = [&](uint64_t chunk) { return static_cast<uint32_t>(std::max<uint64_t>(ceil_div(keys, chunk), 1u)); };
    const bool alone = shared == 0u;
    const double causal = a->picks || a->window != 0u ? 0.0 : std::min(1.0, static_cast<double>(a->b.max_q_len) / std::max<uint64_t>(keys, 1u));
    const Chunks best = faster(&a->own_low, [&] {
        const Kernel k = own_kernel(*a);
        const Cost c = cost_of(k, a->kv);
        units = (a->picks        ? a->b.tokens * ceil_div(group, c.rows)
                 : takes_few(k) ? a->b.seqs * ceil_div(a->b.max_q_len * group, c.rows)
                                : own_tiles(*a, c.rows)) *
                a->kv.kv_heads;
        return chunk_keys(keys, units, sums, a->kv, c, alone && takes_few(k), choice && !takes_few(k) ? causal : 0.0,
                          !alone && takes_few4(k));
    });
    const Kernel own = own_kernel(*a);
    a->own_chunk = best.keys;
    a->own_chunks = chunks(a->own_chunk);
    a->own_cluster = alone && takes_few(own) && a->own_chunks > 1u && a->own_chunks <= kMaxCluster;
    uint64_t grid = units * a->own_chunks, slots = a->own_cluster ? 1u : a->own_chunks;
    // several chunks of few rows of several sequences: as long as their lengths make them, where that can save
    // a round (16 sequences of 2005 to 16001 keys, 15 rows: 71 us, 85 with chunks for 16001 keys), not where
    // chunks are short (7 of 421 keys behind a prefix: 33 us, 28), there are many rounds (32 of up to
    // 32768 keys: 121 us, 119) or more sequences than a warp holds (700 of up to 3000 keys, looked through
    // again for every length tried: 185 us, 104).  What the host cannot see is whether the lengths differ:
    // 40 sequences of 2000 to 16000 keys take 52 us (71 otherwise), 12 of 3750 to 30000 33 (46), but 3
    // that all have 30000 behind a prefix 49 (41), 32 of 8 KV heads and 375 to 3000 93 (79)
    a->balance = 0;
    const uint64_t least = std::min<uint64_t>(std::max<uint64_t>((keys / 32u + 63u) / 64u * 64u, 256u), kBalanceMost);
    const uint64_t each = units * keys / cost_of(own, a->kv).slots;  // keys for each of the items that run at once
    if (takes_few4(own) && !a->picks && a->b.seqs > 1u && a->b.seqs <= kBalanceSeqs && a->own_chunks > 1u && !a->own_cluster &&
        keys > least && each >= 512u && each < 2u * kBalanceMost) {
        a->balance = cost_of(own, a->kv).slots;
        a->own_chunk = static_cast<uint32_t>(least);
        a->own_chunks = chunks(a->own_chunk);
        slots = a->own_chunks;
        // (no more items than in whole rounds of the longest chunks, but for the last of every tile)
        grid = (units * keys / kBalanceMost / a->balance + 1u) * a->balance + units;
        a->balance_grid = grid;
    }
    if (!takes_few(own) && a->b.seqs > 1u && group <= kFewMax) {  // (a larger group has more rows with every token)
        const Cost few = cost_of(few_kernel(*a), a->kv);
        const uint64_t u = static_cast<uint64_t>(a->b.seqs) * a->kv.kv_heads * (kFewMax / few.rows);
        a->few_chunk = chunk_keys(keys, u, sums, a->kv, few, alone).keys;
        a->few_chunks = chunks(a->few_chunk);
        a->few_cluster = alone && a->few_chunks > 1u && a->few_chunks <= kMaxCluster;
        grid = std::max(grid, u * a->few_chunks);
        if (!a->few_cluster) slots = std::max<uint64_t>(slots, a->few_chunks);
    }
    slots += a->prefix_chunks;
    a->workspace = slots == 1u ? 0u : slots * sums + (a->balance ? 16u : 0u);
    // the launches' grids
    return grid <= 0x7FFFFFFFull && prefix_units * a->prefix_chunks <= 0x7FFFFFFFull && rows <= 0x7FFFFFFFull;
}

cudaError_t launch_paged_attention(const PagedAttention& p, const float* q, float* out, float scale, void* workspace,
                                   DeviceStatus* st, cudaStream_t stream) {
    AttnArgs a = {};
    a.kv = p.kv;
    a.b = p.b;
    a.q = q;
    a.out = out;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.heads = p.heads;
    a.group = p.heads / p.kv.kv_heads;
    a.window = p.window;
    a.shared_len = p.picks ? 0u : p.shared_pages << p.kv.page_shift;
    a.blocks = p.blocks;
    a.picks = p.picks;
    a.st = st;
    a.rows_to = kNone;
    const uint64_t slots = std::max(p.own_cluster ? 1u : p.own_chunks, p.few_cluster ? 1u : p.few_chunks) +
                           static_cast<uint64_t>(p.prefix_chunks);
    const uint64_t rows = static_cast<uint64_t>(p.b.tokens) * p.heads;
    const bool own_direct = p.prefix_chunks == 0u && (p.own_chunks == 1u || p.own_cluster);
    const bool few_direct = p.prefix_chunks == 0u && (p.few_chunks <= 1u || p.few_cluster);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * rows * p.kv.head_dim);
    cudaError_t e = cudaSuccess;
    if (p.prefix_chunks != 0u) {
        a.part = kPartPrefix;
        a.chunk = p.prefix_chunk;
        a.chunks = p.prefix_chunks;
        a.slot0 = 0;
        const Kernel k = prefix_kernel(p);
        const uint64_t all = static_cast<uint64_t>(p.b.tokens) * a.group;
        a.row_blocks = static_cast<uint32_t>(ceil_div(all, cost_of(k, p.kv).rows));
        e = launch_part(k, a, a.row_blocks, all, stream);
        if (e != cudaSuccess) return e;
        a.late = 1u;
    }
    a.chunk = p.own_chunk;
    a.chunks = p.own_chunks;
    a.slot0 = p.prefix_chunks;
    a.direct = own_direct;
    a.cluster = p.own_cluster;
    a.balance = p.balance;
    a.chunk_at = reinterpret_cast<uint32_t*>(a.part_ml + slots * rows);
    const Kernel k = own_kernel(p);
    const uint32_t tile = cost_of(k, p.kv).rows;
    if (p.picks) {
        a.part = kPartBlocks;
        a.row_blocks = static_cast<uint32_t>(ceil_div(a.group, tile));
        e = launch_part(k, a, static_cast<uint64_t>(p.b.tokens) * a.row_blocks, a.group, stream);
    } else {
        // sequences with few rows among others go to the few-rows kernel: a tile of many rows
        // would do eight times their work
        const bool mixed = p.few_chunks != 0u;
        const uint64_t max_rows = static_cast<uint64_t>(p.b.max_q_len) * a.group;
        a.part = kPartOwn;
        // (one sequence is in order, many end with small tiles anyway and take longer to look through)
        const uint64_t most = p.window ? std::min<uint64_t>(p.window, p.b.max_kv_len) : p.b.max_kv_len;
        a.depth = p.b.seqs > 1u && p.b.seqs <= 64u ? static_cast<uint32_t>(ceil_div(most, 8u)) : 0u;
        a.rows_from = mixed ? kFewMax + 1u : 0u;
        a.row_blocks = takes_few(k) ? static_cast<uint32_t>(ceil_div(max_rows, tile)) : 1u;
        if (p.balance) e = launch_attention_few4(a, tile, p.balance_grid, stream);
        else e = launch_part(k, a, takes_few(k) ? static_cast<uint64_t>(p.b.seqs) * a.row_blocks : own_tiles(p, tile), max_rows, stream);
        if (e == cudaSuccess && mixed) {
            a.rows_from = 0u;
            a.rows_to = kFewMax;
            const Kernel few = few_kernel(p);
            a.row_blocks = kFewMax / cost_of(few, p.kv).rows;
            a.chunk = p.few_chunk;
            a.chunks = p.few_chunks;
            a.direct = few_direct;
            a.cluster = p.few_cluster;
            a.late = 1u;
            e = launch_part(few, a, static_cast<uint64_t>(p.b.seqs) * a.row_blocks, kFewRows, stream);
        }
    }
    if (e != cudaSuccess || (own_direct && few_direct)) return e;
    CombineArgs c = {};
    c.kv = p.kv;
    c.b = p.b;
    c.out = out;
    c.part_o = a.part_o;
    c.part_ml = a.part_ml;
    c.heads = p.heads;
    c.window = p.window;
    c.shared_len = a.shared_len;
    c.own_chunk = p.own_chunk;
    c.own_chunks = p.own_chunks;
    c.prefix_chunk = p.prefix_chunk;
    c.prefix_chunks = p.prefix_chunks;
    c.few_rows = p.few_chunks != 0u ? kFewMax : 0u;
    c.few_chunk = p.few_chunk;
    c.own_direct = own_direct;
    c.few_direct = few_direct;
    c.group = a.group;
    c.heads_per_cta = own_direct ? p.heads : 1u;
    c.blocks = p.picks != 0u;
    c.chunk_at = p.balance ? a.chunk_at : nullptr;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<uint32_t>(rows / c.heads_per_cta));
    cfg.blockDim = dim3(kCombineThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attention_combine_kernel, c);
}

}  // namespace nedo_gpu

// paged_attention.cu -- softmax attention of a ragged batch of query rows over a
// paged KV cache (the attention step of src/model.cpp:226-247 for many
// sequences), dense (causal, optional sliding window, optional prefix of pages
// that all sequences share) or over a list of pages per query token and KV head.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale * log2(e) * q.k_j
//
// in one pass over the keys with a running maximum m, in 32 bits throughout.  A
// work item is a tile of query rows of one KV head (the heads of its group next
// to each other, so a key is read once for all of them) times a chunk of keys.
// With one chunk per row the item writes the output; otherwise it writes
// (sum_j p_j v_j, m, sum_j p_j) of its chunk, and attention_combine_kernel adds a
// row's chunks in order, so results repeat bit for bit.  The shared prefix is a
// part of its own, whose row tiles run across all sequences: its keys are read
// once for the whole batch.
#include <algorithm>

#include "paged.cuh"

namespace nedo_gpu {
namespace {

enum : uint32_t { kPartOwn = 0, kPartPrefix = 1, kPartBlocks = 2 };

struct AttnArgs {
    PagedKv kv;
    PagedBatch b;
    const float* q;
    float* out;
    float scale_log2;
    uint32_t heads, group, window;
    uint32_t part;
    uint32_t shared_len;     // keys of the shared prefix
    uint32_t chunk, chunks;  // keys per item, items per row tile
    uint32_t slot0;          // first partial slot of this part
    uint32_t direct;         // one item per row: write out
    float* part_o;           // [slots][tokens * heads][head_dim]
    float2* part_ml;         // [slots][tokens * heads]
    const uint32_t* blocks;
    uint32_t picks, row_blocks;
    DeviceStatus* st;
};

// First chunk of sequence `sq` that any of its rows sees (own part).
__device__ __forceinline__ uint32_t own_first_chunk(const PagedSeq& sq, uint32_t window, uint32_t base, uint32_t chunk) {
    const int p0 = sq.pos(0) > 0 ? sq.pos(0) : 0;
    const uint32_t lo = first_key(p0, window);
    return lo > base ? (lo - base) / chunk : 0u;
}

// ---- the general kernel: any type, any head size, CUDA cores ----------------
constexpr uint32_t kRows = 8;   // query rows per tile
constexpr uint32_t kTile = 32;  // keys per step: one per lane
constexpr uint32_t kThreads = 128;

size_t simt_smem(uint32_t hd) { return (kRows + 2u * kTile) * static_cast<size_t>(hd + 4u) * sizeof(float); }

template <typename T>
__global__ void __launch_bounds__(kThreads) attention_simt_kernel(AttnArgs a) {
    extern __shared__ __align__(16) float sm[];
    __shared__ uint32_t row_tok[kRows], row_head[kRows];
    __shared__ int row_pos[kRows];
    __shared__ float pw[kRows][kTile], alpha[kRows], lsum[kRows];
    __shared__ float mrow[kRows];
    __shared__ uint64_t koff[kTile];
    __shared__ uint32_t kpos[kTile];
    __shared__ uint32_t found[2];
    __shared__ uint32_t list[kMaxPicks];
    const uint32_t hd = a.kv.head_dim, pitch = hd + 4u, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    float* qs = sm;
    float* ks = qs + kRows * pitch;
    float* vs = ks + kTile * pitch;
    const uint32_t c = blockIdx.x % a.chunks;
    uint32_t rest = blockIdx.x / a.chunks;
    const uint32_t kh = rest % a.kv.kv_heads;
    rest /= a.kv.kv_heads;

    // the tile's rows
    uint32_t s = kNone, r0 = 0, nrows = 0, t0 = 0;
    PagedSeq sq{0u, 0u, 0u};
    if (a.part == kPartOwn) {
        if (warp == 0) {
            uint32_t seq = kNone, tile = 0, before = 0;
            for (uint32_t s0 = 0; s0 < a.b.seqs; s0 += 32u) {
                uint32_t cnt = 0;
                if (s0 + lane < a.b.seqs) cnt = (load_seq(a.b, s0 + lane, a.st).n * a.group + kRows - 1u) / kRows;
                uint32_t inc = cnt;
                for (uint32_t o = 1; o < 32u; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                    if (lane >= o) inc += v;
                }
                const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + inc > rest);
                if (hit != 0u) {
                    const uint32_t w = __ffs(hit) - 1u;
                    seq = s0 + w;
                    tile = rest - before - __shfl_sync(0xFFFFFFFFu, inc - cnt, w);
                    break;
                }
                before += __shfl_sync(0xFFFFFFFFu, inc, 31);
            }
            if (lane == 0) {
                found[0] = seq;
                found[1] = tile;
            }
        }
        __syncthreads();
        s = found[0];
        if (s == kNone) return;
        sq = load_seq(a.b, s, a.st);
        t0 = sq.t0;
        r0 = found[1] * kRows;
        nrows = min(kRows, sq.n * a.group - r0);
    } else if (a.part == kPartPrefix) {
        r0 = rest * kRows;
        nrows = min(kRows, a.b.tokens * a.group - r0);
    } else {
        t0 = rest / a.row_blocks;
        r0 = (rest % a.row_blocks) * kRows;
        nrows = min(kRows, a.group - r0);
        s = seq_of_token(a.b, t0);
        if (s == kNone) return;
        sq = load_seq(a.b, s, a.st);
        if (sq.n == 0u) return;
    }
    if (tid < kRows) {
        int p = -2;  // no row here
        uint32_t tok = 0, head = 0;
        if (tid < nrows) {
            tok = t0 + (r0 + tid) / a.group;
            head = kh * a.group + (r0 + tid) % a.group;
            if (a.part == kPartPrefix) {
                const uint32_t ss = seq_of_token(a.b, tok);
                if (ss != kNone) {
                    const PagedSeq q2 = load_seq(a.b, ss, a.st);
                    if (q2.n != 0u) p = max(-1, q2.pos(tok - q2.t0));
                }
            } else {
                p = max(-1, sq.pos(tok - sq.t0));
            }
        }
        row_tok[tid] = tok;
        row_head[tid] = head;
        row_pos[tid] = p;
        mrow[tid] = -INFINITY;
        lsum[tid] = 0.f;
    }
    __syncthreads();
    // the tile's keys in this chunk: [kb, ke) positions, or list entries
    uint32_t kb = kNone, ke = 0;
    if (a.part == kPartBlocks) {
        const uint32_t* l = a.blocks + (static_cast<size_t>(t0) * a.kv.kv_heads + kh) * a.picks;
        const int p = row_pos[0];
        // an entry counts when it is above all entries before it and at or below the query's page
        if (warp == 0) {
            int best = -1;
            for (uint32_t i0 = 0; i0 < a.picks; i0 += 32u) {
                const uint32_t v = i0 + lane < a.picks ? l[i0 + lane] : kNone;
                const bool in = p >= 0 && v <= (static_cast<uint32_t>(max(p, 0)) >> a.kv.page_shift);
                int run = in ? static_cast<int>(v) : -1;
                for (uint32_t o = 1; o < 32u; o <<= 1) {
                    const int u = __shfl_up_sync(0xFFFFFFFFu, run, o);
                    if (lane >= o) run = max(run, u);
                }
                int prev = __shfl_up_sync(0xFFFFFFFFu, run, 1);
                if (lane == 0) prev = -1;
                prev = max(prev, best);
                if (i0 + lane < a.picks) list[i0 + lane] = in && static_cast<int>(v) > prev ? v : kNone;
                best = max(best, __shfl_sync(0xFFFFFFFFu, run, 31));
            }
        }
        __syncthreads();
        kb = c * a.chunk;
        ke = min(kb + a.chunk, a.picks << a.kv.page_shift);
    } else {
        for (uint32_t r = 0; r < kRows; ++r) {
            if (row_pos[r] < 0) continue;
            kb = min(kb, first_key(row_pos[r], a.window));
            ke = max(ke, static_cast<uint32_t>(row_pos[r]) + 1u);
        }
        uint32_t base = 0, first = 0;
        if (a.part == kPartOwn) {
            base = a.shared_len;
            first = own_first_chunk(sq, a.window, base, a.chunk);
        } else {
            ke = min(ke, a.shared_len);
        }
        const uint64_t cb = static_cast<uint64_t>(base) + static_cast<uint64_t>(first + c) * a.chunk;
        kb = cb > kb ? static_cast<uint32_t>(cb < kNone ? cb : kNone) : max(kb, base);
        if (cb + a.chunk < ke) ke = static_cast<uint32_t>(cb + a.chunk);
        if (kb >= ke && !a.direct) return;  // no row of the tile sees a key of this chunk
        if (a.part == kPartPrefix) s = 0;
    }
    for (uint32_t i = tid; i < kRows * hd; i += kThreads) {
        const uint32_t r = i / hd, d = i - r * hd;
        qs[r * pitch + d] =
            row_pos[r] >= 0 ? a.q[(static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd + d] * a.scale_log2 : 0.f;
    }
    float acc[kRows][2];
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) acc[r][0] = acc[r][1] = 0.f;

    for (uint32_t j0 = kb; j0 < ke; j0 += kTile) {
        __syncthreads();
        if (tid < kTile) {
            const uint32_t j = j0 + tid;
            uint32_t pos = kNone;
            uint64_t off = ~0ull;
            if (j < ke) {
                const uint32_t lp = a.part == kPartBlocks ? list[j >> a.kv.page_shift] : j >> a.kv.page_shift;
                const uint32_t slot = j & (a.kv.page_size - 1u);
                if (lp != kNone) {
                    const uint32_t at = (lp << a.kv.page_shift) + slot;
                    const uint32_t page = at < sq.kv || a.part == kPartPrefix ? load_page(a.b, a.kv, s, lp, a.st) : kNone;
                    if (page != kNone) {
                        pos = at;
                        off = ((static_cast<uint64_t>(page) * a.kv.kv_heads + kh) * a.kv.page_size + slot) * hd;
                    }
                }
            }
            kpos[tid] = pos;
            koff[tid] = off;
        }
        __syncthreads();
        for (uint32_t i = tid; i < kTile * hd; i += kThreads) {
            const uint32_t j = i / hd, d = i - j * hd;
            const uint64_t off = koff[j];
            // unseen keys count as zero, whatever their memory holds
            ks[j * pitch + d] = off != ~0ull ? kv_float(static_cast<const T*>(a.kv.k)[off + d]) : 0.f;
            vs[j * pitch + d] = off != ~0ull ? kv_float(static_cast<const T*>(a.kv.v)[off + d]) : 0.f;
        }
        __syncthreads();
        for (uint32_t r = warp; r < kRows; r += kThreads / 32u) {
            float sc = 0.f;
            for (uint32_t d = 0; d < hd; d += 4u) {
                const float4 kk = *reinterpret_cast<const float4*>(ks + lane * pitch + d);
                const float4 qq = *reinterpret_cast<const float4*>(qs + r * pitch + d);
                sc = fmaf(kk.x, qq.x, sc);
                sc = fmaf(kk.y, qq.y, sc);
                sc = fmaf(kk.z, qq.z, sc);
                sc = fmaf(kk.w, qq.w, sc);
            }
            const uint32_t at = kpos[lane];
            const int p = row_pos[r];
            const bool see = p >= 0 && at <= static_cast<uint32_t>(p) && at >= first_key(p, a.window);
            if (!see) sc = -INFINITY;
            float m = sc;
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            const float m0 = mrow[r];
            m = fmaxf(m, m0);
            // rows that have seen nothing yet keep m = -inf, factor 1 and weights 0
            const float al = m == -INFINITY ? 1.f : exp2f(m0 - m);
            const float e = see ? exp2f(sc - m) : 0.f;
            const float l = warp_sum(e);
            pw[r][lane] = e;
            __syncwarp();
            if (lane == 0) {
                alpha[r] = al;
                mrow[r] = m;
                lsum[r] = lsum[r] * al + l;
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < 2u; ++u) {
            const uint32_t d = tid + u * kThreads;
            if (d >= hd) continue;
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                float o = acc[r][u] * alpha[r];
                for (uint32_t j = 0; j < kTile; ++j) {
                    const float w = pw[r][j];
                    if (w != 0.f) o = fmaf(w, vs[j * pitch + d], o);  // an unseen value never enters
                }
                acc[r][u] = o;
            }
        }
    }
    __syncthreads();
    const size_t rows_all = static_cast<size_t>(a.b.tokens) * a.heads;
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
        if (row_pos[r] == -2) continue;
        const size_t row = static_cast<size_t>(row_tok[r]) * a.heads + row_head[r];
        const float l = lsum[r];
#pragma unroll
        for (uint32_t u = 0; u < 2u; ++u) {
            const uint32_t d = tid + u * kThreads;
            if (d >= hd) continue;
            if (a.direct) {
                a.out[row * hd + d] = l == 0.f ? 0.f : acc[r][u] / l;  // l = 0: no key seen
            } else {
                a.part_o[((a.slot0 + c) * rows_all + row) * hd + d] = acc[r][u];
            }
        }
        if (!a.direct && tid == 0) a.part_ml[(a.slot0 + c) * rows_all + row] = make_float2(mrow[r], l);
    }
}

// ---- adding a row's chunks ---------------------------------------------------
struct CombineArgs {
    PagedKv kv;
    PagedBatch b;
    float* out;
    const float* part_o;
    const float2* part_ml;
    uint32_t heads, window, shared_len;
    uint32_t own_chunk, own_chunks, prefix_chunk, prefix_chunks;
    uint32_t blocks;  // the sparse call: every slot is written
};

// One warp per (token, head): first the maximum over the row's chunks, then their
// sum in chunk order.  A chunk in which the row sees nothing has weight sum 0.
constexpr uint32_t kCombineWarps = 4;
__global__ void __launch_bounds__(32 * kCombineWarps) attention_combine_kernel(CombineArgs a) {
    const size_t rows_all = static_cast<size_t>(a.b.tokens) * a.heads;
    const size_t row = static_cast<size_t>(blockIdx.x) * kCombineWarps + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31u;
    if (row >= rows_all) return;
    const uint32_t t = static_cast<uint32_t>(row / a.heads);
    const uint32_t s = seq_of_token(a.b, t);
    if (s == kNone) return;
    const PagedSeq sq = load_seq(a.b, s, nullptr);
    if (sq.n == 0u) return;
    const int p = sq.pos(t - sq.t0);
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
            const uint32_t first = own_first_chunk(sq, a.window, a.shared_len, a.own_chunk);
            b1 = a.prefix_chunks + (max(lo, a.shared_len) - a.shared_len) / a.own_chunk - first;
            e1 = a.prefix_chunks + (hi - 1u - a.shared_len) / a.own_chunk + 1u - first;
        }
    }
    const uint32_t n0 = e0 - b0, n = n0 + (e1 - b1);
    float m = -INFINITY;
    for (uint32_t i = lane; i < n; i += 32u) {
        const uint32_t slot = i < n0 ? b0 + i : b1 + (i - n0);
        m = fmaxf(m, a.part_ml[slot * rows_all + row].x);
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const uint32_t hd = a.kv.head_dim;
    float l = 0.f, acc[8];
#pragma unroll
    for (uint32_t u = 0; u < 8u; ++u) acc[u] = 0.f;
    for (uint32_t i = 0; i < n; ++i) {
        const size_t slot = i < n0 ? b0 + i : b1 + (i - n0);
        const float2 ml = a.part_ml[slot * rows_all + row];
        if (ml.y == 0.f) continue;  // the row sees nothing there, or every weight underflowed
        const float w = exp2f(ml.x - m);
        l = fmaf(ml.y, w, l);
        const float* o = a.part_o + (slot * rows_all + row) * hd;
#pragma unroll
        for (uint32_t u = 0; u < 8u; ++u)
            if (lane + 32u * u < hd) acc[u] = fmaf(o[lane + 32u * u], w, acc[u]);
    }
#pragma unroll
    for (uint32_t u = 0; u < 8u; ++u)
        if (lane + 32u * u < hd) a.out[row * hd + lane + 32u * u] = l == 0.f ? 0.f : acc[u] / l;
}

}  // namespace

bool plan_paged_attention(PagedAttention* a) {
    const uint64_t hd = a->kv.head_dim, rows = static_cast<uint64_t>(a->b.tokens) * a->heads;
    const uint32_t shared = a->picks ? 0u : a->shared_pages << a->kv.page_shift;
    a->prefix_chunk = 1024;
    a->own_chunk = 1024;
    a->prefix_chunks = (shared + a->prefix_chunk - 1u) / a->prefix_chunk;
    uint64_t keys = a->picks ? static_cast<uint64_t>(a->picks) << a->kv.page_shift
                             : (a->b.max_kv_len > shared ? a->b.max_kv_len - shared : 0u);
    uint64_t n = (keys + a->own_chunk - 1u) / a->own_chunk;
    if (!a->picks && a->window != 0u)
        n = std::min<uint64_t>(n, (static_cast<uint64_t>(a->window) + a->b.max_q_len + a->own_chunk - 2u) / a->own_chunk + 1u);
    a->own_chunks = static_cast<uint32_t>(std::max<uint64_t>(n, 1u));
    const uint64_t slots = static_cast<uint64_t>(a->own_chunks) + a->prefix_chunks;
    a->workspace = slots == 1u ? 0u : slots * rows * (hd * sizeof(float) + sizeof(float2));
    return true;
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
    const uint64_t slots = static_cast<uint64_t>(p.own_chunks) + p.prefix_chunks;
    const uint64_t rows = static_cast<uint64_t>(p.b.tokens) * p.heads;
    a.direct = slots == 1u;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * rows * p.kv.head_dim);
    const size_t smem = simt_smem(p.kv.head_dim);
    auto* kernel = p.kv.type == kF16 ? attention_simt_kernel<__half> : attention_simt_kernel<float>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (p.prefix_chunks != 0u) {
        a.part = kPartPrefix;
        a.chunk = p.prefix_chunk;
        a.chunks = p.prefix_chunks;
        a.slot0 = 0;
        const uint64_t tiles = (static_cast<uint64_t>(p.b.tokens) * a.group + kRows - 1u) / kRows;
        kernel<<<static_cast<uint32_t>(tiles * p.kv.kv_heads * a.chunks), kThreads, smem, stream>>>(a);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    a.chunk = p.own_chunk;
    a.chunks = p.own_chunks;
    a.slot0 = p.prefix_chunks;
    uint64_t tiles;
    if (p.picks) {
        a.part = kPartBlocks;
        a.row_blocks = (a.group + kRows - 1u) / kRows;
        tiles = static_cast<uint64_t>(p.b.tokens) * a.row_blocks;
    } else {
        a.part = kPartOwn;
        tiles = std::min<uint64_t>(static_cast<uint64_t>(p.b.tokens) * a.group / kRows + p.b.seqs,
                                   static_cast<uint64_t>(p.b.seqs) * ((static_cast<uint64_t>(p.b.max_q_len) * a.group + kRows - 1u) / kRows));
    }
    kernel<<<static_cast<uint32_t>(tiles * p.kv.kv_heads * a.chunks), kThreads, smem, stream>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    if (a.direct) return cudaSuccess;
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
    c.blocks = p.picks != 0u;
    attention_combine_kernel<<<static_cast<uint32_t>((rows + kCombineWarps - 1u) / kCombineWarps), 32 * kCombineWarps, 0,
                               stream>>>(c);
    return cudaGetLastError();
}

}  // namespace nedo_gpu

// paged_attention.cuh -- what the attention kernels over a paged cache share: the
// arguments of a launch, the tile search and the pieces of a work item's set-up.
#pragma once

#include "paged.cuh"

namespace nedo_gpu {

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
    uint32_t direct;         // one item, or one cluster of items, per row: write out
    uint32_t cluster;        // few-rows kernels: a row tile's chunks are the CTAs of a cluster
    uint32_t late;           // launched while another part's kernel may still run
    float* part_o;           // [slots][tokens * heads][head_dim]
    float2* part_ml;         // [slots][tokens * heads]
    uint32_t depth;          // many-rows kernels: keys by which a launch's tiles are put in order
    // own part: rows per sequence that this launch takes, from .. to (the others are another's)
    uint32_t rows_from, rows_to;
    const uint32_t* blocks;
    uint32_t picks, row_blocks;
    DeviceStatus* st;
};

// Where the chunks of sequence `sq`'s own part begin: at the first key that any of its rows
// sees, rounded down to 64 keys from `base`.
__device__ __forceinline__ uint32_t own_begin(const PagedSeq& sq, uint32_t window, uint32_t base) {
    const int p0 = sq.pos(0) > 0 ? sq.pos(0) : 0;
    const uint32_t lo = first_key(p0, window);
    return lo > base ? base + ((lo - base) & ~63u) : base;
}

// First of a sequence's row tiles with rows that see more than `keys` keys (or as many tiles
// as it has): with causal rows the later tiles have the most keys, up to the window.
__device__ __forceinline__ uint32_t first_tile_above(const AttnArgs& a, const PagedSeq& sq, uint32_t tiles, uint32_t tile_rows,
                                                     uint32_t keys) {
    if (a.window != 0u && keys >= a.window) return tiles;
    const int token = static_cast<int>(keys) - static_cast<int>(sq.kv - min(sq.kv, sq.n));  // the first token that does
    if (token <= 0) return 0u;
    if (token >= static_cast<int>(sq.n)) return tiles;
    const uint32_t t = (static_cast<uint32_t>(token) * a.group + tile_rows) / tile_rows;  // tiles up to the one with its first row
    return min(tiles, t - 1u);
}

// One warp: the sequence, and the tile within it, that work item `want` is (kNone: there is no
// such item).  Every sequence that this launch takes has ceil(rows / tile_rows) tiles.  Those with
// many keys come first, in steps of an eighth of the most keys that a row can see (a.depth; 0:
// not in steps), so that the launch does not end with one of them.
__device__ __forceinline__ uint32_t find_tile(const AttnArgs& a, uint32_t want, uint32_t tile_rows, uint32_t* tile) {
    const uint32_t lane = threadIdx.x & 31u;
    // a lane per sequence and step
    const uint32_t steps = a.depth != 0u ? 8u : 1u, all = steps * a.b.seqs;
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < all; e0 += 32u) {
        const uint32_t turn = (e0 + lane) / a.b.seqs, s = e0 + lane - turn * a.b.seqs, step = steps - 1u - turn;
        uint32_t cnt = 0, first = 0;
        if (e0 + lane < all) {
            const PagedSeq sq = load_seq(a.b, s, a.st);
            const uint32_t rows = sq.n * a.group;
            if (rows >= a.rows_from && rows <= a.rows_to) {
                cnt = (rows + tile_rows - 1u) / tile_rows;
                if (a.depth != 0u) {
                    if (step != 0u) first = first_tile_above(a, sq, cnt, tile_rows, step * a.depth);
                    const uint32_t end = step != 7u ? first_tile_above(a, sq, cnt, tile_rows, (step + 1u) * a.depth) : cnt;
                    cnt = end - first;
                }
            }
        }
        uint32_t inc = cnt;
        for (uint32_t o = 1; o < 32u; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
            if (lane >= o) inc += v;
        }
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + inc > want);
        if (hit != 0u) {
            const uint32_t w = __ffs(hit) - 1u;
            // within a sequence the last tile first
            const uint32_t at = want - before - __shfl_sync(0xFFFFFFFFu, inc - cnt, w);
            *tile = __shfl_sync(0xFFFFFFFFu, first + cnt, w) - 1u - at;
            return __shfl_sync(0xFFFFFFFFu, s, w);
        }
        before += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
    *tile = 0;
    return kNone;
}

// Position of the query row of token `tok`: -1 for padding, -2 when it is no row of
// any sequence (whose output is left alone).
__device__ __forceinline__ int row_position(const AttnArgs& a, uint32_t tok) {
    const uint32_t s = seq_of_token(a.b, tok);
    if (s == kNone) return -2;
    const PagedSeq sq = load_seq(a.b, s, a.st);
    return sq.n == 0u ? -2 : max(-1, sq.pos(tok - sq.t0));
}

// One warp: the entries of a page list that count for a query at position p, into
// out[0..n) in place of the others kNone: above every entry before it (`n` of the
// list's entries are looked at) and not beyond the row's own page.
__device__ __forceinline__ void checked_list(const uint32_t* __restrict__ l, uint32_t n, int p, uint32_t page_shift,
                                             uint32_t* out) {
    const uint32_t lane = threadIdx.x & 31u;
    int best = -1;
    for (uint32_t i0 = 0; i0 < n; i0 += 32u) {
        const uint32_t v = i0 + lane < n ? l[i0 + lane] : kNone;
        const bool in = p >= 0 && v <= (static_cast<uint32_t>(max(p, 0)) >> page_shift);
        int run = in ? static_cast<int>(v) : -1;
        for (uint32_t o = 1; o < 32u; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, run, o);
            if (lane >= o) run = max(run, u);
        }
        int prev = __shfl_up_sync(0xFFFFFFFFu, run, 1);
        prev = max(lane == 0u ? -1 : prev, best);
        if (i0 + lane < n) out[i0 + lane] = in && static_cast<int>(v) > prev ? v : kNone;
        best = max(best, __shfl_sync(0xFFFFFFFFu, run, 31));
    }
}

// The sums of up to kAgain query rows over F16 keys, formed by one warp key by key in fp32.  The
// tensor-core kernels multiply with factors split in two halves, and an infinite key or value times
// halves of different sign, or one that is zero, is NaN where the whole factor gives infinity (or,
// for a score of -infinity, no weight at all).  A value that is not finite also reaches the rows of
// its tile that do not see it, as 0 * inf.  Either stays in the running sums, so the kernels look
// at a row's sums once, when they are complete, and take those that are not finite from here.
// A lane takes a key's scores, for all rows, and then channels lane, lane + 32, ... of the values.
// A prompt of 3888 tokens with an infinite value that all rows see: 6 ms (21 a row at a time,
// which reads the cache once for each).
constexpr uint32_t kAgain = 4;
struct RowSums {
    float m[kAgain], l[kAgain], o[kAgain][8];  // sums go by 2^(s - m)
};
struct TileRows {
    const uint32_t *tok, *head;
    const int* pos;
};
// The lowest kAgain rows of a set as bytes, the last one repeated, and taken out of it.
__device__ __forceinline__ uint32_t take_rows(uint32_t* set, uint32_t* n) {
    uint32_t rows = 0, r = 0;
    *n = 0;
#pragma unroll
    for (uint32_t u = 0; u < kAgain; ++u) {
        if (*set != 0u) {
            r = __ffs(*set) - 1u;
            *set &= *set - 1u;
            ++*n;
        }
        rows |= r << (8u * u);
    }
    return rows;
}
// Rows rows & 255, ... (+ `first`); keys `from`, from + 1, ... below `to` in steps of 16 that are
// `stride` apart (from a multiple of 16 where stride is not 16): positions, or places in the page
// list (`list`).
static __device__ __noinline__ void rows_key_by_key(const AttnArgs& a, uint32_t s, uint32_t kh, const uint32_t* list,
                                                    const TileRows& tile, uint32_t first, uint32_t rows, uint32_t from,
                                                    uint32_t to, uint32_t stride, RowSums* sums) {
    const uint32_t lane = threadIdx.x & 31u, hd = a.kv.head_dim, in_page = a.kv.page_size - 1u;
    const __half *k = static_cast<const __half*>(a.kv.k), *v = static_cast<const __half*>(a.kv.v);
    const float* q[kAgain];
    uint32_t lo[kAgain], hi[kAgain], least = kNone, most = 0u;
    RowSums r;
#pragma unroll
    for (uint32_t u = 0; u < kAgain; ++u) {
        const uint32_t i = first + (rows >> (8u * u) & 255u), p = static_cast<uint32_t>(tile.pos[i]);
        q[u] = a.q + (static_cast<size_t>(tile.tok[i]) * a.heads + tile.head[i]) * hd;
        lo[u] = first_key(static_cast<int>(p), a.window);
        hi[u] = p + 1u;
        least = min(least, lo[u]);
        most = max(most, hi[u]);
        r.m[u] = -INFINITY;
        r.l[u] = 0.f;
#pragma unroll
        for (uint32_t d = 0; d < 8u; ++d) r.o[u][d] = 0.f;
    }
    for (uint32_t j0 = from & ~15u; j0 < to; j0 += 2u * stride) {
        const uint32_t j = j0 + (lane >> 4) * stride + (lane & 15u);
        size_t at = 0;
        uint32_t pos = kNone;  // a key that no row sees
        if (j >= from && j < to) {
            const uint32_t lp = list != nullptr ? list[j >> a.kv.page_shift] : j >> a.kv.page_shift;
            const uint32_t x = (lp << a.kv.page_shift) + (j & in_page);
            if (lp != kNone && x >= least && x < most) {
                const uint32_t page = load_page(a.b, a.kv, s, lp, a.st);
                if (page != kNone) {
                    pos = x;
                    at = ((static_cast<size_t>(page) * a.kv.kv_heads + kh) * a.kv.page_size + (j & in_page)) * hd;
                }
            }
        }
        if (!__any_sync(0xFFFFFFFFu, pos != kNone)) continue;
        float sum[kAgain];
#pragma unroll
        for (uint32_t u = 0; u < kAgain; ++u) sum[u] = 0.f;
        if (pos != kNone)
#pragma unroll 2
            for (uint32_t d = 0; d < hd; d += 8u) {
                const uint4 x = *reinterpret_cast<const uint4*>(k + at + d);
                const __half2* h = reinterpret_cast<const __half2*>(&x);
#pragma unroll
                for (uint32_t u = 0; u < kAgain; ++u)
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e) {
                        const float2 f = __half22float2(h[e]), y = *reinterpret_cast<const float2*>(q[u] + d + 2u * e);
                        sum[u] = fmaf(y.y * a.scale_log2, f.y, fmaf(y.x * a.scale_log2, f.x, sum[u]));
                    }
            }
        uint32_t seen[kAgain], any = 0u;
#pragma unroll
        for (uint32_t u = 0; u < kAgain; ++u) {
            const bool see = pos >= lo[u] && pos < hi[u];
            seen[u] = __ballot_sync(0xFFFFFFFFu, see);
            any |= seen[u];
            float m = see ? sum[u] : -INFINITY;
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            m = fmaxf(m, r.m[u]);
            const float ref = m == -INFINITY ? 0.f : m, alpha = exp2f(r.m[u] - ref);
            sum[u] = see ? exp2f(sum[u] - ref) : 0.f;  // the weight
            r.m[u] = m;
            r.l[u] = fmaf(r.l[u], alpha, warp_sum(sum[u]));
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) r.o[u][i] *= alpha;
        }
        for (uint32_t e = 0; e < 32u; e += 2u) {
            if ((any >> e & 3u) == 0u) continue;
            float x[2][8];
#pragma unroll
            for (uint32_t z = 0; z < 2u; ++z) {
                const __half* row = v + __shfl_sync(0xFFFFFFFFu, static_cast<unsigned long long>(at), e + z) + lane;
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i)
                    x[z][i] = lane + 32u * i < hd && (any >> (e + z) & 1u) ? __half2float(row[32u * i]) : 0.f;
            }
#pragma unroll
            for (uint32_t z = 0; z < 2u; ++z)
#pragma unroll
                for (uint32_t u = 0; u < kAgain; ++u) {
                    const float f = __shfl_sync(0xFFFFFFFFu, sum[u], e + z);
                    if (!(seen[u] >> (e + z) & 1u)) continue;
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) r.o[u][i] = fmaf(f, x[z][i], r.o[u][i]);
                }
        }
    }
#pragma unroll
    for (uint32_t u = 0; u < kAgain; ++u)
        if (r.m[u] == -INFINITY) r.m[u] = 0.f;
    *sums = r;
}

constexpr uint32_t kFewRows = 8;
constexpr uint32_t kFewMax = 16;     // rows of a sequence that still go to the few-rows kernels, in tiles of 8 or 16
constexpr uint32_t kMaxCluster = 8;  // chunks that a cluster can hold
// The work item of a few-rows CTA: its row tile (into shared memory: token, head and
// position of each row, position -2 where there is none) and its keys.
struct FewItem {
    uint32_t s, kh, c;       // sequence whose page table serves, KV head, chunk
    uint32_t kb, ke;         // keys: positions, or places in the page list (`list`)
    uint32_t all_b, all_e;   // positions seen by every row
};
// False: nothing to do.  All threads of the CTA.  ROWS: rows of a tile.
template <uint32_t ROWS>
__device__ __forceinline__ bool few_setup(const AttnArgs& a, uint32_t* row_tok, uint32_t* row_head, int* row_pos,
                                          uint32_t* list, FewItem* it) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5;
    const uint32_t c = blockIdx.x % a.chunks;
    uint32_t rest = blockIdx.x / a.chunks;
    const uint32_t kh = rest % a.kv.kv_heads;
    rest /= a.kv.kv_heads;

    // rows
    uint32_t s = 0, r0 = 0, nrows, t0 = 0;
    PagedSeq sq{0u, 0u, 0u};
    r0 = rest % a.row_blocks * ROWS;
    rest /= a.row_blocks;
    if (a.part == kPartPrefix) {
        nrows = min(ROWS, a.b.tokens * a.group - r0);
    } else {
        if (a.part == kPartOwn) {
            s = rest;
        } else {
            t0 = rest;
            s = seq_of_token(a.b, t0);
            if (s == kNone) return false;
        }
        sq = load_seq(a.b, s, a.st);
        if (sq.n == 0u) return false;
        const uint32_t rows = a.part == kPartOwn ? sq.n * a.group : a.group;
        if (a.part == kPartOwn) t0 = sq.t0;
        if (a.part == kPartOwn && rows > a.rows_to) return false;  // the many-rows kernel's
        if (r0 >= rows) return false;
        nrows = min(ROWS, rows - r0);
    }
    if (tid < ROWS) {
        int p = -2;
        uint32_t tok = 0, head = 0;
        if (tid < nrows) {
            tok = t0 + (r0 + tid) / a.group;
            head = kh * a.group + (r0 + tid) % a.group;
            p = a.part == kPartPrefix ? row_position(a, tok) : max(-1, sq.pos(tok - sq.t0));
        }
        row_tok[tid] = tok;
        row_head[tid] = head;
        row_pos[tid] = p;
    }
    __syncthreads();
    // keys [kb, ke): positions, or places in the page list; [all_b, all_e): seen by every row
    uint32_t kb = kNone, ke = 0, all_b = 0, all_e = kNone;
    for (uint32_t r = 0; r < ROWS; ++r) {
        if (row_pos[r] < 0) continue;
        const uint32_t lo = first_key(row_pos[r], a.window), hi = static_cast<uint32_t>(row_pos[r]) + 1u;
        kb = min(kb, lo);
        ke = max(ke, hi);
        all_b = max(all_b, lo);
        all_e = min(all_e, hi);
    }
    if (a.part == kPartBlocks) {
        const uint32_t e0 = (c * a.chunk) >> a.kv.page_shift;
        const uint32_t e1 = min(e0 + (a.chunk >> a.kv.page_shift), a.picks);
        if (warp == 0)
            checked_list(a.blocks + (static_cast<size_t>(t0) * a.kv.kv_heads + kh) * a.picks, e1, row_pos[0],
                         a.kv.page_shift, list);
        __syncthreads();
        kb = e0 << a.kv.page_shift;
        ke = e1 << a.kv.page_shift;
    } else {
        uint32_t base = 0;
        if (a.part == kPartOwn) base = own_begin(sq, a.window, a.shared_len);
        else ke = min(ke, a.shared_len);
        const uint64_t cb = static_cast<uint64_t>(base) + static_cast<uint64_t>(c) * a.chunk;
        kb = cb > kb ? static_cast<uint32_t>(cb < kNone ? cb : kNone) : max(kb, base);
        if (cb + a.chunk < ke) ke = static_cast<uint32_t>(cb + a.chunk);
        if (kb >= ke && !a.direct) return false;  // no row of the tile sees a key of this chunk
    }
    *it = FewItem{s, kh, c, kb, ke, all_b, all_e};
    return true;
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
// This CTA's shared address in CTA `rank` of the cluster, and loads from there.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 load2_cluster(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 load4_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// The warps' sums of a few-rows CTA (part [warp][row][pitch], maxima wm and weight sums wl
// in shared memory) added in warp order and written out, or to the chunk's place, or, where
// the row tile's chunks are a cluster, into shared memory behind `part`: there every CTA adds
// a share of the rows' channels over the chunks, in chunk order, and writes it out.
template <uint32_t WARPS, uint32_t ROWS>
__device__ __forceinline__ void few_finish(const AttnArgs& a, uint32_t c, const uint32_t* row_tok, const uint32_t* row_head,
                                           const int* row_pos, const float (*wm)[ROWS], const float (*wl)[ROWS],
                                           float* part, uint32_t pitch) {
    __shared__ float2 chunk_ml[ROWS];
    const uint32_t tid = threadIdx.x, hd = a.kv.head_dim, hd4 = hd / 4u;
    const size_t rows_all = static_cast<size_t>(a.b.tokens) * a.heads;
    float* const mine = part + WARPS * ROWS * pitch;  // cluster: [row][hd]
    for (uint32_t i = tid; i < ROWS * hd4; i += blockDim.x) {
        const uint32_t r = i / hd4, d = (i - r * hd4) * 4u;
        if (row_pos[r] == -2) continue;
        float top = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < WARPS; ++w)
            if (wl[w][r] != 0.f) top = fmaxf(top, wm[w][r]);
        float sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t w = 0; w < WARPS; ++w) {
            if (wl[w][r] == 0.f) continue;  // nothing seen there
            const float f = exp2f(wm[w][r] - top);
            const float4 x = *reinterpret_cast<const float4*>(part + (w * ROWS + r) * pitch + d);
            sum = fmaf(wl[w][r], f, sum);
            o.x = fmaf(x.x, f, o.x);
            o.y = fmaf(x.y, f, o.y);
            o.z = fmaf(x.z, f, o.z);
            o.w = fmaf(x.w, f, o.w);
        }
        const size_t row = static_cast<size_t>(row_tok[r]) * a.heads + row_head[r];
        if (a.cluster) {
            *reinterpret_cast<float4*>(mine + r * hd + d) = o;
            if (d == 0u) chunk_ml[r] = make_float2(top, sum);
        } else if (a.direct) {
            const bool none = sum == 0.f;
            *reinterpret_cast<float4*>(a.out + row * hd + d) =
                none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x / sum, o.y / sum, o.z / sum, o.w / sum);
        } else {
            *reinterpret_cast<float4*>(a.part_o + ((a.slot0 + c) * rows_all + row) * hd + d) = o;
            if (d == 0u) a.part_ml[(a.slot0 + c) * rows_all + row] = make_float2(top, sum);
        }
    }
    if (!a.cluster) return;
    cluster_sync();
    const uint32_t n = a.chunks, ml_addr = smem_addr(chunk_ml), o_addr = smem_addr(mine);
    for (uint32_t i = cluster_rank() * blockDim.x + tid; i < ROWS * hd4; i += n * blockDim.x) {
        const uint32_t r = i / hd4, d = (i - r * hd4) * 4u;
        if (row_pos[r] == -2) continue;
        float2 ml[kMaxCluster];
        float4 x[kMaxCluster];
        float top = -INFINITY;
#pragma unroll
        for (uint32_t k = 0; k < kMaxCluster; ++k) {
            ml[k] = make_float2(0.f, 0.f);
            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < n) {
                ml[k] = load2_cluster(map_rank(ml_addr + r * 8u, k));
                x[k] = load4_cluster(map_rank(o_addr + (r * hd + d) * 4u, k));
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kMaxCluster; ++k)
            if (ml[k].y != 0.f) top = fmaxf(top, ml[k].x);
        float sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t k = 0; k < kMaxCluster; ++k) {
            if (ml[k].y == 0.f) continue;
            const float f = exp2f(ml[k].x - top);
            sum = fmaf(ml[k].y, f, sum);
            o.x = fmaf(x[k].x, f, o.x);
            o.y = fmaf(x[k].y, f, o.y);
            o.z = fmaf(x[k].z, f, o.z);
            o.w = fmaf(x[k].w, f, o.w);
        }
        const bool none = sum == 0.f;
        *reinterpret_cast<float4*>(a.out + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd + d) =
            none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x / sum, o.y / sum, o.z / sum, o.w / sum);
    }
    cluster_sync();  // no CTA leaves while another still reads its sums
}

// The last step of every CTA: a launch that may overlap the part before it (a.late) ends
// after that part, whatever its CTAs found to do, because what runs next reads both.
__device__ __forceinline__ void end_after_previous(const AttnArgs& a) {
    if (a.late) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// A launch with a cluster of a.chunks CTAs where a.cluster says so, and, where a.late, while
// the kernel before it may still be running (which then ends before this one does).
template <typename... Args>
cudaError_t launch_items(const AttnArgs& a, void (*kernel)(Args...), uint64_t items, uint32_t threads, size_t smem,
                         cudaStream_t stream, Args... args) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<uint32_t>(items));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    uint32_t n = 0;
    if (a.cluster) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = a.chunks;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    if (a.late) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The few-rows kernels: F16 caches on the tensor cores, tiles of `rows` 8 or (heads of up to
// 128 channels) 16 query rows (paged_attention_few.cu), F32 caches on the CUDA cores, tiles of
// 8 (paged_attention_few32.cu).
cudaError_t launch_attention_few(const AttnArgs& a, uint32_t rows, uint64_t items, cudaStream_t stream);
cudaError_t launch_attention_few32(const AttnArgs& a, uint32_t max_rows, uint64_t items, cudaStream_t stream);
// Tiles of `rows` 64 or 128 rows on the tensor cores (paged_attention_many.cu): F16 caches, heads
// above 128.
cudaError_t launch_attention_many(const AttnArgs& a, uint32_t rows, uint64_t tiles, cudaStream_t stream);
// Tiles of many32_rows(head_dim) rows of F32 caches on the tensor cores
// (paged_attention_many32.cu).
uint32_t many32_rows(uint32_t head_dim);
cudaError_t launch_attention_many32(const AttnArgs& a, uint64_t tiles, cudaStream_t stream);
// Tiles of kTcRows rows on the 5th-generation tensor cores (paged_attention_tc.cu): F16
// caches, heads of up to 128 channels.
constexpr uint32_t kTcRows = 128;
cudaError_t launch_attention_tc(const AttnArgs& a, uint64_t tiles, cudaStream_t stream);

}  // namespace nedo_gpu

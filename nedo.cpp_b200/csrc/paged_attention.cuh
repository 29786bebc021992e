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
    uint32_t direct;         // one item per row: write out
    float* part_o;           // [slots][tokens * heads][head_dim]
    float2* part_ml;         // [slots][tokens * heads]
    uint32_t tiles;          // many-rows kernel: row tiles of the launch
    // own part: rows per sequence that this launch takes, from .. to (the others are another's)
    uint32_t rows_from, rows_to;
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

// One warp: the sequence and the tile within it that tile number `want` is, when every
// sequence that this launch takes has ceil(rows / tile_rows) tiles, in order (kNone: there
// is no such tile).
__device__ __forceinline__ uint32_t find_tile(const AttnArgs& a, uint32_t want, uint32_t tile_rows, uint32_t* tile) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < a.b.seqs; s0 += 32u) {
        uint32_t cnt = 0;
        if (s0 + lane < a.b.seqs) {
            const uint32_t rows = load_seq(a.b, s0 + lane, a.st).n * a.group;
            if (rows >= a.rows_from && rows <= a.rows_to) cnt = (rows + tile_rows - 1u) / tile_rows;
        }
        uint32_t inc = cnt;
        for (uint32_t o = 1; o < 32u; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
            if (lane >= o) inc += v;
        }
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + inc > want);
        if (hit != 0u) {
            const uint32_t w = __ffs(hit) - 1u;
            *tile = want - before - __shfl_sync(0xFFFFFFFFu, inc - cnt, w);
            return s0 + w;
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

// The few-rows kernel on the tensor cores (paged_attention_few.cu): F16 caches, up to
// kFewRows query rows per tile.
constexpr uint32_t kFewRows = 8;
cudaError_t launch_attention_few(const AttnArgs& a, uint64_t items, cudaStream_t stream);
// The many-rows kernel on the tensor cores (paged_attention_many.cu): F16 caches, row
// tiles of kManyRows.
constexpr uint32_t kManyRows = 64;
cudaError_t launch_attention_many(const AttnArgs& a, uint64_t tiles, cudaStream_t stream);

}  // namespace nedo_gpu

// paged_attention_many.cu -- attention over a paged F16 or Q4_0 cache for tiles of 128 or 64 query rows of
// heads above 128 channels (prompts, and the tokens of a whole batch over their shared
// prefix): bound by the tensor cores.  (Up to 128 channels a tile's sums fit into the other
// kernel's half of TMEM.)
//
// Mathematics.  As in paged_attention_few.cu the fp32 factors are split in two fp16
// halves; here each half is an operand of its own, the low one first, so that the sums
// can be taken down before the high ones come and grow in few steps (the tensor core cuts its fp32 sums instead of rounding them; a
// tile's weighted values are therefore summed from zero in 4 steps and added to the
// running sums in fp32 with the rescaling by 2^(m_old - m_new)).
//
// Work.  A CTA of a warp for 16 rows takes its rows through its keys in tiles of 32; the tiles of keys and values are shared by the warps, brought in by cp.async two
// tiles deep.  Tiles that none of a warp's rows sees are skipped by it, and only tiles
// seen in part are masked.
//
// 12 query and 4 KV heads of 256 channels, 2048 and 1919 new tokens of two sequences over 4096 and
// 2929 keys: 869 us, 285 TFLOP/s of MMAs (two for each product), in tiles of 128 rows; 64 rows, which
// read the keys twice as often, take 1072.  Where there are few tiles 64 rows reach more SMs: 8 query
// and 2 KV heads, 300 tokens 26 us (128 rows: 30), 37 sequences of 32 tokens over 500 keys 51 us (68).
// The plan takes the height that it expects to end first.
//
// Of a Q4_0 cache (paged_q4.cuh) a thread copies the same blocks of 32 channels of every tile and makes
// fp16 numbers of its own copies.  Under 64 rows, one warp to a scheduler, four more warps do so for
// the tile ahead (300 tokens 30 us, 37 sequences 60; by the warps of the rows 33 and 70); under 128
// those of the rows, before the barrier that the tile waits for anyway (prompts of 1919 and 2048
// tokens over up to 4096 keys 888 us; a tile ahead, around the products of the one before, no faster).
#include "paged_attention.cuh"
#include "paged_mma.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kStages = 2;
constexpr uint32_t HD = 256;                             // channels of a row in shared memory
constexpr uint32_t kKeys = 32;                           // keys per tile
constexpr uint32_t kGroups = kKeys / 16u, kCols = kKeys / 8u;
constexpr uint32_t kRowBytes = HD * 2u;
constexpr uint32_t kTileBytes = kKeys * kRowBytes;       // keys or values of a tile
constexpr uint32_t kStageBytes = 2u * kTileBytes;

template <uint32_t ROWS, bool Q4>
struct Many {
    static constexpr uint32_t kRowThreads = 2u * ROWS;       // a warp for 16 rows
    // Q4_0: those that make the tiles, the last ones (64 rows: warps of their own)
    static constexpr bool kApart = Q4 && ROWS == 64u;
    static constexpr uint32_t kMakers = 2u * ROWS;
    static constexpr uint32_t kThreads = kApart ? kRowThreads + kMakers : kRowThreads;
    static constexpr uint32_t kQBytes = ROWS * kRowBytes;    // one half of the queries
    // Q4_0: a tile's blocks as they come, 16 bytes of numbers and two keys' scales each
    static constexpr uint32_t kRawBlocks = 2u * kKeys * (HD / 32u), kRawBytes = kRawBlocks * 20u;
    static constexpr uint32_t kSmem = 2u * kQBytes + kStages * (kStageBytes + (Q4 ? kRawBytes : 0u));
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) { return r * kRowBytes + ((c ^ (r & 7u)) << 4); }

template <uint32_t ROWS, bool Q4>
__device__ __forceinline__ void attention_many(const AttnArgs& a) {
    using M = Many<ROWS, Q4>;
    constexpr uint32_t kThreads = M::kThreads, kQBytes = M::kQBytes, kSmem = M::kSmem;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ uint32_t row_tok[ROWS], row_head[ROWS];
    __shared__ int row_pos[ROWS];
    __shared__ float row_unscale[ROWS];
    __shared__ uint32_t found[2];
    const uint32_t hd = a.kv.head_dim, tid = threadIdx.x, lane = tid & 31u;
    const uint32_t warp = M::kApart ? (tid >> 5) % (ROWS / 16u) : tid >> 5;  // (of the rows; a maker's does not matter)
    const bool of_rows = !M::kApart || tid < M::kRowThreads, maker = !M::kApart || tid >= M::kRowThreads;
    const uint32_t kh = blockIdx.x % a.kv.kv_heads;
    uint32_t rest = blockIdx.x / a.kv.kv_heads;
    const uint32_t c = rest % a.chunks;
    rest /= a.chunks;

    // rows
    uint32_t s = 0, r0 = 0, nrows, t0 = 0;
    PagedSeq sq{0u, 0u, 0u};
    if (a.part == kPartPrefix) {
        r0 = rest * ROWS;
        nrows = min(ROWS, a.b.tokens * a.group - r0);
    } else {
        if (tid < 32u) {
            uint32_t tile;
            const uint32_t seq = find_tile(a, rest, ROWS, &tile);
            if (lane == 0u) {
                found[0] = seq;
                found[1] = tile;
            }
        }
        __syncthreads();
        s = found[0];
        if (s == kNone) return;
        sq = load_seq(a.b, s, a.st);
        t0 = sq.t0;
        r0 = found[1] * ROWS;
        nrows = min(ROWS, sq.n * a.group - r0);
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
    // keys [kb, ke) of the tile and [wb, we) of this warp; [all_b, all_e): seen by all its rows
    uint32_t kb = kNone, ke = 0, wb = kNone, we = 0, all_b = 0, all_e = kNone;
    {
        uint32_t lo = kNone, hi = 0;
#pragma unroll
        for (uint32_t u = 0; u < ROWS / 32u; ++u) {
            const int p = row_pos[lane + 32u * u];
            if (p >= 0) {
                lo = min(lo, first_key(p, a.window));
                hi = max(hi, static_cast<uint32_t>(p) + 1u);
            }
        }
        kb = __reduce_min_sync(0xFFFFFFFFu, lo);
        ke = __reduce_max_sync(0xFFFFFFFFu, hi);
        const int p = row_pos[warp * 16u + (lane & 15u)];
        const uint32_t l1 = p >= 0 ? first_key(p, a.window) : kNone, h1 = p >= 0 ? static_cast<uint32_t>(p) + 1u : 0u;
        wb = __reduce_min_sync(0xFFFFFFFFu, l1);
        we = __reduce_max_sync(0xFFFFFFFFu, h1);
        all_b = __reduce_max_sync(0xFFFFFFFFu, p >= 0 ? l1 : 0u);
        all_e = __reduce_min_sync(0xFFFFFFFFu, p >= 0 ? h1 : kNone);
    }
    {
        uint32_t base = 0;
        if (a.part == kPartOwn) base = own_begin(sq, a.window, a.shared_len);
        else ke = min(ke, a.shared_len);
        const uint64_t cb = static_cast<uint64_t>(base) + static_cast<uint64_t>(c) * a.chunk;
        kb = cb > kb ? static_cast<uint32_t>(cb < kNone ? cb : kNone) : max(kb, base);
        if (cb + a.chunk < ke) ke = static_cast<uint32_t>(cb + a.chunk);
        if (kb >= ke && !a.direct) return;  // no row of the tile sees a key of this chunk
    }
    const uint32_t j0 = kb & ~(kKeys - 1u), ntiles = kb < ke ? (ke - j0 + kKeys - 1u) / kKeys : 0u;

    const uint32_t q_addr = smem_addr(sm), ring = q_addr + 2u * kQBytes;
    if (hd < HD) {  // channels beyond the head stay zero
        for (uint32_t i = tid; i < kSmem / 16u; i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    }
    const uint32_t chunks16 = hd >> 3;
    const __half* kbase = static_cast<const __half*>(a.kv.k);
    const __half* vbase = static_cast<const __half*>(a.kv.v);
    // pages of the next tile's groups of 16 keys (a group lies within one page)
    uint32_t pages[kGroups];
    auto look_up = [&](uint32_t i) {
#pragma unroll
        for (uint32_t u = 0; u < kGroups; ++u) {
            const uint32_t j = j0 + i * kKeys + u * 16u;
            pages[u] = i < ntiles && j < ke && j + 16u > kb ? load_page(a.b, a.kv, s, j >> a.kv.page_shift, a.st) : kNone;
        }
    };
    constexpr uint32_t kGaps = M::kApart ? 2u * kStages : kStages;
    __shared__ uint32_t tile_gap[kGaps];  // a page of the tile is no page
    // Q4_0: the thread's blocks x of a tile's keys, and of its values behind them
    constexpr uint32_t kMine = M::kRawBlocks / 2u / M::kMakers;
    const uint32_t me = M::kApart ? tid - M::kRowThreads : tid;
    auto raw_at = [&](uint32_t i, uint32_t x) { return 2u * kQBytes + kStages * kStageBytes + (i % kStages) * M::kRawBytes + (x * M::kMakers + me) * 16u; };
    auto raw_scale_at = [&](uint32_t i, uint32_t x) {
        return 2u * kQBytes + kStages * kStageBytes + (i % kStages) * M::kRawBytes + M::kRawBlocks * 16u + (x * M::kMakers + me) * 4u;
    };
    const uint32_t my_key = (me & 7u) + 8u * ((me >> 4) & 3u);
    auto block_of = [&](uint32_t x) { return ((me >> 3) & 1u) + 2u * ((x * M::kMakers + me) >> 6); };
    auto fetch = [&](uint32_t i) {
        if (i < ntiles) {
            const uint32_t dst = ring + (i % kStages) * kStageBytes;
            constexpr uint32_t kPer = kKeys * (HD / 8u) / kThreads;       // copies of 16 bytes per thread, keys and values each
            constexpr uint32_t kRowsAtOnce = kThreads / (HD / 8u);
            const uint32_t ch = tid % (HD / 8u);
            bool gap = false;
#pragma unroll
            for (uint32_t u = 0; u < kGroups; ++u) {
                const uint32_t j = j0 + i * kKeys + u * 16u;
                gap |= pages[u] == kNone && j < ke && j + 16u > kb;
            }
            if (me == 0u) tile_gap[i % kGaps] = gap;
            if constexpr (Q4) {
                const uint32_t j = j0 + i * kKeys + my_key;
                uint32_t page = pages[0];
#pragma unroll
                for (uint32_t u = 1; u < kGroups; ++u) page = my_key >= 16u * u ? pages[u] : page;
                const bool there = page != kNone && j >= kb && j < ke;
                const uint32_t slot = there ? j & (a.kv.page_size - 1u) : 0u, bytes = there ? 16u : 0u;
                const size_t o = ((there ? static_cast<size_t>(page) : 0u) * a.kv.kv_heads + kh) * q4_head_bytes(a.kv);
#pragma unroll
                for (uint32_t x = 0; x < 2u * kMine; ++x) {
                    const uint32_t b = block_of(x % kMine);
                    if (b * 32u >= hd) continue;
                    const uint8_t* from = static_cast<const uint8_t*>(x < kMine ? a.kv.k : a.kv.v) + o;
                    cp_async16(q_addr + raw_at(i, x), from + slot * (hd / 2u) + b * 16u, bytes);
                    cp_async4(q_addr + raw_scale_at(i, x), from + q4_scales_at(a.kv) + (b * a.kv.page_size + (slot & ~1u)) * 2u, bytes / 4u);
                }
            } else if (ch < chunks16) {
#pragma unroll
                for (uint32_t x = 0; x < kPer; ++x) {
                    const uint32_t r = tid / (HD / 8u) + x * kRowsAtOnce;
                    const uint32_t j = j0 + i * kKeys + r;
                    const uint32_t page = pages[x * kRowsAtOnce / 16u];  // r stays within the group
                    const bool there = page != kNone && j >= kb && j < ke;
                    const size_t o = (((there ? static_cast<size_t>(page) : 0u) * a.kv.kv_heads + kh) * a.kv.page_size +
                                      (there ? j & (a.kv.page_size - 1u) : 0u)) * hd + ch * 8u;
                    cp_async16(dst + at(r, ch), kbase + o, there ? 16u : 0u);
                    cp_async16(dst + kTileBytes + at(r, ch), vbase + o, there ? 16u : 0u);
                }
            }
        }
        cp_commit();
    };
    // Q4_0: tile i, once the thread's copies are there (of keys that are not: numbers and scales zero)
    auto make = [&](uint32_t i) {
        cp_wait<1>();
        if (i >= ntiles) return;
#pragma unroll
        for (uint32_t x = 0; x < 2u * kMine; ++x) {
            const uint32_t b = block_of(x % kMine);
            if (b * 32u >= hd) continue;
            const uint4 w = *reinterpret_cast<const uint4*>(sm + raw_at(i, x));
            const __half2 d = __half2half2(*reinterpret_cast<const __half*>(sm + raw_scale_at(i, x) + (my_key & 1u) * 2u));
            uint8_t* const to = sm + 2u * kQBytes + (i % kStages) * kStageBytes + (x < kMine ? 0u : kTileBytes);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (uint32_t u = 0; u < 4u; ++u) {
                __half2 h[4];
                q4_pairs(words[u], h);
                *reinterpret_cast<uint4*>(to + at(my_key, b * 4u + u)) =
                    make_uint4(pack(__hmul2(h[0], d)), pack(__hmul2(h[1], d)), pack(__hmul2(h[2], d)), pack(__hmul2(h[3], d)));
            }
        }
    };
    if (maker) {
        look_up(0);
        fetch(0);
        look_up(1);
    }

    // queries: scaled, split and stored; a row per two threads
    if (of_rows) {
        const uint32_t r = tid >> 1;
        const int p = row_pos[r];
        const float* q = a.q + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd;
        float big = 0.f;
        if (p >= 0)
            for (uint32_t d = (tid & 1u) * 8u; d < hd; d += 16u)
#pragma unroll
                for (uint32_t e = 0; e < 8; e += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(q + d + e);
                    big = fmaxf(big, fmaxf(fmaxf(fabsf(x.x * a.scale_log2), fabsf(x.y * a.scale_log2)),
                                           fmaxf(fabsf(x.z * a.scale_log2), fabsf(x.w * a.scale_log2))));
                }
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
        const int e2 = up_exponent(big);
        const float up = power_of_two(e2);
        if ((tid & 1u) == 0u) row_unscale[r] = power_of_two(-e2);
        for (uint32_t d = (tid & 1u) * 8u; d < HD; d += 16u) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                float2 x = make_float2(0.f, 0.f);
                if (p >= 0 && d < hd) x = *reinterpret_cast<const float2*>(q + d + 2u * e);
                split(x.x * a.scale_log2 * up, x.y * a.scale_log2 * up, &hi[e], &lo[e]);
            }
            *reinterpret_cast<uint4*>(sm + at(r, d >> 3)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(sm + kQBytes + at(r, d >> 3)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
    if (M::kApart && maker) {
        fetch(1);
        look_up(2);
        make(0);
    }
    __syncthreads();

    // this thread's rows g and g + 8 of the warp's 16
    const uint32_t g = lane >> 2, t2 = (lane & 3u) * 2u, mi = lane >> 3, mr = lane & 7u;
    float unscale[2], m[2], l[2];
    uint32_t lo_key[2], hi_key[2];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t r = warp * 16u + g + 8u * h;
        const int p = row_pos[r];
        unscale[h] = row_unscale[r];
        lo_key[h] = p >= 0 ? first_key(p, a.window) : kNone;
        hi_key[h] = p >= 0 ? static_cast<uint32_t>(p) + 1u : 0u;
        m[h] = -INFINITY;
        l[h] = 0.f;
    }
    float acc[HD / 8][4];
#pragma unroll
    for (uint32_t n = 0; n < HD / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;

    for (uint32_t i = 0; i < ntiles; ++i) {
        if constexpr (M::kApart) {  // the next tile is made meanwhile
            if (maker) {
                fetch(i + 2u);
                look_up(i + 3u);
                make(i + 1u);
            }
        } else {
            fetch(i + 1u);
            look_up(i + 2u);
            if constexpr (Q4) make(i);
            else cp_wait<1>();
            __syncthreads();
        }
        const uint32_t j = j0 + i * kKeys;
        if (of_rows && j < we && j + kKeys > wb) {
            const uint32_t ks = ring + (i % kStages) * kStageBytes, vs = ks + kTileBytes;
            float sc[kCols][4];
#pragma unroll
            for (uint32_t n = 0; n < kCols; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
            float low[kCols][4];  // from the low halves: a part of its own, so that the keys are loaded once
#pragma unroll
            for (uint32_t n = 0; n < kCols; ++n) low[n][0] = low[n][1] = low[n][2] = low[n][3] = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < HD / 16; ++k) {
                uint32_t qhi[4], qlo[4];
                const uint32_t q_at = q_addr + at(warp * 16u + (mi & 1u) * 8u + mr, 2u * k + (mi >> 1));
                ldsm4(qhi, q_at);
                ldsm4(qlo, q_at + kQBytes);
#pragma unroll
                for (uint32_t n = 0; n < kGroups; ++n) {
                    uint32_t b[4];
                    ldsm4(b, ks + at(n * 16u + (mi >> 1) * 8u + mr, 2u * k + (mi & 1u)));
                    mma(low[2 * n], qlo, b[0], b[1]);
                    mma(low[2 * n + 1], qlo, b[2], b[3]);
                    mma(sc[2 * n], qhi, b[0], b[1]);
                    mma(sc[2 * n + 1], qhi, b[2], b[3]);
                }
            }
#pragma unroll
            for (uint32_t n = 0; n < kCols; ++n)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) sc[n][e] = fmaf(low[n][e], kLowDown, sc[n][e]);
            const bool gap = tile_gap[i % kGaps] != 0u;
            const bool whole = !gap && j >= all_b && j + kKeys <= all_e && j >= kb && j + kKeys <= ke;
            if (!whole) {
                uint32_t there = ~0u;  // groups of 16 keys whose page is a page
                if (gap) {
                    there = 0u;
#pragma unroll
                    for (uint32_t u = 0; u < kGroups; ++u) {
                        const uint32_t jj = j + u * 16u;
                        if (jj < ke && jj + 16u > kb && load_page(a.b, a.kv, s, jj >> a.kv.page_shift, a.st) != kNone)
                            there |= 1u << u;
                    }
                }
#pragma unroll
                for (uint32_t n = 0; n < kCols; ++n)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const uint32_t key = j + n * 8u + t2 + (e & 1u), h = e >> 1;
                        if (key < lo_key[h] || key >= hi_key[h] || key < kb || key >= ke || !(there >> (n >> 1) & 1u))
                            sc[n][e] = -INFINITY;
                    }
            }
            float alpha[2], ref[2];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                float mt = sc[0][2 * h];
#pragma unroll
                for (uint32_t n = 0; n < kCols; ++n) mt = fmaxf(mt, fmaxf(sc[n][2 * h], sc[n][2 * h + 1]));
                mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 1));
                mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 2));
                const float mn = fmaxf(m[h], mt * unscale[h]);
                alpha[h] = mn == -INFINITY ? 1.f : exp2_fast(m[h] - mn);
                m[h] = mn;
                ref[h] = (mn == -INFINITY ? 0.f : mn) - kUp;
                l[h] *= alpha[h];
            }
            uint32_t phi[kGroups][4], plo[kGroups][4];
#pragma unroll
            for (uint32_t n = 0; n < kCols; ++n) {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    sc[n][e] = exp2_fast(fmaf(sc[n][e], unscale[e >> 1], -ref[e >> 1]));
                    l[e >> 1] += sc[n][e];
                }
                split(sc[n][0], sc[n][1], &phi[n >> 1][(n & 1u) * 2u], &plo[n >> 1][(n & 1u) * 2u]);
                split(sc[n][2], sc[n][3], &phi[n >> 1][(n & 1u) * 2u + 1u], &plo[n >> 1][(n & 1u) * 2u + 1u]);
            }
#pragma unroll
            for (uint32_t n = 0; n < HD / 16; ++n) {
                float o[2][4];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) o[0][e] = o[1][e] = 0.f;
                uint32_t b[kGroups][4];
#pragma unroll
                for (uint32_t k = 0; k < kGroups; ++k)
                    ldsm4t(b[k], vs + at(k * 16u + (mi & 1u) * 8u + mr, 2u * n + (mi >> 1)));
#pragma unroll
                for (uint32_t k = 0; k < kGroups; ++k) {
                    mma(o[0], plo[k], b[k][0], b[k][1]);
                    mma(o[1], plo[k], b[k][2], b[k][3]);
                }
                low_down(o[0]);
                low_down(o[1]);
#pragma unroll
                for (uint32_t k = 0; k < kGroups; ++k) {
                    mma(o[0], phi[k], b[k][0], b[k][1]);
                    mma(o[1], phi[k], b[k][2], b[k][3]);
                }
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    acc[2 * n][e] = fmaf(acc[2 * n][e], alpha[e >> 1], o[0][e]);
                    acc[2 * n + 1][e] = fmaf(acc[2 * n + 1][e], alpha[e >> 1], o[1][e]);
                }
            }
        }
        __syncthreads();
    }
    cp_wait<0>();
    asm volatile("griddepcontrol.launch_dependents;");
    if (!of_rows) return;
    const size_t rows_all = static_cast<size_t>(a.b.tokens) * a.heads;
    uint32_t again = 0;  // rows of the warp whose sums are not finite
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
        const uint32_t r = warp * 16u + g + 8u * h;
        const int p = row_pos[r];
        float odd = l[h] * 0.f;
#pragma unroll
        for (uint32_t n = 0; n < HD / 8; ++n) odd = fmaf(acc[n][2 * h], 0.f, fmaf(acc[n][2 * h + 1], 0.f, odd));
        const bool redo = __ballot_sync(0xFFFFFFFFu, odd != 0.f && p >= 0) >> (lane & ~3u) & 15u;
        if (redo) again |= 1u << (g + 8u * h);
        if (p == -2 || redo) continue;
        if (p < 0) l[h] = 0.f;  // padding sees nothing
        const size_t row = static_cast<size_t>(row_tok[r]) * a.heads + row_head[r];
        float* o = a.direct ? a.out + row * hd : a.part_o + ((a.slot0 + c) * rows_all + row) * hd;
        const float f = !a.direct ? 1.f : l[h] == 0.f ? 0.f : 1.f / l[h];
        const bool none = l[h] == 0.f;
#pragma unroll
        for (uint32_t n = 0; n < HD / 8; ++n) {
            if (n * 8u >= hd) continue;
            *reinterpret_cast<float2*>(o + n * 8u + t2) =
                none ? make_float2(0.f, 0.f) : make_float2(acc[n][2 * h] * f, acc[n][2 * h + 1] * f);
        }
        if (!a.direct && (lane & 3u) == 0u)
            a.part_ml[(a.slot0 + c) * rows_all + row] = make_float2((m[h] == -INFINITY ? 0.f : m[h]) - kUp, l[h]);
    }
    again = __reduce_or_sync(0xFFFFFFFFu, again);
    while (again != 0u) {
        uint32_t n, rows = take_rows(&again, &n);
        RowSums x;
        rows_key_by_key<Q4>(a, s, kh, nullptr, {row_tok, row_head, row_pos}, warp * 16u, rows, kb, ke, 16u, 32u, &x);
        for (uint32_t u = 0; u < n; ++u, rows >>= 8) {
            const uint32_t r = warp * 16u + (rows & 255u);
            const size_t row = static_cast<size_t>(row_tok[r]) * a.heads + row_head[r];
            float* o = a.direct ? a.out + row * hd : a.part_o + ((a.slot0 + c) * rows_all + row) * hd;
            const float f = !a.direct ? 1.f : x.l[u] == 0.f ? 0.f : 1.f / x.l[u];
            for (uint32_t i = 0; lane + 32u * i < hd; ++i) o[lane + 32u * i] = x.o[u][i] * f;
            if (!a.direct && lane == 0u) a.part_ml[(a.slot0 + c) * rows_all + row] = make_float2(x.m[u], x.l[u]);
        }
    }
}

template <uint32_t ROWS, bool Q4>
__global__ void __launch_bounds__(Many<ROWS, Q4>::kThreads, 1) attention_many_kernel(const __grid_constant__ AttnArgs a) {
    attention_many<ROWS, Q4>(a);
    end_after_previous(a);
}

template <uint32_t ROWS, bool Q4>
cudaError_t launch(const AttnArgs& a, uint64_t items, cudaStream_t stream) {
    return launch_items(a, attention_many_kernel<ROWS, Q4>, items, Many<ROWS, Q4>::kThreads, Many<ROWS, Q4>::kSmem, stream, a);
}

}  // namespace

cudaError_t launch_attention_many(const AttnArgs& a, uint32_t rows, uint64_t tiles, cudaStream_t stream) {
    const uint64_t items = tiles * a.kv.kv_heads * a.chunks;
    if (a.kv.type == kQ4_0) return rows <= 64u ? launch<64, true>(a, items, stream) : launch<128, true>(a, items, stream);
    return rows <= 64u ? launch<64, false>(a, items, stream) : launch<128, false>(a, items, stream);
}

}  // namespace nedo_gpu

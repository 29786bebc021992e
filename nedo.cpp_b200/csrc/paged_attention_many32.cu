// paged_attention_many32.cu -- attention over a paged F32 cache for tiles of many query rows
// (prompts, and the tokens of a whole batch over their shared prefix): bound by the tensor
// cores.
//
// Mathematics.  Both factors of each product are fp32 here, so both are split in two fp16
// halves (22 bits), x = hi + 2^-11 lo, and three of the four products are formed: hi hi, and in
// sums of their own lo hi + hi lo; what is left out is 2^-22 of the product.  Queries are scaled by a
// power of two per row, keys and values by one per tile, weights by 2^14.  A tile's weighted values
// are summed from zero and added to the running sums in fp32, which also takes the scales back.
// With the low halves taken up by 2^11 a number keeps its 22 bits down to 2^-27 of the tile's
// largest, and 2^-49 of that below.  A tile in which numbers are below 2^-27 together -- four
// neighbouring channels of a key, or a channel of the keys that a thread looks at -- is done in fp32,
// key by key: a row must not lose its digits to a key that it does not see, nor a channel to its
// neighbours.  So is a tile with numbers that are not finite.
//
// Work.  A CTA of one warp for 16 rows (128 rows, 64 for heads above 128) takes its rows through
// their keys in tiles of 64 (32).  The next tile's keys and values are on their way (cp.async)
// while this one is multiplied; a tile that has landed is read once by all threads, its largest
// magnitudes found, and its halves written next to it for ldmatrix, once for all warps.
//
// 12 query and 4 KV heads of 128 channels, 2048 and 1840 new tokens of two sequences over 4096 and
// 2550 keys, window 2048: 567 us, 230 TFLOP/s of MMAs (three for each product).  With two warps to
// a scheduler the tensor pipe is busy for half of the time; the rest is the halves' making and
// the latency of what stands between the MMAs.
#include "paged_attention.cuh"
#include "paged_mma.cuh"

namespace nedo_gpu {
namespace {

constexpr float kDown = 1.f / 16384.f;  // 2^-kUp
constexpr float kRange = 134217728.f;   // 2^27: numbers of 2^14 and 2^-14 under one scale

template <uint32_t HD>
struct Many32 {
    static constexpr uint32_t kRows = HD <= 128u ? 128u : 64u;
    static constexpr uint32_t kWarps = kRows / 16u;
    static constexpr uint32_t kThreads = 32u * kWarps;
    static constexpr uint32_t kKeys = HD <= 128u ? 64u : 32u;
    static constexpr uint32_t kRowBytes = HD * 2u;                     // a row of halves
    static constexpr uint32_t kQBytes = kRows * kRowBytes;             // one half of the queries
    static constexpr uint32_t kHalfBytes = kKeys * kRowBytes;          // one half of a tile's keys or values
    static constexpr uint32_t kRawBytes = kKeys * HD * 4u;             // a tile's keys or values as they come
    static constexpr uint32_t kSmem = 2u * kQBytes + 4u * kHalfBytes + 2u * kRawBytes;
};

template <uint32_t HD>
__device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) {
    return r * Many32<HD>::kRowBytes + ((c ^ (r & 7u)) << 4);
}

template <uint32_t HD>
__device__ __forceinline__ void attention_many32(const AttnArgs& a) {
    using M = Many32<HD>;
    constexpr uint32_t kRows = M::kRows, kKeys = M::kKeys, kGroups = kKeys / 16u, kCols = kKeys / 8u, kThreads = M::kThreads;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ uint32_t row_tok[kRows], row_head[kRows];
    __shared__ int row_pos[kRows];
    __shared__ float row_unscale[kRows];
    __shared__ uint32_t found[2], size[2][M::kWarps], least[2][M::kWarps];
    const uint32_t hd = a.kv.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t kh = blockIdx.x % a.kv.kv_heads;
    uint32_t rest = blockIdx.x / a.kv.kv_heads;
    const uint32_t c = rest % a.chunks;
    rest /= a.chunks;

    // rows
    uint32_t s = 0, r0 = 0, nrows, t0 = 0;
    PagedSeq sq{0u, 0u, 0u};
    if (a.part == kPartPrefix) {
        r0 = rest * kRows;
        nrows = min(kRows, a.b.tokens * a.group - r0);
    } else {
        if (warp == 0) {
            uint32_t tile;
            const uint32_t seq = find_tile(a, rest, kRows, &tile);
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
        r0 = found[1] * kRows;
        nrows = min(kRows, sq.n * a.group - r0);
    }
    if (tid < kRows) {
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
        for (uint32_t u = 0; u < kRows / 32u; ++u) {
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

    uint8_t* const halves = sm + 2u * M::kQBytes;                 // keys hi, lo, values hi, lo
    uint8_t* const raw = halves + 4u * M::kHalfBytes;             // keys, values
    const uint32_t q_addr = smem_addr(sm), k_addr = smem_addr(halves), v_addr = k_addr + 2u * M::kHalfBytes;
    if (hd < HD) {  // channels beyond the head stay zero
        for (uint32_t i = tid; i < M::kSmem / 16u; i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    }
    const uint32_t chunks16 = hd >> 2;
    const float* kbase = static_cast<const float*>(a.kv.k);
    const float* vbase = static_cast<const float*>(a.kv.v);
    // pages of the next tile's groups of 16 keys (a group lies within one page)
    uint32_t pages[kGroups];
    auto look_up = [&](uint32_t i) {
#pragma unroll
        for (uint32_t u = 0; u < kGroups; ++u) {
            const uint32_t j = j0 + i * kKeys + u * 16u;
            pages[u] = i < ntiles && j < ke && j + 16u > kb ? load_page(a.b, a.kv, s, j >> a.kv.page_shift, a.st) : kNone;
        }
    };
    uint32_t there = 0;  // groups of the tile on its way whose page is a page, or that no row sees
    // 16-byte pieces x of a tile: the same ones are copied and read back by the same thread
    constexpr uint32_t kPieces = kKeys * (HD / 4u) / kThreads, kAtOnce = kThreads / (HD / 4u);
    const uint32_t piece_ch = tid % (HD / 4u), piece_row = tid / (HD / 4u);
    auto fetch = [&](uint32_t i) {
        if (i < ntiles) {
            there = 0u;
#pragma unroll
            for (uint32_t u = 0; u < kGroups; ++u) {
                const uint32_t j = j0 + i * kKeys + u * 16u;
                if (pages[u] != kNone || j >= ke || j + 16u <= kb) there |= 1u << u;
            }
            if (piece_ch < chunks16) {
#pragma unroll
                for (uint32_t x = 0; x < kPieces; ++x) {
                    const uint32_t r = piece_row + x * kAtOnce, j = j0 + i * kKeys + r;
                    uint32_t page = pages[0];
#pragma unroll
                    for (uint32_t u = 1; u < kGroups; ++u) page = r >= 16u * u ? pages[u] : page;
                    const bool in = page != kNone && j >= kb && j < ke;
                    const size_t o = (((in ? static_cast<size_t>(page) : 0u) * a.kv.kv_heads + kh) * a.kv.page_size +
                                      (in ? j & (a.kv.page_size - 1u) : 0u)) * hd + piece_ch * 4u;
                    const uint32_t dst = smem_addr(raw) + (r * (HD / 4u) + piece_ch) * 16u;
                    cp_async16(dst, kbase + o, in ? 16u : 0u);
                    cp_async16(dst + M::kRawBytes, vbase + o, in ? 16u : 0u);
                }
            }
        }
        cp_commit();
    };
    look_up(0);
    fetch(0);
    look_up(1);

    // queries: scaled, split and stored; a row per two threads
    {
        const uint32_t r = tid >> 1;
        const int p = row_pos[r];
        const float* q = a.q + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd;
        float big = 0.f;
        if (p >= 0)
            for (uint32_t d = (tid & 1u) * 4u; d < hd; d += 8u) {
                const float4 x = *reinterpret_cast<const float4*>(q + d);
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
                split(make_float2(x.x * a.scale_log2 * up, x.y * a.scale_log2 * up), &hi[e], &lo[e]);
            }
            *reinterpret_cast<uint4*>(sm + at<HD>(r, d >> 3)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(sm + M::kQBytes + at<HD>(r, d >> 3)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
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
        const uint32_t have = there, j = j0 + i * kKeys;
        cp_wait<0>();
        // the tile as halves: every thread its own pieces (the ones it copied), first their sizes
        // (twice their bits, without the sign; for the smallest less one, which leaves zero out): the
        // largest of all, the smallest of the largest of four channels and of the thread's keys
        uint32_t big[2] = {0u, 0u}, small[2] = {~0u, ~0u}, top[2][4] = {};
        constexpr bool kHold = HD <= 128u;  // in registers from the one pass to the other
        float4 held[kHold ? kPieces : 1u][2];
#pragma unroll
        for (uint32_t x = 0; x < kPieces; ++x) {
            const uint32_t piece = (piece_row + x * kAtOnce) * (HD / 4u) + piece_ch;
#pragma unroll
            for (uint32_t kv = 0; kv < 2u; ++kv) {
                const float4 v = *reinterpret_cast<const float4*>(raw + kv * M::kRawBytes + piece * 16u);
                if constexpr (kHold) held[x][kv] = v;
                const uint32_t e[4] = {__float_as_uint(v.x) << 1, __float_as_uint(v.y) << 1, __float_as_uint(v.z) << 1,
                                       __float_as_uint(v.w) << 1};
                small[kv] = min(small[kv], max(max(e[0], e[1]), max(e[2], e[3])) - 1u);
#pragma unroll
                for (uint32_t u = 0; u < 4u; ++u) top[kv][u] = max(top[kv][u], e[u]);
            }
        }
#pragma unroll
        for (uint32_t kv = 0; kv < 2u; ++kv) {
#pragma unroll
            for (uint32_t u = 0; u < 4u; ++u) {
                big[kv] = max(big[kv], top[kv][u]);
                small[kv] = min(small[kv], top[kv][u] - 1u);
            }
            big[kv] = __reduce_max_sync(0xFFFFFFFFu, big[kv]);
            small[kv] = __reduce_min_sync(0xFFFFFFFFu, small[kv]);
            if (lane == 0u) {
                size[kv][warp] = big[kv];
                least[kv][warp] = small[kv];
            }
        }
        __syncthreads();  // also: all warps are done with the halves of the tile before
#pragma unroll
        for (uint32_t w = 0; w < M::kWarps; ++w) {
#pragma unroll
            for (uint32_t kv = 0; kv < 2u; ++kv) {
                big[kv] = max(big[kv], size[kv][w]);
                small[kv] = min(small[kv], least[kv][w]);
            }
        }
        const float k_big = __uint_as_float(big[0] >> 1), v_big = __uint_as_float(big[1] >> 1);
        auto least_of = [](uint32_t x) { return __uint_as_float((x + 1u) >> 1); };
        const bool slow = max(big[0], big[1]) >= 0xFF000000u || (big[0] != 0u && k_big > least_of(small[0]) * kRange) ||
                          (big[1] != 0u && v_big > least_of(small[1]) * kRange);
        const int ek = up_exponent(k_big), ev = up_exponent(v_big);
        const float k_up = power_of_two(ek), v_up = power_of_two(ev), k_down = power_of_two(-ek);
        // takes the tile's scale back, and the weights': the running sums hold weights of at most 1, or
        // values near fp32's largest would leave it
        const float v_down = power_of_two(-ev) * kDown;
#pragma unroll
        for (uint32_t x = 0; x < kPieces; ++x) {
            const uint32_t r = piece_row + x * kAtOnce, piece = r * (HD / 4u) + piece_ch;
#pragma unroll
            for (uint32_t kv = 0; kv < 2u; ++kv) {
                float4 v;
                if constexpr (kHold) v = held[x][kv];
                else v = *reinterpret_cast<const float4*>(raw + kv * M::kRawBytes + piece * 16u);
                const float up = kv ? v_up : k_up;
                const float2 up2 = make_float2(up, up);
                uint32_t hi[2], lo[2];
                split(__fmul2_rn(make_float2(v.x, v.y), up2), &hi[0], &lo[0]);
                split(__fmul2_rn(make_float2(v.z, v.w), up2), &hi[1], &lo[1]);
                uint8_t* dst = halves + kv * 2u * M::kHalfBytes + at<HD>(r, piece_ch >> 1) + (piece_ch & 1u) * 8u;
                *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(dst + M::kHalfBytes) = make_uint2(lo[0], lo[1]);
            }
        }
        fetch(i + 1u);  // into the thread's own pieces, which it has read
        look_up(i + 2u);
        __syncthreads();
        if (j < we && j + kKeys > wb) {
            const bool whole = have == (1u << kGroups) - 1u && j >= all_b && j + kKeys <= all_e && j >= kb && j + kKeys <= ke;
            float sc[kCols][4];
#pragma unroll
            for (uint32_t n = 0; n < kCols; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
            // where key `key` of the tile lies in the cache, if it is one of the item's
            auto in_tile = [&](uint32_t key) { return key >= kb && key < ke && (have >> ((key - j) >> 4) & 1u); };
            auto place = [&](uint32_t key) -> size_t {
                const uint32_t page = a.b.table[static_cast<size_t>(s) * a.b.max_pages + (key >> a.kv.page_shift)];
                return ((static_cast<size_t>(page) * a.kv.kv_heads + kh) * a.kv.page_size + (key & (a.kv.page_size - 1u))) * hd;
            };
            if (slow) {
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    const uint32_t r = warp * 16u + g + 8u * h;
                    const float* q = a.q + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd;
#pragma unroll
                    for (uint32_t n = 0; n < kCols; ++n)
#pragma unroll
                        for (uint32_t e = 0; e < 2; ++e) {
                            const uint32_t key = j + n * 8u + t2 + e;
                            if (!in_tile(key) || key < lo_key[h] || key >= hi_key[h]) continue;
                            const float* kr = kbase + place(key);
                            float sum = 0.f;
                            for (uint32_t d = 0; d < hd; ++d) sum = fmaf(q[d] * a.scale_log2, kr[d], sum);
                            sc[n][2 * h + e] = sum;
                        }
                }
            } else {
                float low[kCols][4];  // lo hi + hi lo
#pragma unroll
                for (uint32_t n = 0; n < kCols; ++n) low[n][0] = low[n][1] = low[n][2] = low[n][3] = 0.f;
#pragma unroll
                for (uint32_t k = 0; k < HD / 16; ++k) {
                    uint32_t qhi[4], qlo[4];
                    const uint32_t q_at = q_addr + at<HD>(warp * 16u + (mi & 1u) * 8u + mr, 2u * k + (mi >> 1));
                    ldsm4(qhi, q_at);
                    ldsm4(qlo, q_at + M::kQBytes);
#pragma unroll
                    for (uint32_t n = 0; n < kGroups; ++n) {
                        uint32_t bhi[4], blo[4];
                        const uint32_t k_at = k_addr + at<HD>(n * 16u + (mi >> 1) * 8u + mr, 2u * k + (mi & 1u));
                        ldsm4(bhi, k_at);
                        ldsm4(blo, k_at + M::kHalfBytes);
                        mma(low[2 * n], qlo, bhi[0], bhi[1]);
                        mma(low[2 * n + 1], qlo, bhi[2], bhi[3]);
                        mma(sc[2 * n], qhi, bhi[0], bhi[1]);
                        mma(sc[2 * n + 1], qhi, bhi[2], bhi[3]);
                        mma(low[2 * n], qhi, blo[0], blo[1]);
                        mma(low[2 * n + 1], qhi, blo[2], blo[3]);
                    }
                }
#pragma unroll
                for (uint32_t n = 0; n < kCols; ++n)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) sc[n][e] = fmaf(low[n][e], kLowDown, sc[n][e]);
            }
            const float k_one = slow ? 1.f : k_down;
            if (!whole) {
#pragma unroll
                for (uint32_t n = 0; n < kCols; ++n)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const uint32_t key = j + n * 8u + t2 + (e & 1u), h = e >> 1;
                        if (key < lo_key[h] || key >= hi_key[h] || key < kb || key >= ke || !(have >> (n >> 1) & 1u))
                            sc[n][e] = -INFINITY;
                    }
            }
            float alpha[2], ref[2], down[2];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                float mt = sc[0][2 * h];
#pragma unroll
                for (uint32_t n = 0; n < kCols; ++n) mt = fmaxf(mt, fmaxf(sc[n][2 * h], sc[n][2 * h + 1]));
                mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 1));
                mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 2));
                // the two powers one after the other: together they may leave fp32's range
                down[h] = slow ? 1.f : unscale[h];
                const float mn = fmaxf(m[h], mt * down[h] * k_one);
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
                    sc[n][e] = exp2_fast(fmaf(sc[n][e] * down[e >> 1], k_one, -ref[e >> 1]));
                    l[e >> 1] += sc[n][e];
                }
                split(make_float2(sc[n][0], sc[n][1]), &phi[n >> 1][(n & 1u) * 2u], &plo[n >> 1][(n & 1u) * 2u]);
                split(make_float2(sc[n][2], sc[n][3]), &phi[n >> 1][(n & 1u) * 2u + 1u], &plo[n >> 1][(n & 1u) * 2u + 1u]);
            }
            if (!slow) {
#pragma unroll
                for (uint32_t n = 0; n < HD / 16; ++n) {
                    float o[2][4];
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) o[0][e] = o[1][e] = 0.f;
                    const uint32_t v_at = v_addr + at<HD>((mi & 1u) * 8u + mr, 2u * n + (mi >> 1));  // 16 keys: 16 rows on
                    if constexpr (HD <= 128u) {
                        // hi hi on top of lo hi + hi lo: fewer registers (sums of their own took 575 us for the case above)
                        uint32_t b[kGroups][4];
#pragma unroll
                        for (uint32_t k = 0; k < kGroups; ++k) ldsm4t(b[k], v_at + k * 16u * M::kRowBytes + M::kHalfBytes);
#pragma unroll
                        for (uint32_t k = 0; k < kGroups; ++k) {
                            mma(o[0], phi[k], b[k][0], b[k][1]);
                            mma(o[1], phi[k], b[k][2], b[k][3]);
                        }
#pragma unroll
                        for (uint32_t k = 0; k < kGroups; ++k) ldsm4t(b[k], v_at + k * 16u * M::kRowBytes);
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
                    } else {
                        float low[2][4];  // (392 us for prompts of 900 and 671 tokens; as above 413)
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) low[0][e] = low[1][e] = 0.f;
#pragma unroll
                        for (uint32_t k = 0; k < kGroups; ++k) {
                            uint32_t bhi[4], blo[4];
                            ldsm4t(bhi, v_at + k * 16u * M::kRowBytes);
                            ldsm4t(blo, v_at + k * 16u * M::kRowBytes + M::kHalfBytes);
                            mma(low[0], plo[k], bhi[0], bhi[1]);
                            mma(low[1], plo[k], bhi[2], bhi[3]);
                            mma(o[0], phi[k], bhi[0], bhi[1]);
                            mma(o[1], phi[k], bhi[2], bhi[3]);
                            mma(low[0], phi[k], blo[0], blo[1]);
                            mma(low[1], phi[k], blo[2], blo[3]);
                        }
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) {
                            o[0][e] = fmaf(low[0][e], kLowDown, o[0][e]);
                            o[1][e] = fmaf(low[1][e], kLowDown, o[1][e]);
                        }
                    }
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        acc[2 * n][e] = fmaf(acc[2 * n][e], alpha[e >> 1], o[0][e] * v_down);
                        acc[2 * n + 1][e] = fmaf(acc[2 * n + 1][e], alpha[e >> 1], o[1][e] * v_down);
                    }
                }
            } else {
#pragma unroll
                for (uint32_t n = 0; n < HD / 8; ++n)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) acc[n][e] *= alpha[e >> 1];
#pragma unroll
                for (uint32_t n8 = 0; n8 < kCols; ++n8) {
                    for (uint32_t jj = 0; jj < 8; ++jj) {
                        const uint32_t from = (lane & ~3u) | (jj >> 1), key = j + n8 * 8u + jj;
                        float w[2];
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const float w0 = __shfl_sync(0xFFFFFFFFu, sc[n8][2 * h], from);
                            const float w1 = __shfl_sync(0xFFFFFFFFu, sc[n8][2 * h + 1], from);
                            w[h] = (jj & 1u ? w1 : w0) * kDown;
                        }
                        if (!in_tile(key)) continue;
                        const bool see0 = key >= lo_key[0] && key < hi_key[0], see1 = key >= lo_key[1] && key < hi_key[1];
                        const float* vr = vbase + place(key);
#pragma unroll
                        for (uint32_t n = 0; n < HD / 8; ++n) {
                            if (n * 8u >= hd) continue;
                            const float f0 = vr[n * 8u + t2], f1 = vr[n * 8u + t2 + 1u];
                            if (see0) {
                                acc[n][0] = fmaf(w[0], f0, acc[n][0]);
                                acc[n][1] = fmaf(w[0], f1, acc[n][1]);
                            }
                            if (see1) {
                                acc[n][2] = fmaf(w[1], f0, acc[n][2]);
                                acc[n][3] = fmaf(w[1], f1, acc[n][3]);
                            }
                        }
                    }
                }
            }
        }
    }
    cp_wait<0>();
    asm volatile("griddepcontrol.launch_dependents;");
    const size_t rows_all = static_cast<size_t>(a.b.tokens) * a.heads;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
        const uint32_t r = warp * 16u + g + 8u * h;
        const int p = row_pos[r];
        if (p == -2) continue;
        l[h] = p < 0 ? 0.f : l[h] * kDown;  // padding sees nothing
        const size_t row = static_cast<size_t>(row_tok[r]) * a.heads + row_head[r];
        float* o = a.direct ? a.out + row * hd : a.part_o + ((a.slot0 + c) * rows_all + row) * hd;
        const bool none = l[h] == 0.f;
#pragma unroll
        for (uint32_t n = 0; n < HD / 8; ++n) {
            if (n * 8u >= hd) continue;
            const float f = a.direct ? l[h] : 1.f;
            *reinterpret_cast<float2*>(o + n * 8u + t2) =
                none ? make_float2(0.f, 0.f) : make_float2(acc[n][2 * h] / f, acc[n][2 * h + 1] / f);
        }
        if (!a.direct && (lane & 3u) == 0u)
            a.part_ml[(a.slot0 + c) * rows_all + row] = make_float2(m[h] == -INFINITY ? 0.f : m[h], l[h]);
    }
}

template <uint32_t HD>
__global__ void __launch_bounds__(Many32<HD>::kThreads, 1) attention_many32_kernel(const __grid_constant__ AttnArgs a) {
    attention_many32<HD>(a);
    end_after_previous(a);
}

template <uint32_t HD>
cudaError_t launch(const AttnArgs& a, uint64_t items, cudaStream_t stream) {
    return launch_items(a, attention_many32_kernel<HD>, items, Many32<HD>::kThreads, Many32<HD>::kSmem, stream, a);
}

}  // namespace

uint32_t many32_rows(uint32_t head_dim) { return head_dim <= 128u ? 128u : 64u; }

cudaError_t launch_attention_many32(const AttnArgs& a, uint64_t tiles, cudaStream_t stream) {
    const uint64_t items = tiles * a.kv.kv_heads * a.chunks;
    if (a.kv.head_dim <= 64u) return launch<64>(a, items, stream);
    if (a.kv.head_dim <= 128u) return launch<128>(a, items, stream);
    return launch<256>(a, items, stream);
}

}  // namespace nedo_gpu

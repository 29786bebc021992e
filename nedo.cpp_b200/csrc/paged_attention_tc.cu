// paged_attention_tc.cu -- attention over a paged F16 cache for tiles of 128 query rows on
// the 5th-generation tensor cores (prompts, the tokens of a whole batch over their shared
// prefix, groups of more than eight rows), heads of up to 128 channels.
//
// Mathematics.  As in the other tensor-core kernels the fp32 factors are split in two fp16
// halves, low halves first: S = q_lo K^T + q_hi K^T, O = p_lo V + p_hi V, so every 128 x 128
// tile is 32 MMAs of 128 x 128 x 16.  The tensor core cuts its fp32 sums instead of rounding
// them, so a tile's O starts from zero in TMEM and is added to the running sums in fp32
// registers, together with the rescaling by 2^(m_old - m_new).
//
// Work.  A CTA (one per SM, 640 threads) takes 128 rows through their keys in tiles of 128:
//   * warp 16 brings keys and values in by TMA (one 64-channel box per page piece, 128-byte
//     swizzle), in the order of their use, four half-tile slots deep.  Of a tile that the
//     item's key range cuts it zeroes the values outside, whatever the pages hold there;
//   * one thread of warp 17 issues the MMAs: Q K^T of tile i + 1 before P V of tile i, so the
//     tensor core works while a softmax runs;
//   * warps 0-7 take the even and warps 8-15 the odd tiles, two threads to a row, each with
//     half of the tile's keys and half of the channels: they read S from TMEM, agree on the
//     row's maximum, write the split weights over S (the A operand of P V), and add O to their
//     running sums.  The even and the odd sums meet at the end in shared memory.
// TMEM: two S/P and two O tiles of 128 columns each.  Registers: the softmax threads hold 64
// sums each, so they take 104 registers and the other warps give theirs up.
#include <algorithm>

#include "paged_attention.cuh"
#include "paged_mma.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kRows = kTcRows;     // 128
constexpr uint32_t kKeys = 128;         // keys per tile
constexpr uint32_t kSlots = 4;          // ring slots: the keys or the values of one tile
constexpr uint32_t kSoftmax = 512;      // softmax threads: four to a row
constexpr uint32_t kThreads = kSoftmax + 128;
constexpr uint32_t kBlock = kRows * 128u;  // bytes of 64 channels of a tile: rows of 128 bytes
constexpr uint32_t kLoadWarp = 16, kMmaWarp = 17;

template <uint32_t HD>
struct Tc {
    static constexpr uint32_t kBlocks = HD / 64u;
    static constexpr uint32_t kTile = kBlocks * kBlock;   // one half of the queries, or a ring slot
    static constexpr uint32_t kSmem = 2u * kTile + kSlots * kTile + 1024u;
};

struct TcMaps {
    CUtensorMap k, v;  // [num_pages * kv_heads][page_size][head_dim], boxes of 64 channels x box_rows slots
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int32_t c0, int32_t c1, int32_t c2,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
// D (TMEM) = A (shared memory) * B (shared memory) [+ D]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// D (TMEM) = A (TMEM) * B (shared memory) [+ D]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// 16 columns of this warp's 32 lanes, a row per thread: the load is under way until
// tmem_ready, which takes the registers so that nothing reads them before it.
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ready(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::
                     "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
        : "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle, 8-row atoms of 1024 bytes.
// K-major (queries, keys: rows of 64 channels): the next 8 rows 1024 bytes on.
// MN-major (values: N = channels contiguous, K = keys): 8 keys 1024 bytes on, the next 64
// channels one block on.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo) {
    uint64_t d = static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>(lbo >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;  // descriptor version of sm_100
    d |= static_cast<uint64_t>(2u) << 61;  // SWIZZLE_128B
    return d;
}
// kind::f16: fp16 operands, fp32 sums, M = 128, N = n; B K-major or MN-major.
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// Byte offset of 16-byte chunk c (of all the row's channels) of row r.
__device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) {
    return (c >> 3) * kBlock + r * 128u + (((c & 7u) ^ (r & 7u)) << 4);
}

template <uint32_t HD>
__device__ __forceinline__ void attention_tc(const TcMaps& maps, const AttnArgs& a, uint32_t box_shift) {
    using T = Tc<HD>;
    extern __shared__ uint8_t sm_raw[];
    __shared__ uint32_t row_tok[kRows], row_head[kRows];
    __shared__ int row_pos[kRows];
    __shared__ float row_unscale[kRows], tile_max[4][kRows], sum_l[4][kRows], sum_m[2][kRows];
    __shared__ uint64_t full[kSlots], empty[kSlots], cut, s_full[2], p_full[2], o_full[2], done;
    __shared__ uint32_t found[2], tmem_slot, gaps[4];
    const uint32_t s0 = (smem_addr(sm_raw) + 1023u) & ~1023u;
    uint8_t* const sm = sm_raw + (s0 - smem_addr(sm_raw));
    const uint32_t q_addr = s0, ring = s0 + 2u * T::kTile;
    const uint32_t hd = a.kv.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t kh = blockIdx.x % a.kv.kv_heads;
    uint32_t rest = blockIdx.x / a.kv.kv_heads;
    const uint32_t c = rest % a.chunks;
    rest /= a.chunks;

    // what follows on the stream may come up where there is room (it waits for this kernel)
    if (tid == 0u) asm volatile("griddepcontrol.launch_dependents;");
    // ---- the item: rows and keys
    uint32_t s = 0, r0 = 0, nrows, t0 = 0;
    PagedSeq sq{0u, 0u, 0u};
    if (a.part == kPartPrefix) {
        r0 = rest * kRows;
        nrows = min(kRows, a.b.tokens * a.group - r0);
    } else {
        // the last tiles first: with causal rows they have the most keys
        if (warp == 0) {
            uint32_t tile;
            const uint32_t seq = find_tile(a, a.tiles - 1u - rest, kRows, &tile);
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
    uint32_t kb = kNone, ke = 0;
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
        uint32_t base = 0;
        if (a.part == kPartOwn) base = own_begin(sq, a.window, a.shared_len);
        else ke = min(ke, a.shared_len);
        const uint64_t cb = static_cast<uint64_t>(base) + static_cast<uint64_t>(c) * a.chunk;
        kb = cb > kb ? static_cast<uint32_t>(cb < kNone ? cb : kNone) : max(kb, base);
        if (cb + a.chunk < ke) ke = static_cast<uint32_t>(cb + a.chunk);
        if (kb >= ke && !a.direct) return;  // no row of the tile sees a key of this chunk
    }
    const uint32_t j0 = kb & ~(kKeys - 1u), ntiles = kb < ke ? (ke - j0 + kKeys - 1u) / kKeys : 0u;

    // ---- barriers, TMEM, queries
    if (tid == 0u) {
        for (uint32_t i = 0; i < kSlots; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(&cut, 1);
        for (uint32_t i = 0; i < 2u; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 256);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(&done, 1);
        fence_barrier_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid < 256u) {  // a row per two threads: scaled, split, stored
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
            *reinterpret_cast<uint4*>(sm + T::kTile + at(r, d >> 3)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    // Ring order: K0, K1, V0, K2, V1, ..., V(last): the order in which the MMAs use them.
    auto k_at = [&](uint32_t i) { return i == 0u ? 0u : 2u * i - 1u; };
    auto v_at = [&](uint32_t i) { return i + 1u < ntiles ? 2u * i + 2u : 2u * ntiles - 1u; };

    if (warp >= kLoadWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == kLoadWarp) {
            // ---- loads
            const uint32_t box_rows = 1u << box_shift, boxes = kKeys >> box_shift, box_bytes = box_rows * 128u;
            // lane b: page of box b of a tile (kNone: no keys of the item there, or no page)
            auto look_up = [&](uint32_t i) {
                const uint32_t j = j0 + i * kKeys + lane * box_rows;
                return lane < boxes && i < ntiles && j < ke && j + box_rows > kb
                           ? load_page(a.b, a.kv, s, j >> a.kv.page_shift, a.st)
                           : kNone;
            };
            bool ok = true;
            uint32_t issued = 0, cuts = 0;
            auto load = [&](uint32_t n, uint32_t i, uint32_t pages, bool values) {
                const uint32_t slot = n % kSlots, dst = ring + slot * T::kTile;
                if (ok && n >= kSlots) ok = mbar_wait_bounded(&empty[slot], ((n / kSlots) - 1u) & 1u, a.st, 61u);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) return;
                const uint32_t j = j0 + i * kKeys, there = __ballot_sync(0xFFFFFFFFu, pages != kNone);
                const uint32_t want = __ballot_sync(
                    0xFFFFFFFFu, lane < boxes && j + lane * box_rows < ke && j + (lane + 1u) * box_rows > kb);
                const bool whole = there == (1u << boxes) - 1u && j >= kb && j + kKeys <= ke;
                const bool patch = values && !whole;
                uint64_t* bar = patch ? &cut : &full[slot];
                if (lane == 0u) {
                    if (!values) gaps[i & 3u] = want & ~there;
                    const uint32_t bytes = __popc(there) * T::kBlocks * box_bytes;
                    if (bytes != 0u) mbar_arrive_expect_tx(bar, bytes);
                    else mbar_arrive(bar);
                }
                __syncwarp();
                if (pages != kNone) {
                    const int32_t slot_row = static_cast<int32_t>((j + lane * box_rows) & (a.kv.page_size - 1u));
                    const int32_t head = static_cast<int32_t>(pages * a.kv.kv_heads + kh);
#pragma unroll
                    for (uint32_t b = 0; b < T::kBlocks; ++b)
                        tma_load_3d(dst + b * kBlock + lane * box_bytes, values ? &maps.v : &maps.k,
                                    static_cast<int32_t>(64u * b), slot_row, head, bar);
                }
                if (patch) {
                    // values outside the item's keys count as zero
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&cut, cuts & 1u, a.st, 62u));
                    ++cuts;
                    if (!ok) return;
                    for (uint32_t x = lane; x < kKeys * 8u * T::kBlocks; x += 32u) {
                        const uint32_t r = x / (8u * T::kBlocks), ch = x % (8u * T::kBlocks);
                        if (j + r < kb || j + r >= ke || !(there >> (r >> box_shift) & 1u))
                            *reinterpret_cast<uint4*>(sm + (dst - s0) + at(r, ch)) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(&full[slot]);
                }
                issued = n + 1u;
            };
            uint32_t before = kNone, now = look_up(0), next = look_up(1);
            for (uint32_t i = 0; i < ntiles && ok; ++i) {
                const uint32_t after = look_up(i + 2u);
                load(k_at(i), i, now, false);
                if (i > 0u && ok) load(v_at(i - 1u), i - 1u, before, true);
                before = now;
                now = next;
                next = after;
            }
            if (ntiles != 0u && ok) load(v_at(ntiles - 1u), ntiles - 1u, before, true);
            // the last copies into every slot have landed before the CTA ends
            for (uint32_t n = issued > kSlots ? issued - kSlots : 0u; n < issued; ++n)
                mbar_wait_bounded(&full[n % kSlots], (n / kSlots) & 1u, a.st, 63u);
        } else if (warp == kMmaWarp) {
            if (lane == 0u) {
                // ---- MMAs
                bool ok = true;
                constexpr uint32_t kS = idesc(kKeys, false), kO = idesc(HD, true);
                auto qk = [&](uint32_t i) {
                    const uint32_t n = k_at(i), slot = n % kSlots;
                    ok = mbar_wait_bounded(&full[slot], (n / kSlots) & 1u, a.st, 64u);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t d = tmem + (i & 1u) * 128u;
#pragma unroll
                    for (uint32_t half = 0; half < 2u; ++half)  // low halves first
#pragma unroll
                        for (uint32_t k = 0; k < HD / 16u; ++k) {
                            const uint32_t off = (k >> 2) * kBlock + (k & 3u) * 32u;
                            mma_ss(d, desc(q_addr + (half ? 0u : T::kTile) + off, 16u), desc(ring + slot * T::kTile + off, 16u),
                                   kS, half + k != 0u);
                        }
                    tc_commit(&s_full[i & 1u]);
                    tc_commit(&empty[slot]);
                };
                if (ntiles != 0u) qk(0);
                for (uint32_t i = 0; i < ntiles && ok; ++i) {
                    if (i + 1u < ntiles) qk(i + 1u);
                    const uint32_t n = v_at(i), slot = n % kSlots;
                    ok = ok && mbar_wait_bounded(&full[slot], (n / kSlots) & 1u, a.st, 65u);
                    ok = ok && mbar_wait_bounded(&p_full[i & 1u], (i >> 1) & 1u, a.st, 66u);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem + 256u + (i & 1u) * 128u, p = tmem + (i & 1u) * 128u;
#pragma unroll
                    for (uint32_t half = 0; half < 2u; ++half)
#pragma unroll
                        for (uint32_t k = 0; k < kKeys / 16u; ++k)  // 16 keys: 8 + 8 columns of weights, 2048 bytes of values
                            mma_ts(d, p + k * 16u + (half ? 0u : 8u),
                                   desc(ring + slot * T::kTile + k * 2048u, kBlock), kO, half + k != 0u);
                    tc_commit(&o_full[i & 1u]);
                    tc_commit(&empty[slot]);
                }
                tc_commit(&done);  // every MMA issued above has completed when this arrives
                mbar_wait_bounded(&done, 0u, a.st, 67u);
            }
            __syncwarp();
        }
    } else {
        // ---- softmax: tiles half, half + 2, ...; keys and channels of this side
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const uint32_t half = warp >> 3, side = (warp >> 2) & 1u, r = tid & 127u;
        constexpr uint32_t kD = HD / 2u, kC = kKeys / 32u;  // channels and 16-key pieces of a side
        const uint32_t lanes = tmem + ((warp & 3u) << 21);  // the warp's 32 TMEM lanes
        const uint32_t st_addr = lanes + half * 128u + side * 64u, o_addr = lanes + 256u + half * 128u + side * kD;
        const int p = row_pos[r];
        const float unscale = row_unscale[r];
        const uint32_t lo_key = p >= 0 ? first_key(p, a.window) : kNone, hi_key = p >= 0 ? static_cast<uint32_t>(p) + 1u : 0u;
        // keys that some / every row of the warp sees
        const uint32_t wb = __reduce_min_sync(0xFFFFFFFFu, lo_key), we = __reduce_max_sync(0xFFFFFFFFu, hi_key);
        const uint32_t all_b = __reduce_max_sync(0xFFFFFFFFu, p >= 0 ? lo_key : 0u);
        const uint32_t all_e = __reduce_min_sync(0xFFFFFFFFu, p >= 0 ? hi_key : kNone);
        float acc[kD];
#pragma unroll
        for (uint32_t d = 0; d < kD; ++d) acc[d] = 0.f;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (uint32_t i = half; i < ntiles && ok; i += 2u) {
            const uint32_t ph = (i >> 1) & 1u, j = j0 + i * kKeys;
            ok = mbar_wait_bounded(&s_full[half], ph, a.st, 68u);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            const bool mine = j < we && j + kKeys > wb;  // a tile that none of the warp's rows sees is passed over
            float alpha = 1.f, ref = 0.f;
            bool whole = true;
            uint32_t gap = 0u;
            // keys of the tile that this row sees: bits of 16 keys from key 16 k on
            const uint32_t from = max(max(lo_key, kb), j) - j, to = min(min(hi_key, ke), j + kKeys) - min(j, min(hi_key, ke));
            auto seen = [&](uint32_t k) -> uint32_t {
                const uint32_t b = min(max(from, 16u * k) - 16u * k, 16u), e = min(max(to, 16u * k) - 16u * k, 16u);
                return gap >> ((16u * k) >> box_shift) & 1u ? 0u : (0xFFFFu << b) & ((1u << e) - 1u);
            };
            auto mask = [&](uint32_t (&x)[16], uint32_t k) {
                const uint32_t bits = seen(kC * side + k);
#pragma unroll
                for (uint32_t e = 0; e < 16u; ++e)
                    if (!(bits >> e & 1u)) x[e] = 0xFF800000u;
            };
            if (mine) {
                gap = *reinterpret_cast<volatile uint32_t*>(&gaps[i & 3u]);
                whole = gap == 0u && j >= max(all_b, kb) && j + kKeys <= min(all_e, ke);
                float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
                for (uint32_t k = 0; k < kC; k += 2u) {
                    uint32_t x[2][16];
                    tmem_load(st_addr + 16u * k, x[0]);
                    tmem_load(st_addr + 16u * (k + 1u), x[1]);
                    tmem_ready(x[0]);
                    tmem_ready(x[1]);
#pragma unroll
                    for (uint32_t u = 0; u < 2u; ++u) {
                        if (!whole) mask(x[u], k + u);
#pragma unroll
                        for (uint32_t e = 0; e < 16u; e += 2u)
                            mt[(e >> 1) & 1u] =
                                fmaxf(fmaxf(mt[(e >> 1) & 1u], __uint_as_float(x[u][e])), __uint_as_float(x[u][e + 1]));
                    }
                }
                tile_max[half * 2u + side][r] = fmaxf(mt[0], mt[1]);
            }
            named_barrier_sync(1u + half, 256);
            if (mine) {
                const float mt = fmaxf(tile_max[half * 2u][r], tile_max[half * 2u + 1u][r]);
                const float mn = fmaxf(m, mt * unscale);
                alpha = mn == -INFINITY ? 1.f : exp2_fast(m - mn);
                m = mn;
                ref = (mn == -INFINITY ? 0.f : mn) - kUp;
                float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 unscale2 = make_float2(unscale, unscale), ref2 = make_float2(-ref, -ref);
#pragma unroll 1
                for (uint32_t k = 0; k < kC; ++k) {
                    uint32_t x[16], w[16];  // w: 8 columns of high halves, 8 of low halves
                    tmem_load(st_addr + 16u * k, x);
                    tmem_ready(x);
                    if (!whole) mask(x, k);
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) {
                        float2 v = ffma2(make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), unscale2, ref2);
                        v = make_float2(exp2_fast(v.x), exp2_fast(v.y));
                        part[e & 1u] = fadd2(part[e & 1u], v);
                        split(v, &w[e], &w[8 + e]);
                    }
                    tmem_store(st_addr + 16u * k, w);
                }
                l = fmaf(l, alpha, (part[0].x + part[1].x) + (part[0].y + part[1].y));
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            tc_fence_before();
            mbar_arrive(&p_full[half]);
            ok = mbar_wait_bounded(&o_full[half], ph, a.st, 70u);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            if (mine) {
                bool odd = false;
                uint32_t x[2][16];
                if (!whole) {
                    // a value that is not finite must not reach the rows that do not see it, yet
                    // 0 * inf is in their sums: then the tile is done key by key
                    float t = 0.f;
                    tmem_load(o_addr, x[0]);
#pragma unroll
                    for (uint32_t k = 0; k < kD / 16u; ++k) {
                        tmem_ready(x[k & 1u]);
                        if (k + 1u < kD / 16u) tmem_load(o_addr + 16u * (k + 1u), x[(k + 1u) & 1u]);
#pragma unroll
                        for (uint32_t e = 0; e < 16u; ++e) t = fmaf(__uint_as_float(x[k & 1u][e]), 0.f, t);
                    }
                    odd = p >= 0 && t != 0.f;
                }
                if (!__any_sync(0xFFFFFFFFu, odd)) {
                    tmem_load(o_addr, x[0]);
#pragma unroll
                    for (uint32_t k = 0; k < kD / 16u; ++k) {
                        tmem_ready(x[k & 1u]);
                        if (k + 1u < kD / 16u) tmem_load(o_addr + 16u * (k + 1u), x[(k + 1u) & 1u]);
#pragma unroll
                        for (uint32_t e = 0; e < 16u; e += 2u) {
                            const float2 y = ffma2(make_float2(acc[16u * k + e], acc[16u * k + e + 1u]), make_float2(alpha, alpha),
                                                   make_float2(__uint_as_float(x[k & 1u][e]), __uint_as_float(x[k & 1u][e + 1u])));
                            acc[16u * k + e] = y.x;
                            acc[16u * k + e + 1u] = y.y;
                        }
                    }
                } else {
#pragma unroll
                    for (uint32_t d = 0; d < kD; ++d) acc[d] *= alpha;
                    const float* q = a.q + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd;
                    for (uint32_t k = from; k < to; ++k) {
                        if (!(seen(k >> 4) >> (k & 15u) & 1u)) continue;
                        const uint32_t page = a.b.table[static_cast<size_t>(s) * a.b.max_pages + ((j + k) >> a.kv.page_shift)];
                        const size_t off = ((static_cast<size_t>(page) * a.kv.kv_heads + kh) * a.kv.page_size +
                                            ((j + k) & (a.kv.page_size - 1u))) * hd;
                        const __half *kr = static_cast<const __half*>(a.kv.k) + off, *vr = static_cast<const __half*>(a.kv.v) + off;
                        float sum = 0.f;
                        for (uint32_t d = 0; d < hd; ++d) sum = fmaf(q[d] * a.scale_log2, __half2float(kr[d]), sum);
                        const float w = exp2_fast(sum - ref);
#pragma unroll
                        for (uint32_t d = 0; d < kD; ++d)
                            if (side * kD + d < hd) acc[d] = fmaf(w, __half2float(vr[side * kD + d]), acc[d]);
                    }
                    __syncwarp();
                }
            }
        }
        // the halves meet: the odd tiles' sums through shared memory (the ring is done with)
        constexpr uint32_t kPitch = HD + 4u;
        float* sums = reinterpret_cast<float*>(sm + (ring - s0)) + r * kPitch + side * kD;
        sum_l[half * 2u + side][r] = p >= 0 ? l : 0.f;  // padding sees nothing
        if (side == 0u) sum_m[half][r] = m == -INFINITY ? 0.f : m;
        named_barrier_sync(3, kSoftmax);
        if (half == 1u) {
#pragma unroll
            for (uint32_t d = 0; d < kD; d += 4u)
                *reinterpret_cast<float4*>(sums + d) = make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
        }
        named_barrier_sync(3, kSoftmax);
        const float l0 = sum_l[0][r] + sum_l[1][r], l1 = sum_l[2][r] + sum_l[3][r];
        const float top = l0 == 0.f ? sum_m[1][r] : l1 == 0.f ? sum_m[0][r] : fmaxf(sum_m[0][r], sum_m[1][r]);
        const float f0 = l0 == 0.f ? 0.f : exp2_fast(sum_m[0][r] - top), f1 = l1 == 0.f ? 0.f : exp2_fast(sum_m[1][r] - top);
        const float sum = l0 * f0 + l1 * f1;
        if (half == 0u) {
            const float scale = a.direct && sum != 0.f ? 1.f / sum : 1.f;
#pragma unroll
            for (uint32_t d = 0; d < kD; d += 4u) {
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (l1 != 0.f) x = *reinterpret_cast<const float4*>(sums + d);
                if (l1 != 0.f) x = make_float4(x.x * f1, x.y * f1, x.z * f1, x.w * f1);
                if (l0 != 0.f)
                    x = make_float4(fmaf(acc[d], f0, x.x), fmaf(acc[d + 1], f0, x.y), fmaf(acc[d + 2], f0, x.z),
                                    fmaf(acc[d + 3], f0, x.w));
                *reinterpret_cast<float4*>(sums + d) = make_float4(x.x * scale, x.y * scale, x.z * scale, x.w * scale);
            }
        }
        const size_t rows_all = static_cast<size_t>(a.b.tokens) * a.heads;
        if (ok && half == 0u && side == 0u && !a.direct && p != -2)
            a.part_ml[(a.slot0 + c) * rows_all + static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]] =
                make_float2(top - kUp, sum);
        named_barrier_sync(3, kSoftmax);
        if (ok) {
            const float* all = reinterpret_cast<const float*>(sm + (ring - s0));
            const uint32_t hd4 = hd / 4u;
            for (uint32_t x = tid; x < kRows * hd4; x += kSoftmax) {
                const uint32_t rr = x / hd4, d = (x - rr * hd4) * 4u;
                if (row_pos[rr] == -2) continue;
                const size_t row = static_cast<size_t>(row_tok[rr]) * a.heads + row_head[rr];
                float* o = a.direct ? a.out + row * hd : a.part_o + ((a.slot0 + c) * rows_all + row) * hd;
                *reinterpret_cast<float4*>(o + d) = *reinterpret_cast<const float4*>(all + rr * kPitch + d);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

template <uint32_t HD>
__global__ void __launch_bounds__(kThreads, 1)
    attention_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ AttnArgs a, uint32_t box_shift) {
    attention_tc<HD>(maps, a, box_shift);
    end_after_previous(a);
}

bool make_map(CUtensorMap* map, void* base, const PagedKv& kv, uint32_t box_rows) {
    EncodeTiled encode = encode_tiled_fn();
    if (!encode) return false;
    const cuuint64_t dims[3] = {kv.head_dim, kv.page_size, static_cast<cuuint64_t>(kv.num_pages) * kv.kv_heads};
    const cuuint64_t strides[2] = {kv.head_dim * 2ull, static_cast<cuuint64_t>(kv.page_size) * kv.head_dim * 2ull};
    const cuuint32_t box[3] = {64u, box_rows, 1u}, step[3] = {1u, 1u, 1u};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <uint32_t HD>
cudaError_t launch(const AttnArgs& a, uint64_t items, cudaStream_t stream) {
    TcMaps maps;
    const uint32_t box_rows = std::min(a.kv.page_size, kKeys);
    if (!make_map(&maps.k, a.kv.k, a.kv, box_rows) || !make_map(&maps.v, a.kv.v, a.kv, box_rows))
        return cudaErrorInvalidValue;
    return launch_items(a, attention_tc_kernel<HD>, items, kThreads, Tc<HD>::kSmem, stream, maps, a,
                        std::min(a.kv.page_shift, 7u));
}

}  // namespace

cudaError_t launch_attention_tc(const AttnArgs& args, uint64_t tiles, cudaStream_t stream) {
    AttnArgs a = args;
    a.tiles = static_cast<uint32_t>(tiles);
    const uint64_t items = tiles * a.kv.kv_heads * a.chunks;
    return a.kv.head_dim <= 64u ? launch<64>(a, items, stream) : launch<128>(a, items, stream);
}

}  // namespace nedo_gpu

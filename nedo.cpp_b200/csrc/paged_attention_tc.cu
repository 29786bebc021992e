// paged_attention_tc.cu -- attention over a paged F16 or Q4_0 cache for tiles of 128 query rows on
// the 5th-generation tensor cores (prompts, the tokens of a whole batch over their shared
// prefix, groups of more than 16 heads), heads of up to 128 channels.
//
// Mathematics.  As in the other tensor-core kernels the fp32 factors are split in two fp16
// halves, low halves first: S = 2^-11 q_lo K^T + q_hi K^T, O = 2^-11 p_lo V + p_hi V, so every
// 128 x 128 tile is 32 MMAs of 128 x 128 x 16; the first with the high halves scales what is there.  The tensor core cuts its fp32 sums instead of rounding
// them, so a tile's O starts from zero in TMEM and is added to the running sums in fp32
// registers, together with the rescaling by 2^(m_old - m_new).
//
// Work.  A CTA (one per SM, 896 threads) takes 128 rows through their keys in tiles of 128:
//   * one warp brings keys and values in by TMA (one 64-channel box per page piece, 128-byte
//     swizzle), in the order of their use, four half-tile slots deep.  Of a tile that the
//     item's key range cuts it zeroes the values outside, whatever the pages hold there;
//   * one warp issues the MMAs: Q K^T three tiles ahead of P V;
//   * warps 0-7 take the even and warps 8-15 the odd tiles, two threads to a row, each with half
//     of the tile's keys: they read S from TMEM, agree on the row's maximum, and write the split
//     weights over S (the A operand of P V);
//   * warps 16-23 add every tile's O to the running sums, two threads to a row, each with half
//     of the channels, rescaling both to the larger of the maxima they go by (the even and the
//     odd tiles keep maxima of their own, so neither half waits for the other).
// TMEM, 512 columns: three S/P tiles and one O tile.  Two of them with the queries' halves in TMEM
// as well (and six ring slots) took 130 us where this took 126.
// Registers: 56 for the softmax, 112 for the sums, 56 for the others.
//
// Q4_0 caches (paged_q4.cuh), 1024 threads.  The load warp brings in the pages' numbers and scales as
// they are, four half tiles deep next to a ring of three: of each page piece one bulk copy and one TMA
// box with the scales of all blocks (a copy for every block's, five in all, held the warp up: 137 us
// for the prompt below).  Two groups of three warps in turn make the fp16 tiles of them, a block of 32
// channels to a lane, where the swizzled copy would have put them, and zeroes outside the item's keys
// (one group: 220 us).  Registers: 56 for the softmax, 96 for the sums, 48 for the others.  The prompt
// below: 124 us; one or two of a scheduler's eight warps make tiles, and its issue slots are taken for
// 62 % of the cycles (52 with F16 caches).
//
// What bounds it: 12 query and 4 KV heads of 128 channels, 2048 and 1840 new tokens of two
// sequences over 4096 and 2550 keys, window 2048: 104 us, 825 TFLOP/s of fp16 MMAs (two for each
// product of the formula).  An item of 17 tiles is 70,000 cycles: 5,000 until its rows and keys
// are known, 4,500 until the queries are in shared memory, 9,500 until the first tile's sums (the
// softmax of both halves at once), then 2,850 a tile, of which the MMAs run 2,050, and 5,000 for
// the results; and 372 items on 148 SMs leave 17 % of the cycles at the end.
#include <algorithm>

#include "paged_attention.cuh"
#include "paged_mma.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kRows = kTcRows;     // 128
constexpr uint32_t kKeys = 128;         // keys per tile
constexpr uint32_t kSoftmax = 512;      // softmax threads: two to a row, for the even and the odd tiles
constexpr uint32_t kSums = 256;         // threads of the running sums: two to a row
constexpr uint32_t kBuffers = 3;        // S/P tiles
constexpr uint32_t kOColumn = kBuffers * 128u;  // TMEM columns of O
constexpr uint32_t kTmem = 0u;          // where an allocation of the whole TMEM lies
constexpr uint32_t kBlock = kRows * 128u;  // bytes of 64 channels of a tile: rows of 128 bytes
constexpr uint32_t kSumWarp = kSoftmax / 32u, kLoadWarp = kSumWarp + kSums / 32u, kMmaWarp = kLoadWarp + 1u;

// Q4_0: half tiles as the pages hold them, and warps that make fp16 tiles of them, in turn by two groups
constexpr uint32_t kRawSlots = 4;
constexpr uint32_t kMakers = 3, kMakerGroups = 2, kFirstMaker = kMmaWarp + 1u;

template <uint32_t HD, bool Q4>
struct Tc {
    static constexpr uint32_t kThreads = kSoftmax + kSums + (Q4 ? 256u : 128u);
    static constexpr uint32_t kSumRegs = Q4 ? 96u : 112u, kOtherRegs = Q4 ? 48u : 56u;
    static constexpr uint32_t kBlocks = HD / 64u;
    static constexpr uint32_t kSlots = Q4 ? 3u : 4u;      // ring slots: the keys or the values of one tile
    static constexpr uint32_t kTile = kBlocks * kBlock;   // a ring slot
    static constexpr uint32_t kRawScales = kKeys * HD / 2u;                   // where a raw slot's scales begin
    static constexpr uint32_t kRaw = kRawScales + 1024u;
    // the queries' high and low halves, the ring
    static constexpr uint32_t kSmem = 2u * kTile + kSlots * kTile + 1024u + (Q4 ? kRawSlots * kRaw : 0u);
};

// [num_pages * kv_heads][page_size][head_dim], boxes of 64 channels x box_rows slots; Q4_0: the scales,
// [num_pages * kv_heads][head_dim / 32][page_size], boxes of all blocks x box_rows slots.
struct TcMaps {
    CUtensorMap k, v;
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
// D (TMEM) = A (TMEM) * B (shared memory, the low word of its descriptor and the high one) [+ D].
// All operands are the same in the whole warp, so that they live in uniform registers: built
// per lane, each MMA took some 110 cycles to issue, of which it runs 64.
// SCALE: [+ 2^-SCALE D].
template <uint32_t HIGH, uint32_t IDESC, uint32_t SCALE>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_low, bool add) {
    if constexpr (SCALE == 0u)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b_low), "n"(HIGH), "n"(IDESC), "r"(static_cast<uint32_t>(add))
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p, %6;\n\t}" ::"r"(d),
            "r"(a), "r"(b_low), "n"(HIGH), "n"(IDESC), "r"(static_cast<uint32_t>(add)), "n"(SCALE)
            : "memory");
}
template <uint32_t HIGH, uint32_t IDESC, uint32_t SCALE>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, bool add) {
    if constexpr (SCALE == 0u)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
            "r"(a_low), "r"(b_low), "n"(HIGH), "n"(IDESC), "r"(static_cast<uint32_t>(add))
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p, %6;\n\t}" ::"r"(d),
            "r"(a_low), "r"(b_low), "n"(HIGH), "n"(IDESC), "r"(static_cast<uint32_t>(add)), "n"(SCALE)
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
// K-major (keys: rows of 64 channels): the next 8 rows 1024 bytes on.
// MN-major (values: N = channels contiguous, K = keys): 8 keys 1024 bytes on, the next 64
// channels one block on.
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3FFFu) | (lbo >> 4) << 16; }
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;  // stride, sm_100's version, SWIZZLE_128B
// kind::f16: fp16 operands, fp32 sums, M = 128, N = n; B K-major or MN-major.
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// Whether a phase is complete, without waiting.  A look at a barrier takes some 330 cycles here
// (it queues behind the softmax warps' exponentials), so the warp that issues the MMAs looks at
// all that it needs at once and waits only for what is not there.
__device__ __forceinline__ uint32_t is_complete(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return ok;
}
// True in one lane of the (whole) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0u;
}
// One arrival, and one waiting thread, for a whole warp: 32 of them on one barrier are taken one
// after the other (256 arrivals came to some 700 cycles of every tile).
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31u) == 0u) mbar_arrive(bar);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, DeviceStatus* st, uint32_t site) {
    return __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bar, parity, st, site));
}

// Byte offset of 16-byte chunk c (of all the row's channels) of row r.
__device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) {
    return (c >> 3) * kBlock + r * 128u + (((c & 7u) ^ (r & 7u)) << 4);
}

// A run of 16-byte pieces into shared memory, counted by `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}

template <uint32_t HD, bool Q4>
__device__ __forceinline__ void attention_tc(const TcMaps& maps, const AttnArgs& a, uint32_t box_shift) {
    using T = Tc<HD, Q4>;
    constexpr uint32_t kSlots = T::kSlots;
    extern __shared__ uint8_t sm_raw[];
    __shared__ uint32_t row_tok[kRows], row_head[kRows];
    __shared__ int row_pos[kRows];
    __shared__ float row_unscale[kRows], side_max[2][4][kRows], tile_ref[2 * kBuffers][kRows], sum_l[4][kRows], sum_m[2][kRows];
    __shared__ uint64_t full[T::kSlots], empty[T::kSlots], cut, s_full[kBuffers], p_full[kBuffers], o_full, o_empty, q_full, done;
    __shared__ uint32_t found[2], tmem_slot, gaps[8], again[kRows / 32u];
    __shared__ uint64_t raw_full[kRawSlots], raw_empty[kRawSlots];  // Q4_0
    __shared__ uint32_t raw_there[kRawSlots];
    const uint32_t s0 = (smem_addr(sm_raw) + 1023u) & ~1023u;
    uint8_t* const sm = sm_raw + (s0 - smem_addr(sm_raw));
    const uint32_t ring = s0 + 2u * T::kTile;
    const uint32_t hd = a.kv.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t kh = blockIdx.x % a.kv.kv_heads;
    uint32_t rest = blockIdx.x / a.kv.kv_heads;
    const uint32_t c = rest % a.chunks;
    rest /= a.chunks;

    // what follows on the stream may come up where there is room (it waits for this kernel)
    if (tid == 0u) asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 32u * kLoadWarp) {
        for (uint32_t i = 0; i < kSlots; ++i) {
            mbar_init(&full[i], Q4 ? kMakers : 1u);
            mbar_init(&empty[i], 1);
        }
        if constexpr (Q4)
            for (uint32_t i = 0; i < kRawSlots; ++i) {
                mbar_init(&raw_full[i], 1);
                mbar_init(&raw_empty[i], kMakers);
            }
        mbar_init(&cut, 1);
        for (uint32_t i = 0; i < kRows / 32u; ++i) again[i] = 0u;
        for (uint32_t i = 0; i < kBuffers; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 8);
        }
        mbar_init(&o_full, 1);
        mbar_init(&o_empty, kSums / 32u);
        mbar_init(&q_full, kSoftmax / 32u);
        mbar_init(&done, 1);
        fence_barrier_init();
    }
    // ---- the item: rows and keys
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
    uint32_t kb = kNone, ke = 0;
    {
        if (a.part == kPartOwn) {
            // the rows' positions ascend
            const int p0 = sq.pos(r0 / a.group), p1 = sq.pos((r0 + nrows - 1u) / a.group);
            if (p1 >= 0) {
                kb = first_key(max(p0, 0), a.window);
                ke = static_cast<uint32_t>(p1) + 1u;
            }
        } else {
            __syncthreads();
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
        }
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
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    const uint32_t box_rows = 1u << box_shift, boxes = kKeys >> box_shift, box_bytes = box_rows * 128u;
    // lane b: page of box b of a tile (kNone: no keys of the item there, or no page), looked up
    // and, when it is needed, checked; those of the first tiles before the rest is ready
    auto wanted = [&](uint32_t i) {
        const uint32_t j = j0 + i * kKeys + lane * box_rows;
        return lane < boxes && i < ntiles && j < ke && j + box_rows > kb;
    };
    auto look_up = [&](uint32_t i) {
        return wanted(i) ? a.b.table[static_cast<size_t>(s) * a.b.max_pages + ((j0 + i * kKeys + lane * box_rows) >> a.kv.page_shift)] : kNone;
    };
    auto checked = [&](uint32_t i, uint32_t page) {
        if (page < a.kv.num_pages) return page;
        if (wanted(i)) flag_argument(a.st);
        return kNone;
    };
    uint32_t page0 = kNone, page1 = kNone;
    if (warp == kLoadWarp) {
        page0 = look_up(0);
        page1 = look_up(1);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // all 512 columns: they begin at 0
    constexpr uint32_t tmem = kTmem;

    // Ring order: K0, K1, K2, V0, K3, V1, ..., V(last): the order in which the MMAs use them.
    auto k_at = [&](uint32_t i) { return i + (i >= kBuffers ? i - kBuffers + 1u : 0u); };
    auto v_at = [&](uint32_t i) { return i + min(ntiles, i + kBuffers); };

    // Q4_0: half tile n of the ring's order -- the keys of the first tiles, then values and keys in turn,
    // values at the end.
    auto tile_at = [&](uint32_t n, bool* values) -> uint32_t {
        const uint32_t lead = min(kBuffers, ntiles);
        if (n < lead) return *values = false, n;
        const uint32_t x = n - lead, pairs = 2u * (ntiles - lead);
        *values = x >= pairs || (x & 1u) == 0u;
        return x >= pairs ? x - pairs + (ntiles - lead) : (x & 1u) == 0u ? x >> 1 : lead + (x >> 1);
    };
    const uint32_t raw = ring + kSlots * T::kTile, blocks = hd >> 5, halves = 2u * ntiles;
    const uint32_t scale_pitch = max(128u, HD / 32u * box_rows * 2u);  // a box's scales, [block][key]
    auto send_raw = [&]() {  // one warp
        const uint32_t head_bytes = q4_head_bytes(a.kv);
        uint32_t sent = 0, next = page0;
        bool ok = true;
        for (uint32_t n = 0; n < halves; ++n) {
            bool values, v;
            const uint32_t i = tile_at(n, &values), rs = n % kRawSlots, j = j0 + i * kKeys, pages = checked(i, next);
            next = n + 1u < halves ? look_up(tile_at(n + 1u, &v)) : kNone;
            if (n >= kRawSlots) ok = warp_wait(&raw_empty[rs], ((n / kRawSlots) - 1u) & 1u, a.st, 73u);
            if (!ok) break;
            const uint32_t there = __ballot_sync(0xFFFFFFFFu, pages != kNone), want = __ballot_sync(0xFFFFFFFFu, wanted(i));
            if (lane == 0u) {
                if (!values) gaps[i & 7u] = want & ~there;
                raw_there[rs] = there;
                const uint32_t bytes = __popc(there) * box_rows * (hd / 2u + blocks * 2u);
                if (bytes != 0u) mbar_arrive_expect_tx(&raw_full[rs], bytes);
                else mbar_arrive(&raw_full[rs]);
            }
            __syncwarp();
            if (pages != kNone) {
                const uint32_t slot_row = (j + lane * box_rows) & (a.kv.page_size - 1u), head = pages * a.kv.kv_heads + kh;
                const uint32_t dst = raw + rs * T::kRaw;
                bulk_load(dst + lane * box_rows * (hd / 2u),
                          static_cast<const uint8_t*>(values ? a.kv.v : a.kv.k) + static_cast<size_t>(head) * head_bytes + slot_row * (hd / 2u),
                          box_rows * (hd / 2u), &raw_full[rs]);
                tma_load_3d(dst + T::kRawScales + lane * scale_pitch, values ? &maps.v : &maps.k, static_cast<int32_t>(slot_row), 0,
                            static_cast<int32_t>(head), &raw_full[rs]);
            }
            sent = n + 1u;
        }
        // the last copies have landed before the CTA ends
        for (uint32_t n = sent > kRawSlots ? sent - kRawSlots : 0u; n < sent; ++n)
            mbar_wait_bounded(&raw_full[n % kRawSlots], (n / kRawSlots) & 1u, a.st, 63u);
    };
    auto make_tiles = [&]() {
        const uint32_t me = (warp - kFirstMaker) % kMakers;
        // a lane: one block of one key of every 32 / kPer; eight neighbouring lanes write to different banks
        constexpr uint32_t kPer = HD / 32u, kUnits = kKeys * kPer / 32u, kStepKeys = 32u / kPer;
        const uint32_t block = HD == 128u ? ((lane >> 2) & 1u) + 2u * (lane >> 4) : (lane >> 2) & 1u;
        const uint32_t key0 = HD == 128u ? (lane & 3u) + 4u * ((lane >> 3) & 1u) : (lane & 3u) + 4u * (lane >> 3);
        for (uint32_t n = (warp - kFirstMaker) / kMakers; n < halves; n += kMakerGroups) {
            bool values;
            const uint32_t i = tile_at(n, &values), slot = n % kSlots, rs = n % kRawSlots, j = j0 + i * kKeys;
            // (looked at together, as by the warp of the MMAs)
            const uint32_t raw_turn = (n / kRawSlots) & 1u, turn = ((n / kSlots) - 1u) & 1u;
            const uint32_t raw_there_now = is_complete(&raw_full[rs], raw_turn), free_now = n < kSlots ? 1u : is_complete(&empty[slot], turn);
            if (!__all_sync(0xFFFFFFFFu, raw_there_now) && !warp_wait(&raw_full[rs], raw_turn, a.st, 74u)) break;
            if (!__all_sync(0xFFFFFFFFu, free_now) && !warp_wait(&empty[slot], turn, a.st, 61u)) break;
            const uint32_t there = *reinterpret_cast<volatile uint32_t*>(&raw_there[rs]);
            const uint8_t* const from = sm + (raw - s0) + rs * T::kRaw;
            uint8_t* const to = sm + (ring - s0) + slot * T::kTile;
            // (the loads of kAtOnce units first: each takes some 300 cycles, behind the softmax's exponentials)
            constexpr uint32_t kAtOnce = 2;
#pragma unroll 1
            for (uint32_t u0 = (me + n) % kMakers; u0 < kUnits; u0 += kAtOnce * kMakers) {
                uint4 w[kAtOnce];
                __half d[kAtOnce];
#pragma unroll
                for (uint32_t v = 0; v < kAtOnce; ++v) {
                    const uint32_t u = u0 + v * kMakers, r = (u < kUnits ? u : u0) * kStepKeys + key0, b = min(block, blocks - 1u);
                    w[v] = *reinterpret_cast<const uint4*>(from + r * (hd / 2u) + b * 16u);
                    d[v] = *reinterpret_cast<const __half*>(from + T::kRawScales + (r >> box_shift) * scale_pitch + (b * box_rows + (r & (box_rows - 1u))) * 2u);
                }
#pragma unroll
                for (uint32_t v = 0; v < kAtOnce; ++v) {
                    const uint32_t u = u0 + v * kMakers;
                    if (u >= kUnits) break;
                    const uint32_t r = u * kStepKeys + key0;
                    const bool in = block < blocks && (there >> (r >> box_shift) & 1u) && j + r >= kb && j + r < ke;
                    const __half2 scale = __half2half2(in ? d[v] : __ushort_as_half(0));
                    const uint32_t words[4] = {w[v].x, w[v].y, w[v].z, w[v].w};
#pragma unroll
                    for (uint32_t x = 0; x < 4u; ++x) {
                        __half2 h[4];
                        q4_pairs(words[x], h);
                        *reinterpret_cast<uint4*>(to + at(r, block * 4u + x)) =
                            make_uint4(pack(__hmul2(h[0], scale)), pack(__hmul2(h[1], scale)), pack(__hmul2(h[2], scale)), pack(__hmul2(h[3], scale)));
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(&raw_empty[rs]);
            warp_arrive(&full[slot]);
        }
    };

    if (warp >= kLoadWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kOtherRegs));
        if (Q4 && warp != kMmaWarp) {
            if constexpr (Q4) {
                if (warp == kLoadWarp) send_raw();
                else make_tiles();
            }
        } else if (warp == kLoadWarp) {
            // ---- loads
            bool ok = true;
            uint32_t issued = 0, cuts = 0;
            auto load = [&](uint32_t n, uint32_t i, uint32_t pages, bool values) {
                const uint32_t slot = n % kSlots, dst = ring + slot * T::kTile;
                if (ok && n >= kSlots) ok = warp_wait(&empty[slot], ((n / kSlots) - 1u) & 1u, a.st, 61u);
                if (!ok) return;
                const uint32_t j = j0 + i * kKeys, there = __ballot_sync(0xFFFFFFFFu, pages != kNone);
                const uint32_t want = __ballot_sync(
                    0xFFFFFFFFu, lane < boxes && j + lane * box_rows < ke && j + (lane + 1u) * box_rows > kb);
                const bool whole = there == (1u << boxes) - 1u && j >= kb && j + kKeys <= ke;
                const bool patch = values && !whole;
                uint64_t* bar = patch ? &cut : &full[slot];
                if (lane == 0u) {
                    if (!values) gaps[i & 7u] = want & ~there;
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
                    ok = warp_wait(&cut, cuts & 1u, a.st, 62u);
                    ++cuts;
                    if (!ok) return;
                    constexpr uint32_t kChunks = 8u * T::kBlocks;  // of 16 bytes in a row
                    auto clear = [&](uint32_t from, uint32_t to) {
#pragma unroll 4
                        for (uint32_t x = from * kChunks + lane; x < to * kChunks; x += 32u)
                            *reinterpret_cast<uint4*>(sm + (dst - s0) + at(x / kChunks, x % kChunks)) = make_uint4(0u, 0u, 0u, 0u);
                    };
                    if (kb > j) clear(0u, kb - j);
                    if (ke < j + kKeys) clear(ke - j, kKeys);
                    for (uint32_t gone = want & ~there; gone != 0u; gone &= gone - 1u) {
                        const uint32_t b = __ffs(gone) - 1u;
                        clear(b * box_rows, (b + 1u) * box_rows);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(&full[slot]);
                }
                issued = n + 1u;
            };
            // pages of the tiles whose keys are in and whose values are not yet
            uint32_t pages[4] = {checked(0, page0), kNone, kNone, kNone}, next = page1;
            for (uint32_t i = 0; i < ntiles + kBuffers - 1u && ok; ++i) {
                const uint32_t after = look_up(i + 2u);
                if (i < ntiles) load(k_at(i), i, pages[0], false);
                if (i >= kBuffers - 1u && ok) load(v_at(i - (kBuffers - 1u)), i - (kBuffers - 1u), pages[kBuffers - 1u], true);
#pragma unroll
                for (uint32_t u = 3; u > 0u; --u) pages[u] = pages[u - 1u];
                pages[0] = checked(i + 1u, next);
                next = after;
            }
            // the last copies into every slot have landed before the CTA ends
            for (uint32_t n = issued > kSlots ? issued - kSlots : 0u; n < issued; ++n)
                mbar_wait_bounded(&full[n % kSlots], (n / kSlots) & 1u, a.st, 63u);
        } else if (warp == kMmaWarp) {
            // ---- MMAs: the whole warp waits, one lane issues
            bool ok = true;
            constexpr uint32_t kS = idesc(kKeys, false), kO = idesc(HD, true);
            uint32_t slot = 0, turn = 0;  // ring slot of the next keys or values, and its phase
            auto advance = [&]() {
                slot = slot + 1u == kSlots ? 0u : slot + 1u;
                turn ^= slot == 0u;
            };
            auto qk = [&](uint32_t buf, bool there) {
                if (!there) ok = warp_wait(&full[slot], turn, a.st, 64u);
                if (!ok) return;
                tc_fence_after();
                const uint32_t d = kTmem + buf * 128u, k0 = desc_low(ring + slot * T::kTile, 16u), q0 = desc_low(s0, 16u);
                if (elect_one()) {
                    // low halves first, taken down by the first product with the high ones
                    auto at_k = [](uint32_t k) { return ((k >> 2) * kBlock + (k & 3u) * 32u) >> 4; };
#pragma unroll
                    for (uint32_t k = 0; k < HD / 16u; ++k)
                        mma_ss<kDescHigh, kS, 0u>(d, q0 + (T::kTile >> 4) + at_k(k), k0 + at_k(k), k != 0u);
                    mma_ss<kDescHigh, kS, kLowBits>(d, q0, k0, true);
#pragma unroll
                    for (uint32_t k = 1; k < HD / 16u; ++k) mma_ss<kDescHigh, kS, 0u>(d, q0 + at_k(k), k0 + at_k(k), true);
                    tc_commit(&s_full[buf]);
                    tc_commit(&empty[slot]);
                }
                __syncwarp();
                advance();
            };
            if (ntiles != 0u) ok = warp_wait(&q_full, 0u, a.st, 71u);
            for (uint32_t i = 0; i < kBuffers && i < ntiles && ok; ++i) qk(i, false);
            for (uint32_t i = 0; i < ntiles && ok; ++i) {
                const uint32_t buf = i % kBuffers, p_turn = (i / kBuffers) & 1u;
                // the values, the weights, the sums' leave to write O, and the next keys
                const uint32_t slot1 = slot + 1u == kSlots ? 0u : slot + 1u;
                const uint32_t v_there = is_complete(&full[slot], turn), p_there = is_complete(&p_full[buf], p_turn);
                const uint32_t o_there = i == 0u ? 1u : is_complete(&o_empty, (i - 1u) & 1u);
                const uint32_t k_there = is_complete(&full[slot1], turn ^ (slot1 == 0u));
                const bool k_now = __all_sync(0xFFFFFFFFu, k_there);
                ok = (__all_sync(0xFFFFFFFFu, v_there) || warp_wait(&full[slot], turn, a.st, 65u)) &&
                     (__all_sync(0xFFFFFFFFu, p_there) || warp_wait(&p_full[buf], p_turn, a.st, 66u)) &&
                     (__all_sync(0xFFFFFFFFu, o_there) || warp_wait(&o_empty, (i - 1u) & 1u, a.st, 72u));
                if (!ok) break;
                tc_fence_after();
                const uint32_t p = kTmem + buf * 128u, v0 = desc_low(ring + slot * T::kTile, kBlock);
                if (elect_one()) {
                    // 16 keys: 8 + 8 columns of weights, 2048 bytes of values
#pragma unroll
                    for (uint32_t k = 0; k < kKeys / 16u; ++k)
                        mma_ts<kDescHigh, kO, 0u>(kTmem + kOColumn, p + k * 16u + 8u, v0 + k * (2048u >> 4), k != 0u);
                    mma_ts<kDescHigh, kO, kLowBits>(kTmem + kOColumn, p, v0, true);
#pragma unroll
                    for (uint32_t k = 1; k < kKeys / 16u; ++k)
                        mma_ts<kDescHigh, kO, 0u>(kTmem + kOColumn, p + k * 16u, v0 + k * (2048u >> 4), true);
                    tc_commit(&o_full);
                    tc_commit(&empty[slot]);
                }
                __syncwarp();
                advance();
                if (i + kBuffers < ntiles) qk(buf, k_now);
            }
            if (elect_one()) tc_commit(&done);  // every MMA issued above has completed when this arrives
            __syncwarp();
            warp_wait(&done, 0u, a.st, 67u);
        }
    } else {
        const uint32_t r = tid & 127u, side = (warp >> 2) & 1u;
        const uint32_t lanes = tmem + ((warp & 3u) << 21);  // the warp's 32 TMEM lanes
        const int p = row_pos[r];
        const uint32_t lo_key = p >= 0 ? first_key(p, a.window) : kNone, hi_key = p >= 0 ? static_cast<uint32_t>(p) + 1u : 0u;
        // keys that some / every row of the warp sees
        const uint32_t wb = __reduce_min_sync(0xFFFFFFFFu, lo_key), we = __reduce_max_sync(0xFFFFFFFFu, hi_key);
        const uint32_t all_b = max(kb, __reduce_max_sync(0xFFFFFFFFu, p >= 0 ? lo_key : 0u));
        const uint32_t all_e = min(ke, __reduce_min_sync(0xFFFFFFFFu, p >= 0 ? hi_key : kNone));
        const uint32_t row_b = max(lo_key, kb), row_e = min(hi_key, ke);
        // which of 16 keys from key 16 k of the tile at j on this row sees
        auto seen = [&](uint32_t j, uint32_t gap, uint32_t k) -> uint32_t {
            const uint32_t at = j + 16u * k, b = min(max(row_b, at) - at, 16u), e = min(max(row_e, at) - at, 16u);
            return gap >> ((16u * k) >> box_shift) & 1u ? 0u : (0xFFFFu << b) & ((1u << e) - 1u);
        };
        bool ok = true;
        if (warp < kSumWarp) {
            // ---- softmax: tiles half, half + 2, ...; keys of this side
            asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
            const uint32_t half = warp >> 3;
            constexpr uint32_t kC = kKeys / 32u;  // 16-key pieces of a side
            float unscale;
            {
                // queries: a row by HD / 4 lanes next to each other, scaled, split, stored (with a row
                // per thread each load would be 32 cache lines, 4096 cycles of them in all)
                constexpr uint32_t kLanes = HD / 4u, kAtOnce = 32u / kLanes, kTurns = kRows / (kSoftmax / 32u * kAtOnce);
                const uint32_t ch = lane % kLanes * 4u;
                const uint32_t lanes = kLanes == 32u ? 0xFFFFFFFFu : ((1u << (kLanes & 31u)) - 1u) << (lane & ~(kLanes - 1u));
                auto row_of = [&](uint32_t i) { return (i * (kSoftmax / 32u) + warp) * kAtOnce + lane / kLanes; };
                float4 x[kTurns];
#pragma unroll
                for (uint32_t i = 0; i < kTurns; ++i) {
                    const uint32_t rq = row_of(i);
                    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (row_pos[rq] >= 0 && ch < hd)
                        x[i] = *reinterpret_cast<const float4*>(a.q + (static_cast<size_t>(row_tok[rq]) * a.heads + row_head[rq]) * hd + ch);
                }
#pragma unroll
                for (uint32_t i = 0; i < kTurns; ++i) {
                    const uint32_t rq = row_of(i);
                    float4 v = make_float4(x[i].x * a.scale_log2, x[i].y * a.scale_log2, x[i].z * a.scale_log2, x[i].w * a.scale_log2);
                    // (magnitudes order like their bits)
                    const float big = __uint_as_float(__reduce_max_sync(
                        lanes, __float_as_uint(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))))));
                    const int e2 = up_exponent(big);
                    const float up = power_of_two(e2);
                    if (ch == 0u) row_unscale[rq] = power_of_two(-e2);
                    uint32_t hi[2], lo[2];
                    split(v.x * up, v.y * up, &hi[0], &lo[0]);
                    split(v.z * up, v.w * up, &hi[1], &lo[1]);
                    uint8_t* const to = sm + at(rq, ch >> 3) + (ch & 4u) * 2u;
                    *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(to + T::kTile) = make_uint2(lo[0], lo[1]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                warp_arrive(&q_full);
                named_barrier_sync(3, kSoftmax);
                unscale = row_unscale[r];
            }
            float m = -INFINITY, l = 0.f;
            for (uint32_t i = half; i < ntiles; i += 2u) {
                const uint32_t buf = i % kBuffers, j = j0 + i * kKeys, st_addr = lanes + buf * 128u + side * 64u;
                // (a warp whose wait ran out goes on through the barriers that it shares with others)
                if (ok) ok = warp_wait(&s_full[buf], (i / kBuffers) & 1u, a.st, 68u);
                tc_fence_after();
                const bool mine = j < we && j + kKeys > wb;  // a tile that none of the warp's rows sees is passed over
                const uint32_t gap = *reinterpret_cast<volatile uint32_t*>(&gaps[i & 7u]);
                const bool whole = gap == 0u && j >= all_b && j + kKeys <= all_e;
                auto mask = [&](uint32_t (&x)[16], uint32_t k) {
                    const uint32_t bits = seen(j, gap, kC * side + k);
#pragma unroll
                    for (uint32_t e = 0; e < 16u; ++e)
                        if (!(bits >> e & 1u)) x[e] = 0xFF800000u;
                };
                if (mine) {
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
                    side_max[(i >> 1) & 1u][half * 2u + side][r] = fmaxf(mt[0], mt[1]);
                }
                named_barrier_sync(1u + half, 256);
                if (mine) {
                    // (taken in turns: a quick thread may be a tile ahead of its pair)
                    const float(*both)[kRows] = side_max[(i >> 1) & 1u] + half * 2u;
                    const float mn = fmaxf(m, fmaxf(both[0][r], both[1][r]) * unscale);
                    const float alpha = mn == -INFINITY ? 1.f : exp2_fast(m - mn);
                    m = mn;
                    const float ref = (mn == -INFINITY ? 0.f : mn) - kUp;
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
                // read behind P V: its place is free again once the sums have come three tiles further
                if (side == 0u) tile_ref[i % (2u * kBuffers)][r] = m;
                tc_fence_before();
                warp_arrive(&p_full[buf]);
            }
            sum_l[half * 2u + side][r] = p >= 0 ? l : 0.f;  // padding sees nothing
            if (side == 0u) sum_m[half][r] = m == -INFINITY ? 0.f : m;
            asm volatile("bar.arrive 4, %0;" ::"n"(kSoftmax + kSums) : "memory");
        } else {
            // ---- running sums: channels of this side
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kSumRegs));
            constexpr uint32_t kD = HD / 2u;
            const uint32_t o_addr = lanes + kOColumn + side * kD;
            float acc[kD], top = -INFINITY;
#pragma unroll
            for (uint32_t d = 0; d < kD; ++d) acc[d] = 0.f;
            for (uint32_t i = 0; i < ntiles && ok; ++i) {
                const uint32_t j = j0 + i * kKeys;
                ok = warp_wait(&o_full, i & 1u, a.st, 70u);
                if (!ok) break;
                tc_fence_after();
                if (j < we && j + kKeys > wb) {
                    // the tile's weights go by its half's maximum, the sums by the largest so far
                    const float ref = tile_ref[i % (2u * kBuffers)][r], most = fmaxf(top, ref);
                    const float alpha = most == -INFINITY ? 1.f : exp2_fast(top - most);
                    const float beta = ref == -INFINITY ? 0.f : exp2_fast(ref - most);
                    top = most;
                    const float2 alpha2 = make_float2(alpha, alpha), beta2 = make_float2(beta, beta);
#pragma unroll
                    for (uint32_t k = 0; k < kD / 16u; k += 2u) {
                        uint32_t y[2][16];
                        tmem_load(o_addr + 16u * k, y[0]);
                        tmem_load(o_addr + 16u * (k + 1u), y[1]);
                        tmem_ready(y[0]);
                        tmem_ready(y[1]);
#pragma unroll
                        for (uint32_t e = 0; e < 32u; e += 2u) {
                            const float2 o = make_float2(__uint_as_float(y[e >> 4][e & 15u]), __uint_as_float(y[e >> 4][(e & 15u) + 1u]));
                            const float2 z = ffma2(make_float2(acc[16u * k + e], acc[16u * k + e + 1u]), alpha2, __fmul2_rn(o, beta2));
                            acc[16u * k + e] = z.x;
                            acc[16u * k + e + 1u] = z.y;
                        }
                    }
                }
                tc_fence_before();
                warp_arrive(&o_empty);
            }
            // the weight sums of both halves, then the rows' results through shared memory (the ring
            // is done with)
            asm volatile("bar.sync 4, %0;" ::"n"(kSoftmax + kSums) : "memory");
            constexpr uint32_t kPitch = HD + 4u;
            float* sums = reinterpret_cast<float*>(sm + (ring - s0));
            const float l0 = sum_l[0][r] + sum_l[1][r], l1 = sum_l[2][r] + sum_l[3][r];
            const float ref = top == -INFINITY ? 0.f : top;
            const float sum = (l0 == 0.f ? 0.f : l0 * exp2_fast(sum_m[0][r] - ref)) + (l1 == 0.f ? 0.f : l1 * exp2_fast(sum_m[1][r] - ref));
            const float scale = a.direct ? 1.f / sum : 1.f;
            float odd = sum * 0.f;
#pragma unroll
            for (uint32_t d = 0; d < kD; ++d) odd = fmaf(acc[d], 0.f, odd);
            if (odd != 0.f && p >= 0) atomicOr(&again[r >> 5], 1u << (r & 31u));
#pragma unroll
            for (uint32_t d = 0; d < kD; d += 4u)
                *reinterpret_cast<float4*>(sums + r * kPitch + side * kD + d) =
                    sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                               : make_float4(acc[d] * scale, acc[d + 1] * scale, acc[d + 2] * scale, acc[d + 3] * scale);
            const size_t rows_all = static_cast<size_t>(a.b.tokens) * a.heads;
            if (ok && side == 0u && !a.direct && p != -2)
                a.part_ml[(a.slot0 + c) * rows_all + static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]] =
                    make_float2(ref - kUp, sum);
            named_barrier_sync(5, kSums);
            if ((again[0] | again[1] | again[2] | again[3]) != 0u) {  // rows whose sums are not finite
                // 16 rows to a warp
                const uint32_t first = (warp - kSumWarp) * 16u;
                uint32_t set = ok ? again[first >> 5] >> (first & 31u) & 0xFFFFu : 0u;
                while (set != 0u) {
                    uint32_t n, rows = take_rows(&set, &n);
                    RowSums x;
                    rows_key_by_key<Q4>(a, s, kh, nullptr, {row_tok, row_head, row_pos}, first, rows, kb, ke, 16u, 32u, &x);
                    for (uint32_t u = 0; u < n; ++u, rows >>= 8) {
                        const uint32_t rr = first + (rows & 255u);
                        const float f = !a.direct ? 1.f : x.l[u] == 0.f ? 0.f : 1.f / x.l[u];
                        for (uint32_t i = 0; lane + 32u * i < hd; ++i) sums[rr * kPitch + lane + 32u * i] = x.o[u][i] * f;
                        if (!a.direct && lane == 0u)
                            a.part_ml[(a.slot0 + c) * rows_all + static_cast<size_t>(row_tok[rr]) * a.heads + row_head[rr]] =
                                make_float2(x.m[u], x.l[u]);
                    }
                }
                named_barrier_sync(5, kSums);
            }
            if (ok) {
                // rows by lanes next to each other
                constexpr uint32_t kLanes = HD / 4u, kAtOnce = kSums / kLanes;
                const uint32_t d = (tid - kSoftmax) % kLanes * 4u, row0 = (tid - kSoftmax) / kLanes;
                float* const to = a.direct ? a.out : a.part_o + (a.slot0 + c) * rows_all * hd;
                if (d < hd)
#pragma unroll 8
                    for (uint32_t rr = row0; rr < kRows; rr += kAtOnce)
                        if (row_pos[rr] != -2)
                            *reinterpret_cast<float4*>(to + (static_cast<size_t>(row_tok[rr]) * a.heads + row_head[rr]) * hd + d) =
                                *reinterpret_cast<const float4*>(sums + rr * kPitch + d);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_slot), "r"(512u));
    }
}

template <uint32_t HD, bool Q4>
__global__ void __launch_bounds__(Tc<HD, Q4>::kThreads, 1)
    attention_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ AttnArgs a, uint32_t box_shift) {
    attention_tc<HD, Q4>(maps, a, box_shift);
    end_after_previous(a);
}

bool make_map(CUtensorMap* map, void* base, const PagedKv& kv, uint32_t box_rows) {
    EncodeTiled encode = encode_tiled_fn();
    if (!encode) return false;
    const cuuint64_t heads = static_cast<cuuint64_t>(kv.num_pages) * kv.kv_heads;
    const cuuint32_t step[3] = {1u, 1u, 1u};
    if (kv.type == kQ4_0) {
        const cuuint64_t dims[3] = {kv.page_size, kv.head_dim / 32u, heads}, strides[2] = {kv.page_size * 2ull, q4_head_bytes(kv)};
        const cuuint32_t box[3] = {box_rows, kv.head_dim / 32u, 1u};
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, static_cast<uint8_t*>(base) + q4_scales_at(kv), dims, strides, box, step,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    const cuuint64_t dims[3] = {kv.head_dim, kv.page_size, heads};
    const cuuint64_t strides[2] = {kv.head_dim * 2ull, static_cast<cuuint64_t>(kv.page_size) * kv.head_dim * 2ull};
    const cuuint32_t box[3] = {64u, box_rows, 1u};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <uint32_t HD, bool Q4>
cudaError_t launch(const AttnArgs& a, uint64_t items, cudaStream_t stream) {
    TcMaps maps;
    const uint32_t box_rows = std::min(a.kv.page_size, kKeys);
    if (!make_map(&maps.k, a.kv.k, a.kv, box_rows) || !make_map(&maps.v, a.kv.v, a.kv, box_rows))
        return cudaErrorInvalidValue;
    return launch_items(a, attention_tc_kernel<HD, Q4>, items, Tc<HD, Q4>::kThreads, Tc<HD, Q4>::kSmem, stream, maps, a,
                        std::min(a.kv.page_shift, 7u));
}

}  // namespace

cudaError_t launch_attention_tc(const AttnArgs& a, uint64_t tiles, cudaStream_t stream) {
    const uint64_t items = tiles * a.kv.kv_heads * a.chunks;
    if (a.kv.type == kQ4_0) return a.kv.head_dim <= 64u ? launch<64, true>(a, items, stream) : launch<128, true>(a, items, stream);
    return a.kv.head_dim <= 64u ? launch<64, false>(a, items, stream) : launch<128, false>(a, items, stream);
}

}  // namespace nedo_gpu

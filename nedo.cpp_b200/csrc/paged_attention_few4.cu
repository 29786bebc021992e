// paged_attention_few4.cu -- attention over a paged Q4_0 cache for tiles of up to four, eight or
// sixteen query rows (single tokens with their group of heads, a few drafted tokens, the rows of a
// page list): the shape of decoding, bound by reading the cache and by making fp16 numbers of it.
//
// Mathematics.  As over F16 caches the fp32 factors are split in two fp16 halves, x = hi + 2^-11 lo
// (queries scaled by a power of two per row, weights by 2^14), and a tile's weighted values are
// summed from zero.  Keys and values are the A operands here, S^T = K Q^T and O^T = V^T P^T, made in
// registers from the words that the cache holds: which channel stands in which place of a sum, and in
// which row of a product, is free as long as the other factor, and the result, follow.  So a thread
// takes whole blocks, or the largest part of one, of its keys in one load, with one scale for it, and
// nothing is written in between.  The columns are the rows' halves next to each other, (hi, lo) of four rows in the eight columns of an m16n8k16,
// so a row's score is in one thread, and its weight as the pair (hi, lo) is the operand of P^T after
// one transposing register move.
//
// Work.  A CTA of four warps takes one row tile and one chunk of keys; each warp streams every
// fourth 32-key tile through a ring of its own (cp.async), with its own running maximum and sums,
// so the warps meet only at the end.  The halves of a tile lie within one page each.
//
// What bounds it: 32 single tokens of 12 query and 4 KV heads of 128 channels over 8191 to 32768 keys
// 119 us, 400 MB at 3.4 TB/s (F16 caches: 215 us, 6.6 TB/s).  The instructions: some 440 for a warp's
// 16 keys, the schedulers' slots taken for 69 % of the cycles at four CTAs to an SM; of 121 us the making of
// the keys is 18, that of the values 30, the copies 12 (each left out in a copy of the kernel).  Tiles of 16
// keys, a word to a thread: 167 us.  Five CTAs to an SM, loads of the values ahead of the softmax, sums of
// the halves apart: the same or slower.  16 sequences of five tokens (15 rows) over 2005 to 16001 keys:
// 70 us; 64 tokens over 32 picked pages of 64 keys: 31 us.
#include "paged_attention.cuh"
#include "paged_mma.cuh"
#include "paged_q4.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kKeys = 32;           // keys per tile
constexpr uint32_t kGroups = kKeys / 16;  // each within a page

template <uint32_t HD, uint32_t ROWS>
struct Few4 {
    static constexpr uint32_t kStages = 2;
    static constexpr uint32_t kBlocks = HD / 32u;
    static constexpr uint32_t kRowBytes = HD / 2u;
    static constexpr uint32_t kScales = kKeys * kRowBytes;             // where a tile's scales begin: [group][block][key]
    static constexpr uint32_t kTileBytes = kScales + kBlocks * kKeys * 2u;  // keys or values of one tile
    static constexpr uint32_t kStageBytes = 2u * kTileBytes;
    static constexpr uint32_t kPitch = HD + 4u;
    static constexpr uint32_t kQueries = HD / 16u * (ROWS / 4u) * 32u * 8u;  // [product][four rows][lane]
    static constexpr uint32_t kRing = kWarps * kStages * kStageBytes;
    static constexpr uint32_t kEnd = (kWarps * ROWS * kPitch + ROWS * HD) * 4u;  // the warps' sums, and the chunk's
    static constexpr uint32_t kSmem = kQueries + (kRing > kEnd ? kRing : kEnd);
};

// Byte offsets of 16-byte chunk c (a block's numbers) of key r among a tile's keys and values.  What a
// warp loads at once, chunks t of keys g, or parts g of keys 2 t, falls into different banks.
template <uint32_t HD>
__device__ __forceinline__ uint32_t key_at(uint32_t r, uint32_t c) {
    return r * (HD / 2u) + ((HD == 256u ? c ^ (r & 1u) << 2 : c) << 4);
}
template <uint32_t HD>
__device__ __forceinline__ uint32_t value_at(uint32_t r, uint32_t c) {
    if constexpr (HD == 256u) return r * 128u + ((c ^ (r & 6u)) << 4);
    if constexpr (HD == 128u) return (r >> 1) * 128u + ((((r & 1u) * 4u + c) ^ (r & 6u)) << 4);
    return (r >> 2) * 128u + ((((r & 3u) * 2u + c) ^ ((r & 4u) >> 1)) << 4);
}

// N 32-bit words of shared memory in one load.
template <uint32_t N>
__device__ __forceinline__ void load_words(uint32_t addr, uint32_t (&v)[N]) {
    if constexpr (N == 1u) {
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[0]) : "r"(addr) : "memory");
    } else if constexpr (N == 2u) {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory");
    } else {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
    }
}
// A scale in both halves.
__device__ __forceinline__ uint32_t load_scale(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return v * 0x10001u;
}
// The 8 x 8 matrix of 16-bit numbers that the warp holds, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

template <uint32_t HD, uint32_t ROWS, bool BALANCED>
__device__ __forceinline__ void attention_few4(const AttnArgs& a) {
    using F = Few4<HD, ROWS>;
    constexpr uint32_t kN = ROWS / 4u;  // columns of eight: four rows each
    extern __shared__ __align__(128) uint8_t sm[];
    uint8_t* const ring = sm + F::kQueries;
    __shared__ float row_unscale[ROWS];
    __shared__ uint32_t row_tok[ROWS], row_head[ROWS];
    __shared__ int row_pos[ROWS];
    __shared__ float wm[kWarps][ROWS], wl[kWarps][ROWS];
    __shared__ uint32_t list[kMaxPicks];
    const uint32_t hd = a.kv.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    FewItem it;
    if (!few_setup<ROWS, BALANCED>(a, row_tok, row_head, row_pos, list, &it)) return;
    const uint32_t c = it.c, kh = it.kh, s = it.s, kb = it.kb, ke = it.ke, all_b = it.all_b, all_e = it.all_e;
    const uint32_t g = lane >> 2, t = lane & 3u;
    // this warp's tiles: tile i starts at key j0 + 32 (4 i + warp); lane 2 i + h holds the page of its half h
    // and the position of its first key
    const uint32_t j0 = kb & ~15u;
    const uint32_t ntiles_all = kb < ke ? (ke - j0 + kKeys - 1u) / kKeys : 0u;
    const uint32_t ntiles = ntiles_all > warp ? (ntiles_all - warp + kWarps - 1u) / kWarps : 0u;
    uint32_t my_page = kNone, my_pos = 0;
    {
        const uint32_t j = j0 + kKeys * (kWarps * (lane >> 1) + warp) + 16u * (lane & 1u);
        if (lane < 2u * ntiles && j < ke) {
            const uint32_t lp = a.part == kPartBlocks ? list[j >> a.kv.page_shift] : j >> a.kv.page_shift;
            if (lp != kNone) {
                my_pos = (lp << a.kv.page_shift) + (j & (a.kv.page_size - 1u));
                // a list's last page may reach beyond the sequence
                if (a.part != kPartBlocks || my_pos <= static_cast<uint32_t>(row_pos[0]))
                    my_page = load_page(a.b, a.kv, s, lp, a.st);
            }
        }
    }
    const uint32_t ring_addr = smem_addr(ring + warp * F::kStages * F::kStageBytes);
    const uint32_t blocks = hd >> 5;  // of a key
    const uint32_t head_bytes = q4_head_bytes(a.kv), row_bytes = hd / 2u;
    const uint8_t* kbase = static_cast<const uint8_t*>(a.kv.k) + static_cast<size_t>(kh) * head_bytes;
    const uint8_t* vbase = static_cast<const uint8_t*>(a.kv.v) + static_cast<size_t>(kh) * head_bytes;
    const size_t page_bytes = static_cast<size_t>(a.kv.kv_heads) * head_bytes;
    // a tile's keys, whole; of no page: numbers and scales zero
    auto fetch = [&](uint32_t i) {
        if (i < ntiles) {
            const uint32_t dst = ring_addr + (i % F::kStages) * F::kStageBytes;
#pragma unroll
            for (uint32_t h = 0; h < kGroups; ++h) {
                const uint32_t page = __shfl_sync(0xFFFFFFFFu, my_page, 2u * i + h), pos = __shfl_sync(0xFFFFFFFFu, my_pos, 2u * i + h);
                const uint32_t bytes = page == kNone ? 0u : 16u, slot = pos & (a.kv.page_size - 1u);
                const size_t off = (page == kNone ? 0u : page) * page_bytes;
                const uint8_t *kp = kbase + off, *vp = vbase + off;
#pragma unroll
                for (uint32_t x = lane; x < 16u * F::kBlocks; x += 32u) {
                    const uint32_t r = x / F::kBlocks, ch = x % F::kBlocks;
                    if (ch >= blocks) continue;
                    const uint32_t o = (slot + r) * row_bytes + ch * 16u;
                    cp_async16(dst + key_at<HD>(16u * h + r, ch), kp + o, bytes);
                    cp_async16(dst + F::kTileBytes + value_at<HD>(16u * h + r, ch), vp + o, bytes);
                }
                // scales: two pieces of a block, of the keys and of the values
                const uint32_t b = (lane >> 1) % F::kBlocks, v = (lane >> 1) / F::kBlocks, half = (lane & 1u) * 16u;
                if (lane < 4u * F::kBlocks && b < blocks)
                    cp_async16(dst + v * F::kTileBytes + F::kScales + (h * F::kBlocks + b) * 32u + half,
                               (v ? vp : kp) + a.kv.page_size * row_bytes + (b * a.kv.page_size + slot) * 2u + half, bytes);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (uint32_t i = 0; i + 1u < F::kStages; ++i) fetch(i);

    // queries as columns, for all warps: column g of eight is the high (g even) or low half of row 4 n + g / 2;
    // of product s lane t has four channels, of the block(s) that it takes of every key
    constexpr uint32_t kSteps = HD / 16u, kKeyWords = HD / 32u, kValueWords = HD / 64u;
    {
        // 128 / ROWS neighbouring threads to a row, four channels at a time
        constexpr uint32_t kLanes = kThreads / ROWS, kTurns4 = (HD / 4u + kLanes - 1u) / kLanes;
        const uint32_t r = tid / kLanes;
        const float* q = a.q + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd;
        float4 x[kTurns4];
        float big = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < kTurns4; ++i) {
            const uint32_t ch = 4u * (i * kLanes + tid % kLanes);
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row_pos[r] >= 0 && ch < hd) x[i] = *reinterpret_cast<const float4*>(q + ch);
        }
#pragma unroll
        for (uint32_t i = 0; i < kTurns4; ++i) {
            x[i] = make_float4(x[i].x * a.scale_log2, x[i].y * a.scale_log2, x[i].z * a.scale_log2, x[i].w * a.scale_log2);
            big = fmaxf(big, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        }
#pragma unroll
        for (uint32_t o = 1; o < kLanes; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
        const int e2 = up_exponent(big);
        const float up = power_of_two(e2);
        if (tid % kLanes == 0u) row_unscale[r] = power_of_two(-e2);
#pragma unroll
        for (uint32_t i = 0; i < kTurns4; ++i) {
            const uint32_t ch = 4u * (i * kLanes + tid % kLanes);
            // the channels' lane and product
            const uint32_t to = HD == 64u ? ch >> 4 : (ch >> 5) & 3u;
            const uint32_t step = HD == 64u ? (ch & 15u) >> 2 : (ch >> 7) * 8u + ((ch & 31u) >> 2);
            if (ch >= HD) break;
            uint32_t hi[2], lo[2];
            split(x[i].x * up, x[i].y * up, &hi[0], &lo[0]);
            split(x[i].z * up, x[i].w * up, &hi[1], &lo[1]);
            uint2* const at = reinterpret_cast<uint2*>(sm) + (step * kN + (r >> 2)) * 32u + 8u * (r & 3u) + to;
            at[0] = make_uint2(hi[0], hi[1]);
            at[4] = make_uint2(lo[0], lo[1]);
        }
    }
    __syncthreads();
    const uint32_t q_addr = smem_addr(sm) + 8u * lane;
    float unscale[kN], m[kN], l[kN];  // of row 4 n + t, as the scores come
    uint32_t p_lo[kN], p_hi[kN];
#pragma unroll
    for (uint32_t n = 0; n < kN; ++n) {
        unscale[n] = row_unscale[4u * n + t];
        const int p = row_pos[4u * n + t];
        p_lo[n] = p >= 0 ? first_key(p, a.window) : kNone;
        p_hi[n] = p >= 0 ? static_cast<uint32_t>(p) + 1u : 0u;
        m[n] = -INFINITY;
        l[n] = 0.f;
    }
    // sums of row 4 n + t: channels HD / 8 g + 8 y + 2 e + p at [4 y + 2 p + e / 2][n][e % 2]
    float acc[kSteps][kN][2];
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i)
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n) acc[i][n][0] = acc[i][n][1] = 0.f;

    // where this thread's parts of a tile are (keys 8 further, and 16, at fixed distances); blocks that the head
    // does not have count as zero
    const uint32_t key_off = HD == 64u ? key_at<HD>(g, t >> 1) + (t & 1u) * 8u : key_at<HD>(g, t);
    const uint32_t key_scale = F::kScales + (HD == 64u ? t >> 1 : t) * 32u + 2u * g;
    const uint32_t value_block = HD == 64u ? g >> 2 : HD == 128u ? g >> 1 : g;
    const uint32_t value_in = HD == 64u ? (g & 3u) * 4u : HD == 128u ? (g & 1u) * 8u : 0u;
    const uint32_t value_off0 = F::kTileBytes + value_at<HD>(2u * t, value_block) + value_in;
    const uint32_t value_off1 = F::kTileBytes + value_at<HD>(2u * t + 1u, value_block) + value_in;
    const uint32_t value_scale = F::kTileBytes + F::kScales + value_block * 32u + 4u * t;
    const uint32_t key_mask = (HD == 64u ? t >> 1 : t) < blocks ? ~0u : 0u, value_mask = value_block < blocks ? ~0u : 0u;
    const uint32_t far_mask = t + 4u < blocks ? ~0u : 0u;  // HD 256: the second block
    for (uint32_t i = 0; i < ntiles; ++i) {
        fetch(i + F::kStages - 1u);
        cp_wait<F::kStages - 1>();
        __syncwarp();
        const uint32_t stage = ring_addr + (i % F::kStages) * F::kStageBytes;
        uint32_t page[kGroups], pos[kGroups];
        bool whole = true;
#pragma unroll
        for (uint32_t h = 0; h < kGroups; ++h) {
            page[h] = __shfl_sync(0xFFFFFFFFu, my_page, 2u * i + h);
            pos[h] = __shfl_sync(0xFFFFFFFFu, my_pos, 2u * i + h);
            whole = whole && page[h] != kNone && pos[h] >= all_b && pos[h] + 16u <= all_e;
        }
        if (!whole) {
            // values that no row of the item sees count as zero, whatever their scales hold
            const uint32_t h = lane >> 4, key = (h ? pos[1] : pos[0]) + (lane & 15u);
            const uint32_t lo = a.part == kPartBlocks ? 0u : kb;
            const uint32_t hi = a.part == kPartBlocks ? static_cast<uint32_t>(row_pos[0]) + 1u : ke;
            if (key < lo || key >= hi)
                for (uint32_t b = 0; b < blocks; ++b)
                    asm volatile("st.shared.b16 [%0], %1;" ::"r"(stage + F::kTileBytes + F::kScales + (h * F::kBlocks + b) * 32u + (lane & 15u) * 2u),
                                 "h"(static_cast<uint16_t>(0))
                                 : "memory");
            __syncwarp();
        }
        float sc[kGroups][kN][4];  // keys g and g + 8: high and low sums
#pragma unroll
        for (uint32_t h = 0; h < kGroups; ++h)
#pragma unroll
            for (uint32_t n = 0; n < kN; ++n) sc[h][n][0] = sc[h][n][1] = sc[h][n][2] = sc[h][n][3] = 0.f;
#pragma unroll
        for (uint32_t far = 0; far < (HD == 256u ? 2u : 1u); ++far) {
            constexpr uint32_t kWords = HD == 256u ? 4u : kKeyWords;
            uint32_t w[kGroups][2][kWords];
            __half2 d[kGroups][2];
            // (HD 256: the other block, at 64 bytes this or that way)
            const uint32_t from = stage + (far ? key_off ^ 64u : key_off);
#pragma unroll
            for (uint32_t h = 0; h < kGroups; ++h)
#pragma unroll
                for (uint32_t u = 0; u < 2u; ++u) {
                    load_words<kWords>(from + (16u * h + 8u * u) * F::kRowBytes, w[h][u]);
                    const uint32_t x = load_scale(stage + key_scale + far * 128u + h * F::kBlocks * 32u + 16u * u) & (far ? far_mask : key_mask);
                    d[h][u] = *reinterpret_cast<const __half2*>(&x);
                }
#pragma unroll
            for (uint32_t y = 0; y < kWords; ++y) {
                __half2 k[kGroups][2][4];
#pragma unroll
                for (uint32_t h = 0; h < kGroups; ++h)
#pragma unroll
                    for (uint32_t u = 0; u < 2u; ++u) {
                        q4_pairs(w[h][u][y], k[h][u]);
#pragma unroll
                        for (uint32_t e = 0; e < 4u; ++e) k[h][u][e] = __hmul2(k[h][u][e], d[h][u]);
                    }
#pragma unroll
                for (uint32_t e = 0; e < 2u; ++e)
#pragma unroll
                    for (uint32_t n = 0; n < kN; ++n) {
                        uint32_t q[2];
                        load_words<2>(q_addr + ((far * 8u + 2u * y + e) * kN + n) * 256u, q);
#pragma unroll
                        for (uint32_t h = 0; h < kGroups; ++h) {
                            const uint32_t x[4] = {pack(k[h][0][2u * e]), pack(k[h][1][2u * e]), pack(k[h][0][2u * e + 1u]), pack(k[h][1][2u * e + 1u])};
                            mma(sc[h][n], x, q[0], q[1]);
                        }
                    }
            }
        }
        float v[kN][2 * kGroups];
        bool more = false;
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n) {
#pragma unroll
            for (uint32_t e = 0; e < 2u * kGroups; ++e) {
                v[n][e] = fmaf(sc[e >> 1][n][2u * (e & 1u) + 1u], kLowDown, sc[e >> 1][n][2u * (e & 1u)]) * unscale[n];
                if (!whole) {
                    const uint32_t key = pos[e >> 1] + g + 8u * (e & 1u);
                    if (page[e >> 1] == kNone || key < p_lo[n] || key >= p_hi[n]) v[n][e] = -INFINITY;
                }
            }
            more |= fmaxf(fmaxf(v[n][0], v[n][1]), fmaxf(v[n][2], v[n][3])) > m[n];
        }
        if (__any_sync(0xFFFFFFFFu, more)) {
#pragma unroll
            for (uint32_t n = 0; n < kN; ++n) {
                float mn = fmaxf(m[n], fmaxf(fmaxf(v[n][0], v[n][1]), fmaxf(v[n][2], v[n][3])));
#pragma unroll
                for (uint32_t o = 4; o <= 16u; o <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xFFFFFFFFu, mn, o));
                const float al = mn == -INFINITY ? 1.f : exp2f(m[n] - mn);
                m[n] = mn;
                l[n] *= al;
#pragma unroll
                for (uint32_t x = 0; x < kSteps; ++x) {
                    acc[x][n][0] *= al;
                    acc[x][n][1] *= al;
                }
            }
        }
        uint32_t w[kGroups][kN][2];
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n) {
            const float ref = (m[n] == -INFINITY ? 0.f : m[n]) - kUp;
#pragma unroll
            for (uint32_t h = 0; h < kGroups; ++h) {
                const float p0 = exp2_fast(v[n][2u * h] - ref), p1 = exp2_fast(v[n][2u * h + 1u] - ref);
                l[n] += p0 + p1;
                uint32_t hi, lo;
                split(p0, p1, &hi, &lo);
                w[h][n][0] = transposed(prmt(hi, lo, 0x5410u));
                w[h][n][1] = transposed(prmt(hi, lo, 0x7632u));
            }
        }
        // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of either half
        uint32_t x[kGroups][4][kValueWords], d[kGroups][2];
#pragma unroll
        for (uint32_t h = 0; h < kGroups; ++h)
#pragma unroll
            for (uint32_t u = 0; u < 2u; ++u) {
                uint32_t one[1];
                load_words<kValueWords>(stage + value_off0 + (16u * h + 8u * u) * F::kRowBytes, x[h][2u * u]);
                load_words<kValueWords>(stage + value_off1 + (16u * h + 8u * u) * F::kRowBytes, x[h][2u * u + 1u]);
                load_words<1>(stage + value_scale + h * F::kBlocks * 32u + 16u * u, one);
                d[h][u] = one[0] & value_mask;
            }
#pragma unroll
        for (uint32_t y = 0; y < kValueWords; ++y)
#pragma unroll
            for (uint32_t odd = 0; odd < 2u; ++odd) {
                __half2 f[kGroups][2][4];
#pragma unroll
                for (uint32_t h = 0; h < kGroups; ++h)
#pragma unroll
                    for (uint32_t u = 0; u < 2u; ++u) {
                        q4_pairs(prmt(x[h][2u * u][y], x[h][2u * u + 1u][y], odd ? 0x7632u : 0x5410u), f[h][u]);
#pragma unroll
                        for (uint32_t e = 0; e < 4u; ++e) f[h][u][e] = __hmul2(f[h][u][e], *reinterpret_cast<const __half2*>(&d[h][u]));
                    }
#pragma unroll
                for (uint32_t e = 0; e < 2u; ++e)
#pragma unroll
                    for (uint32_t n = 0; n < kN; ++n) {
                        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (uint32_t h = 0; h < kGroups; ++h) {
                            const uint32_t va[4] = {pack(f[h][0][2u * e]), pack(f[h][0][2u * e + 1u]), pack(f[h][1][2u * e]), pack(f[h][1][2u * e + 1u])};
                            mma(o, va, w[h][n][0], w[h][n][1]);
                        }
                        float* const to = acc[4u * y + 2u * odd + e][n];
                        to[0] += fmaf(o[1], kLowDown, o[0]);
                        to[1] += fmaf(o[3], kLowDown, o[2]);
                    }
            }
        __syncwarp();
    }
    cp_wait<0>();
    asm volatile("griddepcontrol.launch_dependents;");  // the combining kernel may come up
    // the warps' sums, in warp order
    uint32_t again = 0;  // rows whose sums are not finite
#pragma unroll
    for (uint32_t n = 0; n < kN; ++n) {
        const uint32_t r = 4u * n + t;
#pragma unroll
        for (uint32_t o = 4; o <= 16u; o <<= 1) l[n] += __shfl_xor_sync(0xFFFFFFFFu, l[n], o);
        if (g == 0u) {
            wm[warp][r] = (m[n] == -INFINITY ? 0.f : m[n]) - kUp;
            wl[warp][r] = row_pos[r] >= 0 ? l[n] : 0.f;  // padding sees nothing
        }
        float odd = l[n] * 0.f;
#pragma unroll
        for (uint32_t i = 0; i < kSteps; ++i) odd = fmaf(acc[i][n][1], 0.f, fmaf(acc[i][n][0], 0.f, odd));
        if (odd != 0.f && row_pos[r] >= 0) again |= 1u << r;
    }
    again = __reduce_or_sync(0xFFFFFFFFu, again);
    __syncthreads();
    float* part = reinterpret_cast<float*>(ring);  // [warp][row][HD + 4]
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i)
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n)
#pragma unroll
            for (uint32_t e = 0; e < 2u; ++e)
                part[(warp * ROWS + 4u * n + t) * F::kPitch + HD / 8u * g + 8u * (i >> 2) + 4u * (i & 1u) + 2u * e + (i >> 1 & 1u)] = acc[i][n][e];
    if (again != 0u) {
        __syncwarp();
        while (again != 0u) {
            uint32_t n, rows = take_rows(&again, &n);
            RowSums x;
            rows_key_by_key<true>(a, s, kh, a.part == kPartBlocks ? list : nullptr, {row_tok, row_head, row_pos}, 0u, rows,
                                  j0 + kKeys * warp, ke, 16u, kKeys * kWarps, &x);
            for (uint32_t u = 0; u < n; ++u, rows >>= 8) {
                const uint32_t r = rows & 255u;
                for (uint32_t i = 0; lane + 32u * i < hd; ++i) part[(warp * ROWS + r) * F::kPitch + lane + 32u * i] = x.o[u][i];
                if (lane == 0u) {
                    wm[warp][r] = x.m[u];
                    wl[warp][r] = x.l[u];
                }
            }
        }
    }
    __syncthreads();
    few_finish<kWarps, ROWS>(a, c, row_tok, row_head, row_pos, wm, wl, part, F::kPitch);
}

template <uint32_t HD, uint32_t ROWS, bool BALANCED>
__global__ void __launch_bounds__(kThreads, HD <= 128u ? (ROWS <= 8u ? 4 : 3) : 2) attention_few4_kernel(const __grid_constant__ AttnArgs a) {
    attention_few4<HD, ROWS, BALANCED>(a);
    end_after_previous(a);
}

template <uint32_t HD, uint32_t ROWS>
cudaError_t launch(const AttnArgs& a, uint64_t items, cudaStream_t stream) {
    return launch_items(a, a.balance ? attention_few4_kernel<HD, ROWS, true> : attention_few4_kernel<HD, ROWS, false>, items, kThreads,
                        Few4<HD, ROWS>::kSmem, stream, a);
}

}  // namespace

cudaError_t launch_attention_few4(const AttnArgs& a, uint32_t rows, uint64_t items, cudaStream_t stream) {
    if (a.kv.head_dim > 128u) return rows <= 4u ? launch<256, 4>(a, items, stream) : launch<256, 8>(a, items, stream);
    if (a.kv.head_dim <= 64u)
        return rows <= 4u ? launch<64, 4>(a, items, stream) : rows <= 8u ? launch<64, 8>(a, items, stream) : launch<64, 16>(a, items, stream);
    return rows <= 4u ? launch<128, 4>(a, items, stream) : rows <= 8u ? launch<128, 8>(a, items, stream) : launch<128, 16>(a, items, stream);
}

}  // namespace nedo_gpu

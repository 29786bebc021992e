// paged_attention_few4.cu -- attention over a paged Q4_0 cache for tiles of up to four, eight or
// sixteen query rows (single tokens with their group of heads, a few drafted tokens, the rows of a
// page list): the shape of decoding, bound by reading the cache and by making fp16 numbers of it.
//
// Mathematics.  As over F16 caches the fp32 factors are split in two fp16 halves, x = hi + 2^-11 lo
// (queries scaled by a power of two per row, weights by 2^14), and a tile's weighted values are
// summed from zero.  Keys and values are the A operands here, S^T = K Q^T and O^T = V^T P^T, made in
// registers from the words that the cache holds: which channel or key stands in which place of a sum
// is free as long as the other factor follows, so a thread's word of eight channels is its part of
// both operands of a 32-channel block, and neither is written anywhere.  The columns are the rows'
// halves next to each other, (hi, lo) of four rows in the eight columns of an m16n8k16, so a row's
// score is in one thread, and its weight as the pair (hi, lo) is the operand of P^T after one
// transposing register move.
//
// Work.  A CTA of four warps takes one row tile and one chunk of keys; each warp streams every
// fourth 16-key tile through a ring of its own (cp.async), with its own running maximum and sums,
// so the warps meet only at the end.  A 16-key tile lies within one page.
#include "paged_attention.cuh"
#include "paged_mma.cuh"
#include "paged_q4.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kKeys = 16;  // keys per tile

template <uint32_t HD, uint32_t ROWS>
struct Few4 {
    static constexpr uint32_t kStages = 4;
    static constexpr uint32_t kBlocks = HD / 32u;
    static constexpr uint32_t kRowBytes = HD / 2u;
    static constexpr uint32_t kScales = kKeys * kRowBytes;             // where a tile's scales begin: [block][key]
    static constexpr uint32_t kTileBytes = kScales + kBlocks * kKeys * 2u;  // keys or values of one tile
    static constexpr uint32_t kStageBytes = 2u * kTileBytes;
    static constexpr uint32_t kPitch = HD + 4u;
    static constexpr uint32_t kRing = kWarps * kStages * kStageBytes;
    static constexpr uint32_t kEnd = (kWarps * ROWS * kPitch + ROWS * HD) * 4u;  // the warps' sums, and the chunk's
    static constexpr uint32_t kSmem = kRing > kEnd ? kRing : kEnd;
};

// Byte offset of 16-byte chunk c (a block's numbers) of key r in a tile: eight keys' same chunk, and
// the same chunk of every other of eight keys, fall into different bank groups.
template <uint32_t HD>
__device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) {
    const uint32_t x = HD == 256u ? r & 7u : HD == 128u ? (r >> 1) & 3u : (r >> 2) & 1u;
    return r * (HD / 2u) + ((c ^ x) << 4);
}

__device__ __forceinline__ uint32_t load_word(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ __half2 load_twice(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return __half2half2(__ushort_as_half(v));
}
// The 8 x 8 matrix of 16-bit numbers that the warp holds, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

template <uint32_t HD, uint32_t ROWS>
__device__ __forceinline__ void attention_few4(const AttnArgs& a) {
    using F = Few4<HD, ROWS>;
    constexpr uint32_t kN = ROWS / 4u;  // columns of eight: four rows each
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint32_t row_tok[ROWS], row_head[ROWS];
    __shared__ int row_pos[ROWS];
    __shared__ float wm[kWarps][ROWS], wl[kWarps][ROWS];
    __shared__ uint32_t list[kMaxPicks];
    const uint32_t hd = a.kv.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    FewItem it;
    if (!few_setup<ROWS>(a, row_tok, row_head, row_pos, list, &it)) return;
    const uint32_t c = it.c, kh = it.kh, s = it.s, kb = it.kb, ke = it.ke, all_b = it.all_b, all_e = it.all_e;
    const uint32_t g = lane >> 2, t = lane & 3u;
    // this warp's tiles: tile i starts at key j0 + 16 (4 i + warp); lane i holds its page and
    // the position of its first key
    const uint32_t j0 = kb & ~(kKeys - 1u);
    const uint32_t ntiles_all = kb < ke ? (ke - j0 + kKeys - 1u) / kKeys : 0u;
    const uint32_t ntiles = ntiles_all > warp ? (ntiles_all - warp + kWarps - 1u) / kWarps : 0u;
    uint32_t my_page = kNone, my_pos = 0;
    if (lane < ntiles) {
        const uint32_t j = j0 + kKeys * (kWarps * lane + warp);
        const uint32_t lp = a.part == kPartBlocks ? list[j >> a.kv.page_shift] : j >> a.kv.page_shift;
        if (lp != kNone) {
            my_pos = (lp << a.kv.page_shift) + (j & (a.kv.page_size - 1u));
            // a list's last page may reach beyond the sequence
            if (a.part != kPartBlocks || my_pos <= static_cast<uint32_t>(row_pos[0]))
                my_page = load_page(a.b, a.kv, s, lp, a.st);
        }
    }
    uint8_t* my_ring = ring + warp * F::kStages * F::kStageBytes;
    const uint32_t ring_addr = smem_addr(my_ring);
    const uint32_t blocks = hd >> 5;  // of a key; the last ones of HD are passed over
    const uint32_t head_bytes = q4_head_bytes(a.kv), scales_at = q4_scales_at(a.kv);
    const uint8_t* kbase = static_cast<const uint8_t*>(a.kv.k);
    const uint8_t* vbase = static_cast<const uint8_t*>(a.kv.v);
    // a tile's sixteen keys, whole; of no page: numbers and scales zero
    auto fetch = [&](uint32_t i) {
        if (i < ntiles) {
            const uint32_t page = __shfl_sync(0xFFFFFFFFu, my_page, i), pos = __shfl_sync(0xFFFFFFFFu, my_pos, i);
            const uint32_t dst = ring_addr + (i % F::kStages) * F::kStageBytes;
            const uint32_t bytes = page == kNone ? 0u : 16u, slot = pos & (a.kv.page_size - 1u);
            const size_t off = (static_cast<size_t>(page == kNone ? 0u : page) * a.kv.kv_heads + kh) * head_bytes;
            const uint8_t *kp = kbase + off, *vp = vbase + off;
#pragma unroll
            for (uint32_t x = lane; x < kKeys * F::kBlocks; x += 32u) {
                const uint32_t r = x / F::kBlocks, ch = x % F::kBlocks;
                if (ch >= blocks) continue;
                const uint32_t o = (slot + r) * (hd / 2u) + ch * 16u;
                cp_async16(dst + at<HD>(r, ch), kp + o, bytes);
                cp_async16(dst + F::kTileBytes + at<HD>(r, ch), vp + o, bytes);
            }
            if (lane < 4u * F::kBlocks) {  // scales: two pieces of a block, of the keys and of the values
                const uint32_t b = (lane >> 1) % F::kBlocks, v = (lane >> 1) / F::kBlocks, half = (lane & 1u) * 16u;
                if (b < blocks)
                    cp_async16(dst + v * F::kTileBytes + F::kScales + b * (kKeys * 2u) + half,
                               (v ? vp : kp) + scales_at + (b * a.kv.page_size + slot) * 2u + half, bytes);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (uint32_t i = 0; i + 1u < F::kStages; ++i) fetch(i);

    // queries as columns: column g of eight is the high (g even) or low half of row 4 n + g / 2, its
    // places of a block's two products channels 8 t .. 8 t + 7
    uint32_t qf[kN][F::kBlocks][4];
    float unscale[kN], m[kN], l[kN];  // of row 4 n + t, as the scores come
    uint32_t p_lo[kN], p_hi[kN];
#pragma unroll
    for (uint32_t n = 0; n < kN; ++n) {
        const uint32_t r = 4u * n + (g >> 1);
        const float* q = a.q + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd;
        float2 x[F::kBlocks][4];
        float big = 0.f;
#pragma unroll
        for (uint32_t b = 0; b < F::kBlocks; ++b) {
            float4 y[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
            if (row_pos[r] >= 0 && b < blocks) {
                y[0] = *reinterpret_cast<const float4*>(q + 32u * b + 8u * t);
                y[1] = *reinterpret_cast<const float4*>(q + 32u * b + 8u * t + 4u);
            }
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) {
                x[b][e] = e & 1u ? make_float2(y[e >> 1].z, y[e >> 1].w) : make_float2(y[e >> 1].x, y[e >> 1].y);
                x[b][e].x *= a.scale_log2;
                x[b][e].y *= a.scale_log2;
                big = fmaxf(big, fmaxf(fabsf(x[b][e].x), fabsf(x[b][e].y)));
            }
        }
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
        const int e2 = up_exponent(big);
        const float up = power_of_two(e2);
#pragma unroll
        for (uint32_t b = 0; b < F::kBlocks; ++b)
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) {
                uint32_t hi, lo;
                split(x[b][e].x * up, x[b][e].y * up, &hi, &lo);
                qf[n][b][e] = g & 1u ? lo : hi;
            }
        unscale[n] = power_of_two(-__shfl_sync(0xFFFFFFFFu, e2, 8u * t));
        const int p = row_pos[4u * n + t];
        p_lo[n] = p >= 0 ? first_key(p, a.window) : kNone;
        p_hi[n] = p >= 0 ? static_cast<uint32_t>(p) + 1u : 0u;
        m[n] = -INFINITY;
        l[n] = 0.f;
    }
    // sums of row 4 n + t: channels 32 b + 8 (g % 4) + g / 4 + 0, 2, 4, 6
    float acc[F::kBlocks][kN][4];
#pragma unroll
    for (uint32_t b = 0; b < F::kBlocks; ++b)
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n) acc[b][n][0] = acc[b][n][1] = acc[b][n][2] = acc[b][n][3] = 0.f;

    const uint32_t pick = g & 4u ? 0x7632u : 0x5410u;  // the odd or the even channels of two keys' words
    for (uint32_t i = 0; i < ntiles; ++i) {
        fetch(i + F::kStages - 1u);
        cp_wait<F::kStages - 1>();
        __syncwarp();
        const uint32_t ks = ring_addr + (i % F::kStages) * F::kStageBytes, vs = ks + F::kTileBytes;
        const uint32_t page = __shfl_sync(0xFFFFFFFFu, my_page, i), pos = __shfl_sync(0xFFFFFFFFu, my_pos, i);
        const bool whole = page != kNone && pos >= all_b && pos + kKeys <= all_e;
        if (!whole && page != kNone) {
            // values that no row of the item sees count as zero, whatever their scales hold
            const uint32_t key = pos + (lane & 15u);
            const uint32_t lo = a.part == kPartBlocks ? 0u : kb;
            const uint32_t hi = a.part == kPartBlocks ? static_cast<uint32_t>(row_pos[0]) + 1u : ke;
            if (key < lo || key >= hi)
                for (uint32_t b = lane >> 4; b < blocks; b += 2u)
                    asm volatile("st.shared.b16 [%0], %1;" ::"r"(vs + F::kScales + b * (kKeys * 2u) + (lane & 15u) * 2u),
                                 "h"(static_cast<uint16_t>(0))
                                 : "memory");
            __syncwarp();
        }
        float sc[kN][4];  // keys g and g + 8: high and low sums
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
        for (uint32_t b = 0; b < F::kBlocks; ++b) {
            if (b >= blocks) continue;
            __half2 k[2][4];
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                q4_pairs(load_word(ks + at<HD>(g + 8u * h, b) + 4u * t), k[h]);
                const __half2 d = load_twice(ks + F::kScales + b * (kKeys * 2u) + (g + 8u * h) * 2u);
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) k[h][e] = __hmul2(k[h][e], d);
            }
            const uint32_t a0[4] = {pack(k[0][0]), pack(k[1][0]), pack(k[0][1]), pack(k[1][1])};
            const uint32_t a1[4] = {pack(k[0][2]), pack(k[1][2]), pack(k[0][3]), pack(k[1][3])};
#pragma unroll
            for (uint32_t n = 0; n < kN; ++n) {
                mma(sc[n], a0, qf[n][b][0], qf[n][b][1]);
                mma(sc[n], a1, qf[n][b][2], qf[n][b][3]);
            }
        }
        float v[kN][2];
        bool more = false;
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n) {
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                v[n][h] = fmaf(sc[n][2u * h + 1u], kLowDown, sc[n][2u * h]) * unscale[n];
                if (!whole) {
                    const uint32_t key = pos + g + 8u * h;
                    if (page == kNone || key < p_lo[n] || key >= p_hi[n]) v[n][h] = -INFINITY;
                }
            }
            more |= fmaxf(v[n][0], v[n][1]) > m[n];
        }
        if (__any_sync(0xFFFFFFFFu, more)) {
#pragma unroll
            for (uint32_t n = 0; n < kN; ++n) {
                float mn = fmaxf(m[n], fmaxf(v[n][0], v[n][1]));
#pragma unroll
                for (uint32_t o = 4; o <= 16u; o <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xFFFFFFFFu, mn, o));
                const float al = mn == -INFINITY ? 1.f : exp2f(m[n] - mn);
                m[n] = mn;
                l[n] *= al;
#pragma unroll
                for (uint32_t b = 0; b < F::kBlocks; ++b)
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e) acc[b][n][e] *= al;
            }
        }
        uint32_t w[kN][2];
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n) {
            const float ref = (m[n] == -INFINITY ? 0.f : m[n]) - kUp;
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) v[n][h] = exp2_fast(v[n][h] - ref);
            l[n] += v[n][0] + v[n][1];
            uint32_t hi, lo;
            split(v[n][0], v[n][1], &hi, &lo);
            w[n][0] = transposed(prmt(hi, lo, 0x5410u));
            w[n][1] = transposed(prmt(hi, lo, 0x7632u));
        }
#pragma unroll
        for (uint32_t b = 0; b < F::kBlocks; ++b) {
            if (b >= blocks) continue;
            __half2 y[2][4];  // keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                const uint32_t r = 2u * t + 8u * h;
                const uint32_t w0 = load_word(vs + at<HD>(r, b) + 4u * (g & 3u));
                const uint32_t w1 = load_word(vs + at<HD>(r + 1u, b) + 4u * (g & 3u));
                q4_pairs(prmt(w0, w1, pick), y[h]);
                const uint32_t d = load_word(vs + F::kScales + b * (kKeys * 2u) + r * 2u);
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) y[h][e] = __hmul2(y[h][e], *reinterpret_cast<const __half2*>(&d));
            }
#pragma unroll
            for (uint32_t u = 0; u < 2u; ++u) {
                const uint32_t x[4] = {pack(y[0][2u * u]), pack(y[0][2u * u + 1u]), pack(y[1][2u * u]), pack(y[1][2u * u + 1u])};
#pragma unroll
                for (uint32_t n = 0; n < kN; ++n) {
                    float o[4] = {0.f, 0.f, 0.f, 0.f};
                    mma(o, x, w[n][0], w[n][1]);
                    acc[b][n][2u * u] += fmaf(o[1], kLowDown, o[0]);
                    acc[b][n][2u * u + 1u] += fmaf(o[3], kLowDown, o[2]);
                }
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
        for (uint32_t b = 0; b < F::kBlocks; ++b)
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) odd = fmaf(acc[b][n][e], 0.f, odd);
        if (odd != 0.f && row_pos[r] >= 0) again |= 1u << r;
    }
    again = __reduce_or_sync(0xFFFFFFFFu, again);
    __syncthreads();
    float* part = reinterpret_cast<float*>(ring);  // [warp][row][HD + 4]
#pragma unroll
    for (uint32_t b = 0; b < F::kBlocks; ++b)
#pragma unroll
        for (uint32_t n = 0; n < kN; ++n)
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e)
                part[(warp * ROWS + 4u * n + t) * F::kPitch + 32u * b + 8u * (g & 3u) + (g >> 2) + 2u * e] = acc[b][n][e];
    if (again != 0u) {
        __syncwarp();
        while (again != 0u) {
            uint32_t n, rows = take_rows(&again, &n);
            RowSums x;
            rows_key_by_key<true>(a, s, kh, a.part == kPartBlocks ? list : nullptr, {row_tok, row_head, row_pos}, 0u, rows,
                                  j0 + kKeys * warp, ke, kKeys * kWarps, &x);
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

template <uint32_t HD, uint32_t ROWS>
__global__ void __launch_bounds__(kThreads) attention_few4_kernel(const __grid_constant__ AttnArgs a) {
    attention_few4<HD, ROWS>(a);
    end_after_previous(a);
}

template <uint32_t HD, uint32_t ROWS>
cudaError_t launch(const AttnArgs& a, uint64_t items, cudaStream_t stream) {
    return launch_items(a, attention_few4_kernel<HD, ROWS>, items, kThreads, Few4<HD, ROWS>::kSmem, stream, a);
}

}  // namespace

cudaError_t launch_attention_few4(const AttnArgs& a, uint32_t rows, uint64_t items, cudaStream_t stream) {
    if (a.kv.head_dim > 128u) return rows <= 4u ? launch<256, 4>(a, items, stream) : launch<256, 8>(a, items, stream);
    if (a.kv.head_dim <= 64u)
        return rows <= 4u ? launch<64, 4>(a, items, stream) : rows <= 8u ? launch<64, 8>(a, items, stream) : launch<64, 16>(a, items, stream);
    return rows <= 4u ? launch<128, 4>(a, items, stream) : rows <= 8u ? launch<128, 8>(a, items, stream) : launch<128, 16>(a, items, stream);
}

}  // namespace nedo_gpu

// paged_attention_few.cu -- attention over a paged F16 cache for tiles of up to eight or
// sixteen query rows (single tokens with their group of heads, a few tokens of small
// groups, the rows of a page list): the shape of decoding, bound by reading the cache.
//
// Mathematics.  Queries and weights are fp32 and the cache is fp16, so every product
// runs on the fp16 tensor cores with the fp32 side split in two halves,
// x = hi + 2^-11 lo, that keep 22 bits of it: q is scaled by a power of two per row (its
// largest channel to [2^13, 2^14)), and the weights p = 2^(s - m + 14) are taken up by the same
// factor in numerator and sum.  The
// two halves ride in one m16n8k16 operand, rows 0-7 the high and rows 8-15 the low half
// of the same eight query rows, so the split costs no extra instruction: both parts of a
// row's sum land in the same thread, which adds them.  With more than eight rows the halves
// are operands of their own.  Every tile's weighted values are summed from zero and added in
// fp32: the tensor core cuts its sums instead of rounding them, by up to a step every time.
//
// Work.  A CTA of four warps takes one row tile and one chunk of keys; each warp streams
// every fourth 16-key tile through a ring of its own (cp.async, three stages), with its
// own running maximum and sums, so the warps meet only at the end.  A 16-key tile lies
// within one page.  Two CTAs share an SM.
//
// 32 single tokens of 12 query and 4 KV heads of 128 channels over 8191 to 32768 keys: 215 us,
// 6.6 TB/s.  32 query heads over 2 KV heads, 5000 to 20000 keys: 90 us in tiles of 16 rows, 4.8
// TB/s (118 us in two tiles of 8, which both read the cache).  Heads above 128 keep to 8: the
// queries and sums of 16 rows would not stay in registers.
#include "paged_attention.cuh"
#include "paged_mma.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kKeys = 16;         // keys per tile

template <uint32_t HD>
struct Few {
    static constexpr uint32_t kStages = HD == 256 ? 2 : 3;
    static constexpr uint32_t kRowBytes = HD * 2u;
    static constexpr uint32_t kTileBytes = kKeys * kRowBytes;      // keys or values of one tile
    static constexpr uint32_t kStageBytes = 2u * kTileBytes;
    static constexpr uint32_t kSmem = kWarps * kStages * kStageBytes;
};

// Byte offset of 16-byte chunk `c` of row `r` in a tile: chunks swapped by the row's
// number so that eight rows' same chunk falls into eight different bank groups.
template <uint32_t HD>
__device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) {
    return r * Few<HD>::kRowBytes + ((c ^ (r & 7u)) << 4);
}

// up_exponent in other words: with the exponent taken from the number's bits the compiler orders
// the loop over the keys worse (16 rows, the case above: 90.5 us instead of 86.6).
__device__ __forceinline__ int row_exponent(float big) {
    return big > 0.f && big < INFINITY ? min(126, 13 - static_cast<int>(ilogbf(big))) : 0;
}

template <uint32_t HD, uint32_t ROWS>
__device__ __forceinline__ void attention_few(const AttnArgs& a) {
    using F = Few<HD>;
    constexpr uint32_t kMine = ROWS / 8u;  // rows of a thread: g, and g + 8 of 16
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint32_t row_tok[ROWS], row_head[ROWS];
    __shared__ int row_pos[ROWS];
    __shared__ float wm[kWarps][ROWS], wl[kWarps][ROWS];
    __shared__ uint32_t list[kMaxPicks];
    const uint32_t hd = a.kv.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    FewItem it;
    if (!few_setup<ROWS>(a, row_tok, row_head, row_pos, list, &it)) return;
    const uint32_t c = it.c, kh = it.kh, s = it.s, kb = it.kb, ke = it.ke, all_b = it.all_b, all_e = it.all_e;
    // the queries, on their way while the pages are looked up
    const uint32_t g = lane >> 2, t2 = (lane & 3u) * 2u;
    float2 qx[kMine][HD / 8];
#pragma unroll
    for (uint32_t h = 0; h < kMine; ++h) {
        const uint32_t r = g + 8u * h;
        const float* q = a.q + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd;
#pragma unroll
        for (uint32_t i = 0; i < HD / 8; ++i) {
            qx[h][i] = make_float2(0.f, 0.f);
            if (row_pos[r] >= 0 && i * 8u < hd) qx[h][i] = *reinterpret_cast<const float2*>(q + i * 8u + t2);
        }
    }
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
    if (hd < HD) {  // channels beyond the head stay zero
        for (uint32_t i = lane; i < F::kStages * F::kStageBytes / 16u; i += 32u)
            reinterpret_cast<uint4*>(my_ring)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncwarp();
    }
    const uint32_t chunks16 = hd >> 3;  // 16-byte chunks of a row
    const __half* kbase = static_cast<const __half*>(a.kv.k);
    const __half* vbase = static_cast<const __half*>(a.kv.v);
    // the keys of a tile that some row may see are copied, the others are zero
    auto fetch = [&](uint32_t i) {
        if (i < ntiles) {
            const uint32_t page = __shfl_sync(0xFFFFFFFFu, my_page, i), pos = __shfl_sync(0xFFFFFFFFu, my_pos, i);
            const uint32_t dst = ring_addr + (i % F::kStages) * F::kStageBytes;
            const size_t off = ((static_cast<size_t>(page == kNone ? 0u : page) * a.kv.kv_heads + kh) * a.kv.page_size +
                                (pos & (a.kv.page_size - 1u))) * hd;
            const uint32_t lo = a.part == kPartBlocks ? 0u : kb;
            const uint32_t hi = page == kNone ? 0u : a.part == kPartBlocks ? static_cast<uint32_t>(row_pos[0]) + 1u : ke;
#pragma unroll
            for (uint32_t x = lane; x < kKeys * (HD / 8u); x += 32u) {
                const uint32_t r = x / (HD / 8u), ch = x % (HD / 8u);
                if (ch >= chunks16) continue;
                const uint32_t bytes = pos + r >= lo && pos + r < hi ? 16u : 0u;
                const size_t o = off + static_cast<size_t>(bytes ? r : 0u) * hd + ch * 8u;
                cp_async16(dst + at<HD>(r, ch), kbase + o, bytes);
                cp_async16(dst + F::kTileBytes + at<HD>(r, ch), vbase + o, bytes);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (uint32_t i = 0; i + 1u < F::kStages; ++i) fetch(i);

    // this thread's query rows: g (and g + 8), channels 2t, 2t + 1, 2t + 8, 2t + 9 of every 16
    uint32_t qf[kMine][HD / 16][4];  // 8 rows: both halves in one operand; 16: the high and the low halves
    float unscale[kMine], m[kMine], l[kMine];
    uint32_t p_lo[kMine], p_hi[kMine];
#pragma unroll
    for (uint32_t h = 0; h < kMine; ++h) {
        const uint32_t r = g + 8u * h;
        const int p = row_pos[r];
        float2* const x = qx[h];
        float big = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < HD / 8; ++i) {
            x[i].x *= a.scale_log2;
            x[i].y *= a.scale_log2;
            big = fmaxf(big, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
        }
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
        const int e = row_exponent(big);
        const float up = power_of_two(e);
        unscale[h] = power_of_two(-e);
#pragma unroll
        for (uint32_t i = 0; i < HD / 16; ++i)
#pragma unroll
            for (uint32_t k = 0; k < 2u; ++k) {
                uint32_t* const high = &qf[0][i][2u * k + h];
                uint32_t* const low = kMine == 1u ? &qf[0][i][2u * k + 1u] : &qf[kMine - 1u][i][2u * k + h];
                split(x[2 * i + k].x * up, x[2 * i + k].y * up, high, low);
            }
        p_lo[h] = p >= 0 ? first_key(p, a.window) : kNone;
        p_hi[h] = p >= 0 ? static_cast<uint32_t>(p) + 1u : 0u;
        m[h] = -INFINITY;
        l[h] = 0.f;
    }
    float acc[HD / 8][4];
#pragma unroll
    for (uint32_t n = 0; n < HD / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;

    const uint32_t mi = lane >> 3, mr = lane & 7u;  // ldmatrix: this lane's matrix and row
    for (uint32_t i = 0; i < ntiles; ++i) {
        fetch(i + F::kStages - 1u);
        cp_wait<F::kStages - 1>();
        __syncwarp();
        const uint32_t ks = ring_addr + (i % F::kStages) * F::kStageBytes, vs = ks + F::kTileBytes;
        float sc[kMine][2][4];  // 16 rows: from the high and from the low halves
#pragma unroll
        for (uint32_t h = 0; h < kMine; ++h)
#pragma unroll
            for (uint32_t n = 0; n < 2; ++n) sc[h][n][0] = sc[h][n][1] = sc[h][n][2] = sc[h][n][3] = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < HD / 16; ++k) {
            uint32_t b[4];
            ldsm4(b, ks + at<HD>((mi >> 1) * 8u + mr, 2u * k + (mi & 1u)));
#pragma unroll
            for (uint32_t h = 0; h < kMine; ++h) {
                mma(sc[h][0], qf[h][k], b[0], b[1]);
                mma(sc[h][1], qf[h][k], b[2], b[3]);
            }
        }
        const uint32_t page = __shfl_sync(0xFFFFFFFFu, my_page, i), pos = __shfl_sync(0xFFFFFFFFu, my_pos, i);
        const bool whole = page != kNone && pos >= all_b && pos + kKeys <= all_e;
        float v[kMine][4], mn[kMine];  // keys pos + 2t, 2t + 1, 2t + 8, 2t + 9
        bool more = false;
#pragma unroll
        for (uint32_t h = 0; h < kMine; ++h) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const float high = sc[0][j >> 1][(j & 1u) + 2u * h];
                const float low = kMine == 1u ? sc[0][j >> 1][(j & 1u) + 2u] : sc[kMine - 1u][j >> 1][(j & 1u) + 2u * h];
                v[h][j] = fmaf(low, kLowDown, high) * unscale[h];
                if (!whole) {
                    const uint32_t at_key = pos + t2 + (j & 1u) + (j >> 1) * 8u;
                    if (page == kNone || at_key < p_lo[h] || at_key >= p_hi[h]) v[h][j] = -INFINITY;
                }
            }
            float mt = fmaxf(fmaxf(v[h][0], v[h][1]), fmaxf(v[h][2], v[h][3]));
            mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 1));
            mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 2));
            mn[h] = fmaxf(m[h], mt);
            more |= mt > m[h];
        }
        if (__any_sync(0xFFFFFFFFu, more)) {
            float al[kMine];
#pragma unroll
            for (uint32_t h = 0; h < kMine; ++h) {
                al[h] = mn[h] == -INFINITY ? 1.f : exp2f(m[h] - mn[h]);
                m[h] = mn[h];
                l[h] *= al[h];
            }
#pragma unroll
            for (uint32_t n = 0; n < HD / 8; ++n)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) acc[n][e] *= al[kMine == 1u ? 0u : e >> 1];
        }
        uint32_t pf[kMine][4];
#pragma unroll
        for (uint32_t h = 0; h < kMine; ++h) {
            const float ref = (m[h] == -INFINITY ? 0.f : m[h]) - kUp;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) v[h][j] = exp2_fast(v[h][j] - ref);
            l[h] += (v[h][0] + v[h][1]) + (v[h][2] + v[h][3]);
#pragma unroll
            for (uint32_t k = 0; k < 2u; ++k)
                split(v[h][2u * k], v[h][2u * k + 1u], &pf[0][2u * k + h], kMine == 1u ? &pf[0][2u * k + 1u] : &pf[kMine - 1u][2u * k + h]);
        }
#pragma unroll
        for (uint32_t n = 0; n < HD / 16; ++n) {
            uint32_t b[4];
            ldsm4t(b, vs + at<HD>((mi & 1u) * 8u + mr, 2u * n + (mi >> 1)));
            float o[2][4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) o[0][e] = o[1][e] = 0.f;
            if constexpr (kMine == 2u) {
                mma(o[0], pf[kMine - 1u], b[0], b[1]);
                mma(o[1], pf[kMine - 1u], b[2], b[3]);
                low_down(o[0]);
                low_down(o[1]);
            }
            mma(o[0], pf[0], b[0], b[1]);
            mma(o[1], pf[0], b[2], b[3]);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                acc[2 * n][e] += o[0][e];
                acc[2 * n + 1][e] += o[1][e];
            }
        }
        __syncwarp();
    }
    cp_wait<0>();
    asm volatile("griddepcontrol.launch_dependents;");  // the combining kernel may come up
    // the warps' sums, in warp order
    uint32_t again = 0;  // rows whose sums are not finite
#pragma unroll
    for (uint32_t h = 0; h < kMine; ++h) {
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
        if ((lane & 3u) == 0u) {
            wm[warp][g + 8u * h] = (m[h] == -INFINITY ? 0.f : m[h]) - kUp;
            wl[warp][g + 8u * h] = row_pos[g + 8u * h] >= 0 ? l[h] : 0.f;  // padding sees nothing
        }
        float odd = l[h] * 0.f;
#pragma unroll
        for (uint32_t n = 0; n < HD / 8; ++n)
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e)
                if (kMine == 1u || e >> 1 == h) odd = fmaf(acc[n][e], 0.f, odd);
        if (odd != 0.f && row_pos[g + 8u * h] >= 0) again |= 1u << (g + 8u * h);
    }
    again = __reduce_or_sync(0xFFFFFFFFu, again);
    __syncthreads();
    float* part = reinterpret_cast<float*>(ring);  // [warp][row][HD + 4]
    constexpr uint32_t kPitch = HD + 4u;
#pragma unroll
    for (uint32_t n = 0; n < HD / 8; ++n) {
        float* to = part + (warp * ROWS + g) * kPitch + n * 8u + t2;
        if constexpr (kMine == 1u) {
            *reinterpret_cast<float2*>(to) = make_float2(fmaf(acc[n][2], kLowDown, acc[n][0]), fmaf(acc[n][3], kLowDown, acc[n][1]));
        } else {
            *reinterpret_cast<float2*>(to) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2*>(to + 8u * kPitch) = make_float2(acc[n][2], acc[n][3]);
        }
    }
    if (again != 0u) {
        __syncwarp();
        while (again != 0u) {
            uint32_t n, rows = take_rows(&again, &n);
            RowSums x;
            rows_key_by_key(a, s, kh, a.part == kPartBlocks ? list : nullptr, {row_tok, row_head, row_pos}, 0u, rows,
                            j0 + kKeys * warp, ke, kKeys * kWarps, &x);
            for (uint32_t u = 0; u < n; ++u, rows >>= 8) {
                const uint32_t r = rows & 255u;
                for (uint32_t i = 0; lane + 32u * i < hd; ++i) part[(warp * ROWS + r) * kPitch + lane + 32u * i] = x.o[u][i];
                if (lane == 0u) {
                    wm[warp][r] = x.m[u];
                    wl[warp][r] = x.l[u];
                }
            }
        }
    }
    __syncthreads();
    few_finish<kWarps, ROWS>(a, c, row_tok, row_head, row_pos, wm, wl, part, kPitch);
}

template <uint32_t HD, uint32_t ROWS>
__global__ void __launch_bounds__(kThreads, 2) attention_few_kernel(const __grid_constant__ AttnArgs a) {
    attention_few<HD, ROWS>(a);
    end_after_previous(a);
}

template <uint32_t HD, uint32_t ROWS>
cudaError_t launch(const AttnArgs& a, uint64_t items, cudaStream_t stream) {
    return launch_items(a, attention_few_kernel<HD, ROWS>, items, kThreads, Few<HD>::kSmem, stream, a);
}

}  // namespace

cudaError_t launch_attention_few(const AttnArgs& a, uint32_t rows, uint64_t items, cudaStream_t stream) {
    if (a.kv.head_dim > 128u) return launch<256, 8>(a, items, stream);
    if (a.kv.head_dim <= 64u) return rows <= 8u ? launch<64, 8>(a, items, stream) : launch<64, 16>(a, items, stream);
    return rows <= 8u ? launch<128, 8>(a, items, stream) : launch<128, 16>(a, items, stream);
}

}  // namespace nedo_gpu

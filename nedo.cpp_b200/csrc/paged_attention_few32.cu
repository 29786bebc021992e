// paged_attention_few32.cu -- attention over a paged F32 cache for tiles of at most eight
// query rows: bound by reading the cache, on the CUDA cores in fp32.
//
// Work.  As in paged_attention_few.cu a CTA of four warps takes one row tile and one chunk
// of keys, each warp every fourth tile (of 8 keys here) through a cp.async ring of its own,
// three stages deep.  Within a warp every lane owns the same few channels of all keys, so
// shared memory is read without conflicts and the queries stay in registers.  The 32
// lanes' partial dots of 8 keys and up to 4 rows are added by halving exchanges (31
// shuffles for 32 sums), which leave lane 4 k + r with the score of key k and row r: the
// softmax then costs one maximum and one exponential per lane.  The number of rows is a
// compile-time 1, 2, 4 or 8.
//
// 24 single tokens of 12 heads (each its own keys) of 128 channels over up to 4096 keys, window
// 2048: 83 us, 6.2 TB/s, of 78 for a copy of the same bytes.
#include "paged_attention.cuh"
#include "paged_mma.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kKeys = 8;  // keys per tile
constexpr uint32_t kStages = 3;

template <uint32_t HD>
struct Few32 {
    static constexpr uint32_t kRowBytes = HD * 4u;
    static constexpr uint32_t kTileBytes = kKeys * kRowBytes;
    static constexpr uint32_t kStageBytes = 2u * kTileBytes;
    static constexpr uint32_t kSmem = kWarps * kStages * kStageBytes;
    static constexpr uint32_t kDims = HD / 32u;  // channels of a lane
};

// A lane's channels of a row: HD / 32 of them, in pieces of 16 (8) bytes.
template <uint32_t HD>
__device__ __forceinline__ void load_dims(const uint8_t* row, uint32_t lane, float (&x)[HD / 32]) {
    if constexpr (HD == 64) {
        const float2 v = *reinterpret_cast<const float2*>(row + lane * 8u);
        x[0] = v.x;
        x[1] = v.y;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < HD / 128; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(row + i * 512u + lane * 16u);
            x[4 * i] = v.x;
            x[4 * i + 1] = v.y;
            x[4 * i + 2] = v.z;
            x[4 * i + 3] = v.w;
        }
    }
}
// First channel of the lane's piece i (pieces of 4 channels, 2 for heads of 64).
template <uint32_t HD>
__device__ __forceinline__ uint32_t dim_of(uint32_t lane, uint32_t i) {
    return HD == 64 ? lane * 2u + i : (i / 4u) * 128u + lane * 4u + (i & 3u);
}

// a and b summed with the lane `mask` away, which keeps b's sum where this one keeps a's:
// the lanes with `up` get the sum of b.
__device__ __forceinline__ float exchange(float a, float b, bool up, uint32_t mask) {
    const float keep = up ? b : a, send = up ? a : b;
    return keep + __shfl_xor_sync(0xFFFFFFFFu, send, mask);
}

template <uint32_t HD, uint32_t R>
__device__ __forceinline__ void attention_few32(const AttnArgs& a) {
    using F = Few32<HD>;
    constexpr uint32_t kD = F::kDims;
    constexpr uint32_t kGroup = R < 4u ? R : 4u;   // rows whose sums are exchanged together
    constexpr uint32_t kVals = R / kGroup;         // scores a lane ends up with
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint32_t row_tok[kFewRows], row_head[kFewRows];
    __shared__ int row_pos[kFewRows];
    __shared__ float wm[kWarps][kFewRows], wl[kWarps][kFewRows];
    __shared__ uint32_t list[kMaxPicks];
    const uint32_t hd = a.kv.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    FewItem it;
    if (!few_setup<kFewRows>(a, row_tok, row_head, row_pos, list, &it)) return;
    const uint32_t kb = it.kb, ke = it.ke, kh = it.kh;
    // this warp's tiles: tile i starts at key j0 + 8 (4 i + warp); lane i holds the pages of
    // tiles i and i + 32 and the positions of their first keys
    const uint32_t j0 = kb & ~(kKeys - 1u);
    const uint32_t ntiles_all = kb < ke ? (ke - j0 + kKeys - 1u) / kKeys : 0u;
    const uint32_t ntiles = ntiles_all > warp ? (ntiles_all - warp + kWarps - 1u) / kWarps : 0u;
    uint32_t my_page[2] = {kNone, kNone}, my_pos[2] = {0u, 0u};
#pragma unroll
    for (uint32_t u = 0; u < 2u; ++u) {
        if (lane + 32u * u >= ntiles) continue;
        const uint32_t j = j0 + kKeys * (kWarps * (lane + 32u * u) + warp);
        const uint32_t lp = a.part == kPartBlocks ? list[j >> a.kv.page_shift] : j >> a.kv.page_shift;
        if (lp != kNone) {
            my_pos[u] = (lp << a.kv.page_shift) + (j & (a.kv.page_size - 1u));
            // a list's last page may reach beyond the sequence
            if (a.part != kPartBlocks || my_pos[u] <= static_cast<uint32_t>(row_pos[0]))
                my_page[u] = load_page(a.b, a.kv, it.s, lp, a.st);
        }
    }
    auto page_of = [&](uint32_t i) { return __shfl_sync(0xFFFFFFFFu, i < 32u ? my_page[0] : my_page[1], i & 31u); };
    auto pos_of = [&](uint32_t i) { return __shfl_sync(0xFFFFFFFFu, i < 32u ? my_pos[0] : my_pos[1], i & 31u); };
    uint8_t* my_ring = ring + warp * kStages * F::kStageBytes;
    const uint32_t ring_addr = smem_addr(my_ring);
    if (hd < HD) {  // channels beyond the head stay zero
        for (uint32_t i = lane; i < kStages * F::kStageBytes / 16u; i += 32u)
            reinterpret_cast<uint4*>(my_ring)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncwarp();
    }
    const uint32_t chunks16 = hd >> 2;
    const float* kbase = static_cast<const float*>(a.kv.k);
    const float* vbase = static_cast<const float*>(a.kv.v);
    auto fetch = [&](uint32_t i) {
        if (i < ntiles) {
            const uint32_t page = page_of(i), pos = pos_of(i);
            const uint32_t dst = ring_addr + (i % kStages) * F::kStageBytes;
            const size_t off = ((static_cast<size_t>(page == kNone ? 0u : page) * a.kv.kv_heads + kh) * a.kv.page_size +
                                (pos & (a.kv.page_size - 1u))) * hd;
            const uint32_t lo = a.part == kPartBlocks ? 0u : kb;
            const uint32_t hi = page == kNone ? 0u : a.part == kPartBlocks ? static_cast<uint32_t>(row_pos[0]) + 1u : ke;
#pragma unroll
            for (uint32_t x = lane; x < kKeys * (HD / 4u); x += 32u) {
                const uint32_t r = x / (HD / 4u), ch = x % (HD / 4u);
                if (ch >= chunks16) continue;
                const uint32_t bytes = pos + r >= lo && pos + r < hi ? 16u : 0u;
                const size_t o = off + static_cast<size_t>(bytes ? r : 0u) * hd + ch * 4u;
                cp_async16(dst + r * F::kRowBytes + ch * 16u, kbase + o, bytes);
                cp_async16(dst + F::kTileBytes + r * F::kRowBytes + ch * 16u, vbase + o, bytes);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (uint32_t i = 0; i + 1u < kStages; ++i) fetch(i);

    float q[R][kD], acc[R][kD];
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
        const float* src = a.q + (static_cast<size_t>(row_tok[r]) * a.heads + row_head[r]) * hd;
#pragma unroll
        for (uint32_t i = 0; i < kD; ++i) {
            const uint32_t d = dim_of<HD>(lane, i);
            q[r][i] = row_pos[r] >= 0 && d < hd ? src[d] * a.scale_log2 : 0.f;
            acc[r][i] = 0.f;
        }
    }
    // this lane's scores: key lane / 4 of the tile, rows row_of(0 .. kVals - 1)
    auto row_of = [&](uint32_t i) -> uint32_t {
        return R >= 4u ? i * 4u + (lane & 3u) : R == 2u ? (lane >> 1) & 1u : 0u;
    };
    float m[kVals], l[kVals];
    uint32_t lo_key[kVals], hi_key[kVals];
#pragma unroll
    for (uint32_t i = 0; i < kVals; ++i) {
        const int p = row_pos[row_of(i)];
        lo_key[i] = p >= 0 ? first_key(p, a.window) : kNone;
        hi_key[i] = p >= 0 ? static_cast<uint32_t>(p) + 1u : 0u;
        m[i] = -INFINITY;
        l[i] = 0.f;
    }

    for (uint32_t t = 0; t < ntiles; ++t) {
        fetch(t + kStages - 1u);
        cp_wait<kStages - 1>();
        __syncwarp();
        const uint8_t* ks = my_ring + (t % kStages) * F::kStageBytes;
        const uint8_t* vs = ks + F::kTileBytes;
        const uint32_t page = page_of(t), pos = pos_of(t);
        const bool whole = page != kNone && pos >= it.all_b && pos + kKeys <= it.all_e;
        float sc[kVals];
#pragma unroll
        for (uint32_t i = 0; i < kVals; ++i) {
            float v[kGroup][kKeys];
#pragma unroll
            for (uint32_t k = 0; k < kKeys; ++k) {
                float x[kD];
                load_dims<HD>(ks + k * F::kRowBytes, lane, x);
#pragma unroll
                for (uint32_t r = 0; r < kGroup; ++r) {
                    float sum = x[0] * q[i * 4u + r][0];
#pragma unroll
                    for (uint32_t d = 1; d < kD; ++d) sum = fmaf(x[d], q[i * 4u + r][d], sum);
                    v[r][k] = sum;
                }
            }
            float u[kGroup];
#pragma unroll
            for (uint32_t r = 0; r < kGroup; ++r) {
                float w[4], y[2];
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) w[k] = exchange(v[r][k], v[r][k + 4], lane & 16u, 16u);
#pragma unroll
                for (uint32_t k = 0; k < 2; ++k) y[k] = exchange(w[k], w[k + 2], lane & 8u, 8u);
                u[r] = exchange(y[0], y[1], lane & 4u, 4u);
            }
            if constexpr (kGroup == 4u) {
                const float a0 = exchange(u[0], u[2], lane & 2u, 2u), a1 = exchange(u[1], u[3], lane & 2u, 2u);
                sc[i] = exchange(a0, a1, lane & 1u, 1u);
            } else if constexpr (kGroup == 2u) {
                sc[i] = exchange(u[0], u[1], lane & 2u, 2u);
                sc[i] += __shfl_xor_sync(0xFFFFFFFFu, sc[i], 1);
            } else {
                sc[i] = u[0] + __shfl_xor_sync(0xFFFFFFFFu, u[0], 2);
                sc[i] += __shfl_xor_sync(0xFFFFFFFFu, sc[i], 1);
            }
        }
        uint32_t seen[kVals];
        float alpha[kVals];
        bool more = false;
#pragma unroll
        for (uint32_t i = 0; i < kVals; ++i) {
            const uint32_t key = pos + (lane >> 2);
            const bool see = whole || (page != kNone && key >= lo_key[i] && key < hi_key[i]);
            seen[i] = whole ? 0xFFFFFFFFu : __ballot_sync(0xFFFFFFFFu, see);
            if (!see) sc[i] = -INFINITY;
            float mt = sc[i];
            mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 4));
            mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 8));
            mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 16));
            more |= mt > m[i];
            const float mn = fmaxf(m[i], mt);
            alpha[i] = mn == -INFINITY ? 1.f : exp2_fast(m[i] - mn);
            m[i] = mn;
            sc[i] = exp2_fast(sc[i] - (mn == -INFINITY ? 0.f : mn));
            l[i] = fmaf(l[i], alpha[i], sc[i]);
        }
        if (__any_sync(0xFFFFFFFFu, more)) {
#pragma unroll
            for (uint32_t r = 0; r < R; ++r) {
                const float al = __shfl_sync(0xFFFFFFFFu, alpha[r / 4u], R == 2u ? r * 2u : r & 3u);
#pragma unroll
                for (uint32_t d = 0; d < kD; ++d) acc[r][d] *= al;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kKeys; ++k) {
            float x[kD];
            load_dims<HD>(vs + k * F::kRowBytes, lane, x);
#pragma unroll
            for (uint32_t r = 0; r < R; ++r) {
                const uint32_t from = k * 4u + (R == 2u ? r * 2u : r & 3u);
                const float w = __shfl_sync(0xFFFFFFFFu, sc[r / 4u], from);
                if (whole || (seen[r / 4u] >> from & 1u)) {  // an unseen value never enters (0 * inf)
#pragma unroll
                    for (uint32_t d = 0; d < kD; ++d) acc[r][d] = fmaf(w, x[d], acc[r][d]);
                }
            }
        }
        __syncwarp();
    }
    cp_wait<0>();
    asm volatile("griddepcontrol.launch_dependents;");  // the combining kernel may come up
    // the warps' sums, in warp order
#pragma unroll
    for (uint32_t i = 0; i < kVals; ++i) {
        l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 4);
        l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 8);
        l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 16);
        if (lane < 4u) {
            wm[warp][row_of(i)] = m[i] == -INFINITY ? 0.f : m[i];
            wl[warp][row_of(i)] = row_pos[row_of(i)] >= 0 ? l[i] : 0.f;  // padding sees nothing
        }
    }
    if (lane >= R && lane < kFewRows) wl[warp][lane] = 0.f;
    __syncthreads();
    float* part = reinterpret_cast<float*>(ring);  // [warp][row][HD + 4]
    constexpr uint32_t kPitch = HD + 4u;
#pragma unroll
    for (uint32_t r = 0; r < R; ++r)
#pragma unroll
        for (uint32_t d = 0; d < kD; ++d) part[(warp * kFewRows + r) * kPitch + dim_of<HD>(lane, d)] = acc[r][d];
    __syncthreads();
    few_finish<kWarps, kFewRows>(a, it.c, row_tok, row_head, row_pos, wm, wl, part, kPitch);
}

template <uint32_t HD, uint32_t R>
__global__ void __launch_bounds__(kThreads, HD == 256 ? 1 : 2) attention_few32_kernel(const __grid_constant__ AttnArgs a) {
    attention_few32<HD, R>(a);
    end_after_previous(a);
}

template <uint32_t HD, uint32_t R>
cudaError_t launch(const AttnArgs& a, uint64_t items, cudaStream_t stream) {
    return launch_items(a, attention_few32_kernel<HD, R>, items, kThreads, Few32<HD>::kSmem, stream, a);
}

template <uint32_t HD>
cudaError_t launch(const AttnArgs& a, uint32_t rows, uint64_t items, cudaStream_t stream) {
    if (rows <= 1u) return launch<HD, 1>(a, items, stream);
    if (rows <= 2u) return launch<HD, 2>(a, items, stream);
    if (rows <= 4u) return launch<HD, 4>(a, items, stream);
    return launch<HD, 8>(a, items, stream);
}

}  // namespace

cudaError_t launch_attention_few32(const AttnArgs& a, uint32_t max_rows, uint64_t items, cudaStream_t stream) {
    if (a.kv.head_dim <= 64u) return launch<64>(a, max_rows, items, stream);
    if (a.kv.head_dim <= 128u) return launch<128>(a, max_rows, items, stream);
    return launch<256>(a, max_rows, items, stream);
}

}  // namespace nedo_gpu

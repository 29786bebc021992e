// kv_append.cu -- the new tokens' keys and values into a paged cache, with the
// position rotation of queries and keys applied on the way (the RoPE and
// cache-write steps of src/model.cpp:218-225 and src/kernels.cpp:93-105, for a
// ragged batch over pages).
//
// Token row t of sequence s stands at position p = kv_len[s] - (q_start[s+1] - t).
// Channel pair (i, i + hd/2) of a query or key head turns by p * theta^(-2i/hd).
// The angle is formed in 64 bits, as a fraction of a turn: p * frequency loses
// nothing that matters at any position (32 bits are 1e-3 of a turn off at position
// 10^5), and the sine and cosine of the remaining fraction are taken in 32 bits.
//
// One launch with two kinds of CTAs, bound by the copies, and for single tokens by the launch
// and three dependent loads.
//   * Rows: a CTA takes one or four token rows and up to 256 pieces of 16 bytes of each (a
//     piece pair of a query head, a piece of a value), one per thread, so that a thread's loads
//     are all on their way before the first is used, and before the rows' sequences and pages
//     are known; their sines and cosines are computed once for the CTA.
//   * Keys, where a sequence can have several new tokens: a CTA takes one page that the call
//     writes and one KV head, because the minimum and maximum of the page's channels over the
//     new tokens need them in one place (the tokens spread over the thread groups, one round of
//     loads for a page of 64).  With one token per sequence they are pieces of its row.
#include <algorithm>

#include "paged.cuh"

namespace nedo_gpu {
namespace {

constexpr uint32_t kMaxRows = 4;  // token rows of a query CTA

struct AppendArgs {
    PagedKv kv;
    PagedBatch b;
    const float* qkv;
    float* q_out;
    double log2_theta;
    uint32_t heads, rotate;
    uint32_t segs;      // pages that a sequence's new tokens can touch
    uint32_t key_ctas;  // CTAs of the first kind
    uint32_t rows;      // token rows of a CTA of the other kind
    uint32_t pieces, blocks;  // 16-byte pieces (pairs) of a row, and CTAs that share them
    uint32_t row_keys;  // the keys are pieces of their rows
    DeviceStatus* st;
};

// Turns per position of channel pair i.
__device__ __forceinline__ double turns_of(const AppendArgs& a, uint32_t i) {
    return exp2(-2.0 * i / a.kv.head_dim * a.log2_theta) * 0.15915494309189535;  // 1 / (2 pi)
}
// Cosine and sine of position p's rotation.
__device__ __forceinline__ float2 rotation(int p, double turns) {
    double turn = static_cast<double>(p) * turns;
    turn -= rint(turn);
    // what the fraction loses in 32 bits turns the result by the rest of the angle
    const float f = static_cast<float>(turn), rest = static_cast<float>((turn - f) * 6.283185307179586);
    float c, s;
    sincospif(2.f * f, &s, &c);
    return make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
}
__device__ __forceinline__ void rotate4(float4& x, float4& y, const float2* c) {
    const float4 u = x, w = y;
    x = make_float4(u.x * c[0].x - w.x * c[0].y, u.y * c[1].x - w.y * c[1].y, u.z * c[2].x - w.z * c[2].y,
                    u.w * c[3].x - w.w * c[3].y);
    y = make_float4(u.x * c[0].y + w.x * c[0].x, u.y * c[1].y + w.y * c[1].x, u.z * c[2].y + w.z * c[2].x,
                    u.w * c[3].y + w.w * c[3].x);
}
// Four values into the cache, and what they are there.
__device__ __forceinline__ void store4(float* dst, float4& x) { *reinterpret_cast<float4*>(dst) = x; }
__device__ __forceinline__ void store4(__half* dst, float4& x) {
    __half2 h[2] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(h);
    const float2 lo = __half22float2(h[0]), hi = __half22float2(h[1]);
    x = make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ __forceinline__ float4 min4(const float4& a, const float4& b) {
    return make_float4(fminf(a.x, b.x), fminf(a.y, b.y), fminf(a.z, b.z), fminf(a.w, b.w));
}
__device__ __forceinline__ float4 max4(const float4& a, const float4& b) {
    return make_float4(fmaxf(a.x, b.x), fmaxf(a.y, b.y), fmaxf(a.z, b.z), fmaxf(a.w, b.w));
}

// The keys of one page and KV head, and its bounds (fminf / fmaxf leave NaN out).  A page
// whose first slot is written begins anew.
template <typename T>
__device__ void append_keys(const AppendArgs& a, float4* sums) {
    const uint32_t h = blockIdx.x % a.kv.kv_heads, i = blockIdx.x / a.kv.kv_heads, s = i / a.segs, seg = i % a.segs;
    const PagedSeq sq = load_seq(a.b, s, a.st);
    const uint32_t fresh = min(sq.n, sq.kv);  // rows that are tokens
    if (fresh == 0u) return;
    const uint32_t begin = sq.kv - fresh, lp = (begin >> a.kv.page_shift) + seg, first = lp << a.kv.page_shift;
    if (first >= sq.kv) return;
    const uint32_t page = load_page(a.b, a.kv, s, lp, a.st);
    if (page == kNone) return;
    const uint32_t j0 = first < begin ? begin - first : 0u, j1 = min(sq.kv - first, a.kv.page_size);
    const uint32_t hd = a.kv.head_dim, half = hd / 2u, quads = half / 4u, width = (a.heads + 2u * a.kv.kv_heads) * hd;
    const uint32_t groups = blockDim.x / quads, g = threadIdx.x / quads, d = (threadIdx.x - g * quads) * 4u;
    const float* src = a.qkv + static_cast<size_t>(a.heads + h) * hd + d;
    const size_t head = static_cast<size_t>(page) * a.kv.kv_heads + h;
    T* dst = static_cast<T*>(a.kv.k) + head * a.kv.page_size * hd + d;
    float4 lo[2], hi[2];
    lo[0] = lo[1] = make_float4(INFINITY, INFINITY, INFINITY, INFINITY);
    hi[0] = hi[1] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (g < groups) {
        double turns[4];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) turns[e] = a.rotate ? turns_of(a, d + e) : 0.0;
#pragma unroll 4
        for (uint32_t j = j0 + g; j < j1; j += groups) {
            const uint32_t p = first + j;
            const float* row = src + static_cast<size_t>(sq.t0 + sq.n - (sq.kv - p)) * width;
            float4 x = *reinterpret_cast<const float4*>(row), y = *reinterpret_cast<const float4*>(row + half);
            if (a.rotate) {
                float2 c[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) c[e] = rotation(static_cast<int>(p), turns[e]);
                rotate4(x, y, c);
            }
            store4(dst + static_cast<size_t>(j) * hd, x);
            store4(dst + static_cast<size_t>(j) * hd + half, y);
            lo[0] = min4(lo[0], x);
            lo[1] = min4(lo[1], y);
            hi[0] = max4(hi[0], x);
            hi[1] = max4(hi[1], y);
        }
    }
    if (a.kv.bounds == nullptr) return;
    // the groups' extremes meet, by halves
    float4* mine = sums + threadIdx.x * 4u;
    mine[0] = lo[0];
    mine[1] = lo[1];
    mine[2] = hi[0];
    mine[3] = hi[1];
    for (uint32_t n = min(groups, j1 - j0); n > 1u; n = (n + 1u) / 2u) {
        __syncthreads();
        const uint32_t from = g + (n + 1u) / 2u;
        if (from < n) {
            const float4* other = sums + (threadIdx.x + (from - g) * quads) * 4u;
            mine[0] = lo[0] = min4(lo[0], other[0]);
            mine[1] = lo[1] = min4(lo[1], other[1]);
            mine[2] = hi[0] = max4(hi[0], other[2]);
            mine[3] = hi[1] = max4(hi[1], other[3]);
        }
    }
    if (g != 0u) return;
    T* bo = static_cast<T*>(a.kv.bounds) + head * 2u * hd + d;
    if (j0 != 0u) {
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            const T* o = bo + k * half;
            lo[k] = min4(lo[k], make_float4(kv_float(o[0]), kv_float(o[1]), kv_float(o[2]), kv_float(o[3])));
            hi[k] = max4(hi[k], make_float4(kv_float(o[hd]), kv_float(o[hd + 1]), kv_float(o[hd + 2]), kv_float(o[hd + 3])));
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
        store4(bo + k * half, lo[k]);
        store4(bo + hd + k * half, hi[k]);
    }
}

// One piece of ROWS token rows per thread: of the query heads, of the keys (a.row_keys), of the
// values.
template <typename T, uint32_t ROWS>
__device__ void append_rows(const AppendArgs& a, float2 (*cs)[128]) {
    __shared__ int row_pos[kMaxRows];
    __shared__ uint32_t row_page[kMaxRows];
    const uint32_t item = blockIdx.x - a.key_ctas, t0 = item / a.blocks * ROWS, tid = threadIdx.x, nt = blockDim.x;
    const uint32_t hd = a.kv.head_dim, half = hd / 2u, kvh = a.kv.kv_heads, quads = half / 4u;
    const uint32_t piece = item % a.blocks * nt + tid, turned = (a.heads + (a.row_keys ? kvh : 0u)) * quads;
    const bool turns = piece < turned, there = piece < a.pieces;
    // where the piece is in its row: a pair of pieces half a head apart, or one of the values
    const uint32_t h = piece / quads, d = (piece - h * quads) * 4u;
    const uint32_t off = turns ? h * hd + d : (a.heads + kvh) * hd + (piece - turned) * 4u;
    const size_t width = static_cast<size_t>(a.heads + 2u * kvh) * hd;
    float4 x[ROWS], y[ROWS];
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        x[r] = y[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!there || t0 + r >= a.b.tokens) continue;
        const float* src = a.qkv + (t0 + r) * width + off;
        x[r] = __ldg(reinterpret_cast<const float4*>(src));
        if (turns) y[r] = __ldg(reinterpret_cast<const float4*>(src + half));
    }
    const uint32_t mine = nt - 1u - tid;  // by the last threads: the first ones form the powers meanwhile
    if (mine < ROWS) {
        int p = -1;
        uint32_t page = kNone;
        if (t0 + mine < a.b.tokens) {
            const uint32_t s = seq_of_token(a.b, t0 + mine);
            if (s != kNone) {
                const PagedSeq sq = load_seq(a.b, s, a.st);
                if (sq.n != 0u) p = sq.pos(t0 + mine - sq.t0);
                if (p >= 0) page = load_page(a.b, a.kv, s, static_cast<uint32_t>(p) >> a.kv.page_shift, a.st);
            }
        }
        row_pos[mine] = p;
        row_page[mine] = page;
    }
    if (a.rotate) {
        // a thread takes one channel pair of its rows: its power once, ahead of the positions
        // (a power for each row and pair took prompts from 13.9 to 14.8 us)
        const uint32_t k = tid % half, groups = min(nt / half, ROWS);
        const double turns_k = tid < groups * half ? turns_of(a, k) : 0.0;
        __syncthreads();
        for (uint32_t r = tid / half; r < ROWS && tid < groups * half; r += groups)
            if (row_pos[r] >= 0) cs[r][k] = rotation(row_pos[r], turns_k);
    }
    __syncthreads();
    if (!there) return;
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        const int p = row_pos[r];
        if (p < 0) continue;
        if (turns && a.rotate) rotate4(x[r], y[r], &cs[r][d]);
        if (piece < a.heads * quads) {
            float* o = a.q_out + (static_cast<size_t>(t0 + r) * a.heads + h) * hd + d;
            *reinterpret_cast<float4*>(o) = x[r];
            *reinterpret_cast<float4*>(o + half) = y[r];
        } else if (row_page[r] != kNone) {
            const uint32_t e = (piece - turned) * 4u, kh = turns ? h - a.heads : e / hd;
            const size_t head = static_cast<size_t>(row_page[r]) * kvh + kh;
            const uint32_t slot = static_cast<uint32_t>(p) & (a.kv.page_size - 1u);
            if (!turns) {
                store4(static_cast<T*>(a.kv.v) + (head * a.kv.page_size + slot) * hd + (e - kh * hd), x[r]);
                continue;
            }
            T* dst = static_cast<T*>(a.kv.k) + (head * a.kv.page_size + slot) * hd + d;
            store4(dst, x[r]);
            store4(dst + half, y[r]);
            if (a.kv.bounds == nullptr) continue;
            T* bo = static_cast<T*>(a.kv.bounds) + head * 2u * hd + d;
#pragma unroll
            for (uint32_t k = 0; k < 2u; ++k) {
                const float4 v = k ? y[r] : x[r], none = make_float4(INFINITY, INFINITY, INFINITY, INFINITY);
                const float4 least = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                T* o = bo + k * half;
                float4 lo = min4(none, v), hi = max4(least, v);
                if (slot != 0u) {  // a page whose first slot is written begins anew
                    lo = min4(lo, make_float4(kv_float(o[0]), kv_float(o[1]), kv_float(o[2]), kv_float(o[3])));
                    hi = max4(hi, make_float4(kv_float(o[hd]), kv_float(o[hd + 1]), kv_float(o[hd + 2]), kv_float(o[hd + 3])));
                }
                store4(o, lo);
                store4(o + hd, hi);
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) kv_append_kernel(AppendArgs a) {
    __shared__ __align__(16) uint8_t sm[256 * 4 * sizeof(float4)];
    if (blockIdx.x < a.key_ctas) append_keys<T>(a, reinterpret_cast<float4*>(sm));
    else if (a.rows == 1u) append_rows<T, 1>(a, reinterpret_cast<float2(*)[128]>(sm));
    else append_rows<T, kMaxRows>(a, reinterpret_cast<float2(*)[128]>(sm));
}

}  // namespace

cudaError_t launch_kv_append(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* qkv, double theta,
                             float* q_out, DeviceStatus* st, cudaStream_t stream) {
    AppendArgs a = {};
    a.kv = kv;
    a.b = b;
    a.qkv = qkv;
    a.q_out = q_out;
    a.rotate = theta > 0.0;
    a.log2_theta = a.rotate ? log2(theta) : 0.0;
    a.heads = heads;
    a.segs = (b.max_q_len + kv.page_size - 2u) / kv.page_size + 1u;
    a.rows = b.tokens >= 4u * 148u ? kMaxRows : 1u;  // four rows share their sines where there are CTAs enough
    a.row_keys = b.max_q_len <= 1u;
    const uint32_t quads = kv.head_dim / 8u;
    a.pieces = (heads + (a.row_keys ? kv.kv_heads : 0u)) * quads + kv.kv_heads * kv.head_dim / 4u;
    a.blocks = (a.pieces + 255u) / 256u;
    // a thread for every piece, and for every channel pair
    const uint32_t threads = (std::max((a.pieces + a.blocks - 1u) / a.blocks, kv.head_dim / 2u) + 31u) / 32u * 32u;
    a.st = st;
    const uint64_t keys = a.row_keys ? 0u : static_cast<uint64_t>(b.seqs) * a.segs * kv.kv_heads;
    const uint64_t grid = keys + static_cast<uint64_t>((b.tokens + a.rows - 1u) / a.rows) * a.blocks;
    if (grid > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    a.key_ctas = static_cast<uint32_t>(keys);
    if (kv.type == kF16) kv_append_kernel<__half><<<static_cast<uint32_t>(grid), threads, 0, stream>>>(a);
    else kv_append_kernel<float><<<static_cast<uint32_t>(grid), threads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace nedo_gpu

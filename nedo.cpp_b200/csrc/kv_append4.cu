// kv_append4.cu -- the new tokens' keys and values into a paged Q4_0 cache (paged_q4.cuh), with the
// position rotation of queries and keys on the way, and the tokens' keys and values out of a cache.
//
// A block of 32 channels becomes numbers n and a scale d:
//   d = -x / 8 for the number x of largest magnitude (the negative one where both signs reach it),
//       in eight significant bits, to the nearest (even) one, in steps of no less than 2^-24 and
//       with a magnitude of at most 8160 = 255 * 2^5;
//   n = floor(x / d + 8.5) within 0..15, 8 where d is 0;
// and the scale NaN where a number of it is not finite.  A rounding error in x moves n by a whole
// step where x is next to a border of two, so nothing is rounded on the way: keys turn in 64 bits,
// by angles, sines and cosines of 64 bits, and n, found with a reciprocal, is set right by comparing x
// with the products d (n - 8.5), which are exact.
//
// One launch with two kinds of CTAs, as over F16 and F32 caches: rows (pieces of queries and values,
// and of keys where no sequence has several new tokens), and pages of keys, whose bounds need the
// page's new tokens in one place.  A thread takes four channels of a token, eight neighbouring threads
// a block, which agree on its extremes by shuffles.  Over the tokens of a page a thread's sines and
// cosines follow from its first token's by a fixed turn, in 64 bits as well: one pair of them for a
// channel instead of one for a channel and token, and what 15 products lose is some 2^-49.
#include "kv_append.cuh"
#include "paged_q4.cuh"

namespace nedo_gpu {
namespace {

// Cosine and sine of position p's rotation in 64 bits.
__device__ __forceinline__ double2 rotation64(double p, double turns) {
    double turn = p * turns, c, s;
    turn -= rint(turn);
    sincospi(2.0 * turn, &s, &c);
    return make_double2(c, s);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
__device__ __forceinline__ bool finite(double x) { return fabs(x) < static_cast<double>(INFINITY); }
__device__ __forceinline__ float least(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double least(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float below(float x) { return floorf(x); }
__device__ __forceinline__ double below(double x) { return floor(x); }

// An eighth of a magnitude as a scale.
__device__ __forceinline__ float scale_of(double size) {
    const double d = size * 0.125;
    // the exponent of d, of its eighth bit, and no less than -24
    const int e = max(static_cast<int>(__double_as_longlong(d) >> 52) - 1023 - 7, -24);
    const double step = __longlong_as_double(static_cast<long long>(1023 + e) << 52);
    const double up = __longlong_as_double(static_cast<long long>(1023 - e) << 52);
    return static_cast<float>(fmin(rint(d * up) * step, 8160.0));
}

// Four numbers of a block of 32, which eight neighbouring lanes have: the block's numbers to `words`
// and its scale to `scale`, and what the cache then holds for the four.
template <typename X>
__device__ __forceinline__ float4 store_block(const X (&x)[4], uint32_t* words, __half* scale) {
    const uint32_t lane = threadIdx.x & 31u, eight = 0xFFu << (lane & 24u);
    X lo = least(least(x[0], x[1]), least(x[2], x[3])), hi = most(most(x[0], x[1]), most(x[2], x[3]));
    const bool odd = !(finite(x[0]) && finite(x[1]) && finite(x[2]) && finite(x[3]));
#pragma unroll
    for (uint32_t o = 1; o < 8u; o <<= 1) {
        lo = least(lo, __shfl_xor_sync(eight, lo, o));
        hi = most(hi, __shfl_xor_sync(eight, hi, o));
    }
    const bool bad = (__ballot_sync(eight, odd) & eight) != 0u, negative = -lo >= hi;
    const float d = bad ? 0.f : scale_of(negative ? -lo : hi);
    const X inv = X(1) / X(d);
    uint32_t mine = 0;
    float out[4];
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
        const X v = negative ? x[e] : -x[e];
        X n = below(v * inv + X(8.5));
        n = most(least(n, X(16)), X(-1));
        // the largest n with d (n - 8.5) <= v
        if ((n + X(1) - X(8.5)) * X(d) <= v) n += X(1);
        else if ((n - X(8.5)) * X(d) > v) n -= X(1);
        n = d == 0.f ? X(8) : most(least(n, X(15)), X(0));
        const uint32_t i = static_cast<uint32_t>(static_cast<int>(n));
        mine |= i << ((e & 1u) * 16u + (e >> 1) * 4u);
        out[e] = (negative ? d : -d) * static_cast<float>(static_cast<int>(i) - 8);
    }
    mine <<= (lane & 1u) * 8u;
    mine |= __shfl_xor_sync(eight, mine, 1);
    if ((lane & 1u) == 0u) words[(lane & 7u) >> 1] = mine;
    if ((lane & 7u) == 0u) *scale = bad ? __ushort_as_half(0x7FFF) : __float2half_rn(negative ? d : -d);
    if (bad) out[0] = out[1] = out[2] = out[3] = __int_as_float(0x7FFFFFFF);
    return make_float4(out[0], out[1], out[2], out[3]);
}
// Where channel d's block of a token is, in a page and head at `at`.
__device__ __forceinline__ uint32_t* words_at(const PagedKv& kv, uint8_t* at, uint32_t slot, uint32_t d) {
    return reinterpret_cast<uint32_t*>(at + slot * (kv.head_dim / 2u) + (d >> 5) * 16u);
}
__device__ __forceinline__ __half* scale_at(const PagedKv& kv, uint8_t* at, uint32_t slot, uint32_t d) {
    return reinterpret_cast<__half*>(at + q4_scales_at(kv)) + (d >> 5) * kv.page_size + slot;
}
// The bounds of four channels (fp16: what the cache holds is an fp16 number) taken on to lo and hi.
__device__ __forceinline__ void store_bounds(__half* at, uint32_t hd, float4 lo, float4 hi, bool anew) {
    if (!anew) {
        lo = min4(lo, make_float4(__half2float(at[0]), __half2float(at[1]), __half2float(at[2]), __half2float(at[3])));
        hi = max4(hi, make_float4(__half2float(at[hd]), __half2float(at[hd + 1]), __half2float(at[hd + 2]), __half2float(at[hd + 3])));
    }
    const __half2 l[2] = {__floats2half2_rn(lo.x, lo.y), __floats2half2_rn(lo.z, lo.w)};
    const __half2 h[2] = {__floats2half2_rn(hi.x, hi.y), __floats2half2_rn(hi.z, hi.w)};
    *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(l);
    *reinterpret_cast<uint2*>(at + hd) = *reinterpret_cast<const uint2*>(h);
}

// The turned channels d .. d + 3 of a head's row: with those half a head on (or back) they are pairs.
__device__ __forceinline__ void turned(const float4& x, const float4& other, bool second, const double2 (&c)[4], double (&v)[4]) {
    const double u[4] = {x.x, x.y, x.z, x.w}, w[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) v[e] = second ? w[e] * c[e].y + u[e] * c[e].x : u[e] * c[e].x - w[e] * c[e].y;
}

// The keys of one page and KV head, and its bounds (fminf / fmaxf leave NaN out).  A page whose
// first slot is written begins anew.
__device__ __forceinline__ void append_keys4(const AppendArgs& a, float4* sums) {
    const uint32_t h = blockIdx.x % a.kv.kv_heads, i = blockIdx.x / a.kv.kv_heads, s = i / a.segs, seg = i % a.segs;
    const PagedSeq sq = load_seq(a.b, s, a.st);
    const uint32_t fresh = min(sq.n, sq.kv);  // rows that are tokens
    if (fresh == 0u) return;
    const uint32_t begin = sq.kv - fresh, lp = (begin >> a.kv.page_shift) + seg, first = lp << a.kv.page_shift;
    if (first >= sq.kv) return;
    const uint32_t page = load_page(a.b, a.kv, s, lp, a.st);
    if (page == kNone) return;
    const uint32_t j0 = first < begin ? begin - first : 0u, j1 = min(sq.kv - first, a.kv.page_size);
    const uint32_t hd = a.kv.head_dim, half = hd / 2u, quads = hd / 4u;
    const size_t width = static_cast<size_t>(a.heads + 2u * a.kv.kv_heads) * hd;
    const uint32_t groups = blockDim.x / quads, g = threadIdx.x / quads, d = (threadIdx.x - g * quads) * 4u;
    const bool second = d >= half;
    const size_t head = static_cast<size_t>(page) * a.kv.kv_heads + h;
    uint8_t* const at = static_cast<uint8_t*>(a.kv.k) + head * q4_head_bytes(a.kv);
    float4 lo = make_float4(INFINITY, INFINITY, INFINITY, INFINITY), hi = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (g < groups) {
        const float* src = a.qkv + static_cast<size_t>(a.heads + h) * hd + d;
        const int to = second ? -static_cast<int>(half) : static_cast<int>(half);
        double2 c[4], step[4];
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) {
            c[e] = step[e] = make_double2(1.0, 0.0);
            if (a.rotate && j0 + g < j1) {
                const double turns = turns_of(a, (second ? d - half : d) + e);
                c[e] = rotation64(first + j0 + g, turns);
                if (j0 + g + groups < j1) step[e] = rotation64(groups, turns);
            }
        }
        for (uint32_t j = j0 + g; j < j1; j += groups) {
            const float* row = src + static_cast<size_t>(sq.t0 + sq.n - (sq.kv - (first + j))) * width;
            double v[4];
            // (a pair's other half is read only to turn with it: 0 times infinity is not 0)
            const float4 x = *reinterpret_cast<const float4*>(row);
            if (a.rotate) {
                turned(x, *reinterpret_cast<const float4*>(row + to), second, c, v);
            } else {
                v[0] = x.x;
                v[1] = x.y;
                v[2] = x.z;
                v[3] = x.w;
            }
            const float4 y = store_block(v, words_at(a.kv, at, j, d), scale_at(a.kv, at, j, d));
            lo = min4(lo, y);
            hi = max4(hi, y);
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e)
                c[e] = make_double2(c[e].x * step[e].x - c[e].y * step[e].y, c[e].x * step[e].y + c[e].y * step[e].x);
        }
    }
    if (a.kv.bounds == nullptr) return;
    // the groups' extremes meet, by halves
    float4* mine = sums + threadIdx.x * 2u;
    mine[0] = lo;
    mine[1] = hi;
    for (uint32_t n = min(groups, j1 - j0); n > 1u; n = (n + 1u) / 2u) {
        __syncthreads();
        const uint32_t from = g + (n + 1u) / 2u;
        if (from < n) {
            const float4* other = sums + (threadIdx.x + (from - g) * quads) * 2u;
            mine[0] = lo = min4(lo, other[0]);
            mine[1] = hi = max4(hi, other[1]);
        }
    }
    if (g == 0u) store_bounds(static_cast<__half*>(a.kv.bounds) + head * 2u * hd + d, hd, lo, hi, j0 == 0u);
}

// One piece of ROWS token rows per thread: pairs of pieces of the query heads, then, from a multiple
// of eight threads on, pieces of the keys (a.row_keys) and of the values.
template <uint32_t ROWS>
__device__ __forceinline__ void append_rows4(const AppendArgs& a, float2 (*cs)[128], double2 (*cd)[128]) {
    __shared__ int row_pos[kMaxRows];
    __shared__ uint32_t row_page[kMaxRows];
    const uint32_t item = blockIdx.x - a.key_ctas, t0 = item / a.blocks * ROWS, tid = threadIdx.x, nt = blockDim.x;
    const uint32_t hd = a.kv.head_dim, half = hd / 2u, kvh = a.kv.kv_heads, quads = half / 4u;
    const uint32_t piece = item % a.blocks * nt + tid, q_pieces = a.heads * quads, from = (q_pieces + 7u) & ~7u;
    const bool query = piece < q_pieces, block = piece >= from && piece < a.pieces;
    // where the piece is in its row
    const uint32_t first = (a.row_keys ? a.heads : a.heads + kvh) * hd;  // channel of the first block
    const uint32_t h = query ? piece / quads : 0u;
    const uint32_t off = query ? h * hd + (piece - h * quads) * 4u : block ? first + (piece - from) * 4u : 0u;
    const bool key = block && off < (a.heads + kvh) * hd;
    const uint32_t d = query ? off - h * hd : off % hd;  // channel of its head
    const bool second = key && d >= half;
    const size_t width = static_cast<size_t>(a.heads + 2u * kvh) * hd;
    float4 x[ROWS], y[ROWS];
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        x[r] = y[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if ((!query && !block) || t0 + r >= a.b.tokens) continue;
        const float* src = a.qkv + (t0 + r) * width + off;
        x[r] = __ldg(reinterpret_cast<const float4*>(src));
        if (query || (key && a.rotate)) y[r] = __ldg(reinterpret_cast<const float4*>(second ? src - half : src + half));
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
        const uint32_t k = tid % half, groups = min(nt / half, ROWS);
        const double turns_k = tid < groups * half ? turns_of(a, k) : 0.0;
        __syncthreads();
        for (uint32_t r = tid / half; r < ROWS && tid < groups * half; r += groups) {
            if (row_pos[r] < 0) continue;
            if (a.row_keys) {
                const double2 c = rotation64(row_pos[r], turns_k);
                cd[r][k] = c;
                cs[r][k] = make_float2(static_cast<float>(c.x), static_cast<float>(c.y));
            } else {
                cs[r][k] = rotation(row_pos[r], turns_k);
            }
        }
    }
    __syncthreads();
    if (!query && !block) return;
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        const int p = row_pos[r];
        if (p < 0) continue;
        if (query) {
            if (a.rotate) rotate4(x[r], y[r], &cs[r][d]);
            float* o = a.q_out + (static_cast<size_t>(t0 + r) * a.heads + h) * hd + d;
            *reinterpret_cast<float4*>(o) = x[r];
            *reinterpret_cast<float4*>(o + half) = y[r];
        } else if (row_page[r] != kNone) {
            const uint32_t kh = (off / hd - a.heads) % kvh, slot = static_cast<uint32_t>(p) & (a.kv.page_size - 1u);
            const size_t head = static_cast<size_t>(row_page[r]) * kvh + kh;
            uint8_t* const at = static_cast<uint8_t*>(key ? a.kv.k : a.kv.v) + head * q4_head_bytes(a.kv);
            // (a block's eight threads have the same row, page and kind)
            if (!key || !a.rotate) {
                const float v[4] = {x[r].x, x[r].y, x[r].z, x[r].w};
                x[r] = store_block(v, words_at(a.kv, at, slot, d), scale_at(a.kv, at, slot, d));
            } else {
                double2 c[4];
                double v[4];
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) c[e] = cd[r][(second ? d - half : d) + e];
                turned(x[r], y[r], second, c, v);
                x[r] = store_block(v, words_at(a.kv, at, slot, d), scale_at(a.kv, at, slot, d));
            }
            if (key && a.kv.bounds != nullptr) {
                const float4 none = make_float4(INFINITY, INFINITY, INFINITY, INFINITY);
                const float4 least = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                store_bounds(static_cast<__half*>(a.kv.bounds) + head * 2u * hd + d, hd, min4(none, x[r]), max4(least, x[r]), slot == 0u);
            }
        }
    }
}

__global__ void __launch_bounds__(256) kv_append4_kernel(AppendArgs a) {
    __shared__ __align__(16) uint8_t sm[kMaxRows * 128 * (sizeof(float2) + sizeof(double2))];  // 12 KB
    if (blockIdx.x < a.key_ctas) append_keys4(a, reinterpret_cast<float4*>(sm));               // 256 * 32 bytes of it
    else if (a.rows == 1u) append_rows4<1>(a, reinterpret_cast<float2(*)[128]>(sm + kMaxRows * 128 * sizeof(double2)), reinterpret_cast<double2(*)[128]>(sm));
    else append_rows4<kMaxRows>(a, reinterpret_cast<float2(*)[128]>(sm + kMaxRows * 128 * sizeof(double2)), reinterpret_cast<double2(*)[128]>(sm));
}

// ---- reading ------------------------------------------------------------------
struct ReadArgs {
    PagedKv kv;
    PagedBatch b;
    float *k, *v;
    uint32_t pieces, blocks;  // pieces of eight channels of a row (keys, then values), CTAs that share them
    DeviceStatus* st;
};

// Eight channels of a token's keys or values per thread.
__global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
    const uint32_t t = blockIdx.x / a.blocks, piece = blockIdx.x % a.blocks * blockDim.x + threadIdx.x;
    if (piece >= a.pieces) return;
    const uint32_t s = seq_of_token(a.b, t);
    if (s == kNone) return;
    const PagedSeq sq = load_seq(a.b, s, a.st);
    if (sq.n == 0u) return;
    const int p = sq.pos(t - sq.t0);
    const uint32_t hd = a.kv.head_dim, kvh = a.kv.kv_heads, row = kvh * hd;
    const bool values = piece * 8u >= row;
    const uint32_t e = piece * 8u - (values ? row : 0u), kh = e / hd, d = e - kh * hd;
    float4 x[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    const uint32_t page = p >= 0 ? load_page(a.b, a.kv, s, static_cast<uint32_t>(p) >> a.kv.page_shift, a.st) : kNone;
    if (page != kNone) {
        const uint32_t slot = static_cast<uint32_t>(p) & (a.kv.page_size - 1u);
        const void* cache = values ? a.kv.v : a.kv.k;
        const size_t head = static_cast<size_t>(page) * kvh + kh, at = (head * a.kv.page_size + slot) * hd + d;
        if (a.kv.type == kF32) {
            x[0] = *reinterpret_cast<const float4*>(static_cast<const float*>(cache) + at);
            x[1] = *reinterpret_cast<const float4*>(static_cast<const float*>(cache) + at + 4u);
        } else {
            __half2 h[4];
            if (a.kv.type == kF16) {
                *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(static_cast<const __half*>(cache) + at);
            } else {
                const uint8_t* from = static_cast<const uint8_t*>(cache) + head * q4_head_bytes(a.kv);
                q4_pairs(*reinterpret_cast<const uint32_t*>(from + slot * (hd / 2u) + (d >> 3) * 4u), h);
                const __half2 scale = __half2half2(q4_scale(a.kv, from, slot, d));
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) h[i] = __hmul2(h[i], scale);
            }
            const float2 f[4] = {__half22float2(h[0]), __half22float2(h[1]), __half22float2(h[2]), __half22float2(h[3])};
            x[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
            x[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
        }
    }
    float* to = (values ? a.v : a.k) + static_cast<size_t>(t) * row + e;
    *reinterpret_cast<float4*>(to) = x[0];
    *reinterpret_cast<float4*>(to + 4u) = x[1];
}

}  // namespace

cudaError_t launch_kv_append4(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* qkv, double theta,
                              float* q_out, DeviceStatus* st, cudaStream_t stream) {
    const uint32_t q_pieces = heads * (kv.head_dim / 8u);
    const AppendLaunch l = append_launch(kv, b, heads, qkv, theta, q_out, st, kv.kv_heads * (kv.head_dim / 4u), (8u - q_pieces % 8u) % 8u);
    if (l.grid > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    kv_append4_kernel<<<static_cast<uint32_t>(l.grid), l.threads, 0, stream>>>(l.a);
    return cudaGetLastError();
}

cudaError_t launch_kv_read(const PagedKv& kv, const PagedBatch& b, float* k, float* v, DeviceStatus* st, cudaStream_t stream) {
    ReadArgs a = {};
    a.kv = kv;
    a.b = b;
    a.k = k;
    a.v = v;
    a.pieces = 2u * kv.kv_heads * (kv.head_dim / 8u);
    a.blocks = (a.pieces + 255u) / 256u;
    a.st = st;
    const uint64_t grid = static_cast<uint64_t>(b.tokens) * a.blocks;
    if (grid > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    const uint32_t threads = ((a.pieces + a.blocks - 1u) / a.blocks + 31u) / 32u * 32u;
    kv_read_kernel<<<static_cast<uint32_t>(grid), threads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace nedo_gpu

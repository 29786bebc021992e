// kv_append4.cu -- the new tokens' keys and values into a paged Q4_0 cache (paged_q4.cuh), with the
// position rotation of queries and keys on the way, and the tokens' keys and values out of a cache.
//
// A block of 32 channels becomes numbers n and a scale d:
//   d = -x / 8 for the number x of largest magnitude (the negative one where both signs reach it),
//       in eight significant bits, to the nearest (even) one, in steps of no less than 2^-24 and
//       with a magnitude of at most 8160 = 255 * 2^5;
//   n = floor(x / d + 8.5) within 0..15, 8 where d is 0;
// and the scale NaN where a number of it is not finite.  A rounding error in x moves n by a whole
// step where x is next to a border of two, so nothing is rounded on the way: angles, sines and cosines of keys are
// formed in 64 bits and the products as pairs of 32-bit numbers, x = hi + lo, exact to some 2^-46 (in 64 bits
// the extremes alone, which have no instruction, took as long as all of this does); and n, found with a
// reciprocal, is set right by comparing x with the product d (n - 8.5), which is exact.
//
// One launch with two kinds of CTAs, as over F16 and F32 caches: rows (pieces of queries and values,
// and of keys where no sequence has several new tokens), and keys: a block of channels of one page,
// because the bounds need the page's new tokens in one place.  A thread takes four channels of a token,
// eight neighbouring threads a block, which agree on its extremes by shuffles.  Over the tokens of a
// page sines and cosines are products of those of every eighth token and those of a token's place among
// eight: a quarter of them at pages of 64.
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

// An eighth of a magnitude as a scale.
__device__ __forceinline__ float scale_of(double size) {
    const double d = size * 0.125;
    // the exponent of d, of its eighth bit, and no less than -24
    const int e = max(static_cast<int>(__double_as_longlong(d) >> 52) - 1023 - 7, -24);
    const double step = __longlong_as_double(static_cast<long long>(1023 + e) << 52);
    const double up = __longlong_as_double(static_cast<long long>(1023 - e) << 52);
    return static_cast<float>(fmin(rint(d * up) * step, 8160.0));
}

// A number as hi + lo, hi the nearest of 32 bits.
struct Pair {
    float hi, lo;
};
__device__ __forceinline__ Pair pair_of(double x) {
    const float hi = static_cast<float>(x);
    return {hi, static_cast<float>(x - hi)};
}
// Four numbers of a block of 32, which eight neighbouring lanes have (LOW: as pairs): the block's numbers to
// `words` and its scale to `scale`, and what the cache then holds for the four.
template <bool LOW>
__device__ __forceinline__ float4 store_block(const Pair (&x)[4], uint32_t* words, __half* scale) {
    const uint32_t lane = threadIdx.x & 31u, eight = 0xFFu << (lane & 24u);
    float low = fminf(fminf(x[0].hi, x[1].hi), fminf(x[2].hi, x[3].hi)), high = fmaxf(fmaxf(x[0].hi, x[1].hi), fmaxf(x[2].hi, x[3].hi));
#pragma unroll
    for (uint32_t o = 1; o < 8u; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(eight, low, o));
        high = fmaxf(high, __shfl_xor_sync(eight, high, o));
    }
    float low2 = 0.f, high2 = 0.f;
    if constexpr (LOW) {
        low2 = INFINITY;
        high2 = -INFINITY;
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) {
            if (x[e].hi == low) low2 = fminf(low2, x[e].lo);
            if (x[e].hi == high) high2 = fmaxf(high2, x[e].lo);
        }
#pragma unroll
        for (uint32_t o = 1; o < 8u; o <<= 1) {
            low2 = fminf(low2, __shfl_xor_sync(eight, low2, o));
            high2 = fmaxf(high2, __shfl_xor_sync(eight, high2, o));
        }
    }
    const float odd = fmaf(x[0].hi, 0.f, fmaf(x[1].hi, 0.f, fmaf(x[2].hi, 0.f, x[3].hi * 0.f)));  // NaN
    const bool bad = (__ballot_sync(eight, odd != 0.f) & eight) != 0u;
    const bool negative = LOW ? -low > high || (-low == high && -low2 >= high2) : -low >= high;
    const double size = negative ? -static_cast<double>(low) - low2 : static_cast<double>(high) + high2;
    const float d = bad ? 0.f : scale_of(size), inv = d == 0.f ? 0.f : 1.f / d;
    const uint32_t sign = negative ? 0u : 0x80000000u;
    uint32_t mine = 0;
    float out[4];
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
        const float v = __uint_as_float(__float_as_uint(x[e].hi) ^ sign);
        // n or the one below it (adding 1.5 2^23 rounds to a whole number), then the largest with
        // d (n - 8.5) <= v
        const float t = fminf(fmaxf(v * inv, -9.f), 9.f) + (8.f - 1.f / 1024.f);
        const float n = (t + 12582912.f) - 12582912.f, next = (n - 7.5f) * d;
        bool up = next <= v;
        if constexpr (LOW) up = next < v || (next == v && __uint_as_float(__float_as_uint(x[e].lo) ^ sign) >= 0.f);
        const float m = d == 0.f ? 8.f : fminf(fmaxf(up ? n + 1.f : n, 0.f), 15.f);
        mine |= (__float_as_uint(m + 8388608.f) & 15u) << ((e & 1u) * 16u + (e >> 1) * 4u);
        out[e] = __uint_as_float(__float_as_uint(d * (m - 8.f)) ^ sign);
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

// Channel u of a head turned by cosine and sine c, with channel w half a head on (or, of the second half,
// back): u c -+ w s as a pair.
__device__ __forceinline__ Pair turned(float u, float w, bool second, double2 c) {
    if (fmaxf(fabsf(u), fabsf(w)) > 1e37f) {  // (what leaves 32 bits has the largest scale, and counts as 3e38)
        const double x = u * c.x + w * (second ? c.y : -c.y);
        return pair_of(fabs(x) < static_cast<double>(INFINITY) ? fmin(fmax(x, -3e38), 3e38) : x);
    }
    const Pair cos = pair_of(c.x), sin = pair_of(second ? c.y : -c.y);
    const float p = u * cos.hi, q = w * sin.hi;
    const float p2 = fmaf(u, cos.lo, fmaf(u, cos.hi, -p)), q2 = fmaf(w, sin.lo, fmaf(w, sin.hi, -q));
    const float s = p + q, r = s - p;
    const float low = ((p - (s - r)) + (q - r)) + (p2 + q2);
    const float hi = s + low;
    return {hi, low - (hi - s)};
}

constexpr uint32_t kEighth = 8;  // tokens that share a sine
// One block of 32 channels of the keys of one page and KV head, and its bounds (fminf / fmaxf leave NaN
// out).  A page whose first slot is written begins anew.
__device__ __forceinline__ void append_keys4(const AppendArgs& a, double2 (*far)[32], double2 (*near)[32], float4* sums) {
    const uint32_t blocks = a.kv.head_dim / 32u, block = blockIdx.x % blocks, x0 = blockIdx.x / blocks;
    const uint32_t h = x0 % a.kv.kv_heads, i = x0 / a.kv.kv_heads, s = i / a.segs, seg = i % a.segs;
    const PagedSeq sq = load_seq(a.b, s, a.st);
    const uint32_t fresh = min(sq.n, sq.kv);  // rows that are tokens
    if (fresh == 0u) return;
    const uint32_t begin = sq.kv - fresh, lp = (begin >> a.kv.page_shift) + seg, first = lp << a.kv.page_shift;
    if (first >= sq.kv) return;
    const uint32_t page = load_page(a.b, a.kv, s, lp, a.st);
    if (page == kNone) return;
    const uint32_t j0 = first < begin ? begin - first : 0u, j1 = min(sq.kv - first, a.kv.page_size);
    const uint32_t hd = a.kv.head_dim, half = hd / 2u, tid = threadIdx.x, groups = blockDim.x / 8u, g = tid / 8u;
    const size_t width = static_cast<size_t>(a.heads + 2u * a.kv.kv_heads) * hd;
    const size_t head = static_cast<size_t>(page) * a.kv.kv_heads + h;
    uint8_t* const at = static_cast<uint8_t*>(a.kv.k) + head * q4_head_bytes(a.kv);
    if (a.rotate) {
        // (a warp: the 32 channels of one place)
        const uint32_t ch = 32u * block + (tid & 31u);
        const double turns = turns_of(a, ch >= half ? ch - half : ch);
        const uint32_t e0 = j0 / kEighth, e1 = (j1 + kEighth - 1u) / kEighth;
        for (uint32_t e = tid / 32u; e < e1 - e0 + kEighth; e += blockDim.x / 32u) {
            if (e < kEighth) near[e][tid & 31u] = rotation64(e, turns);
            else far[e - kEighth][tid & 31u] = rotation64(first + (e0 + e - kEighth) * kEighth, turns);
        }
        __syncthreads();
    }
    float4 lo = make_float4(INFINITY, INFINITY, INFINITY, INFINITY), hi = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    const uint32_t c = (tid & 7u) * 4u, d = 32u * block + c;
    const bool second = d >= half;
    const float* src = a.qkv + static_cast<size_t>(a.heads + h) * hd + d;
    const int to = second ? -static_cast<int>(half) : static_cast<int>(half);
    for (uint32_t j = j0 + g; j < j1; j += groups) {
        const float* row = src + static_cast<size_t>(sq.t0 + sq.n - (sq.kv - (first + j))) * width;
        const float4 x = __ldg(reinterpret_cast<const float4*>(row));
        float4 y;
        if (a.rotate) {
            // (a pair's other half is read only to turn with it: 0 times infinity is not 0)
            const float4 w = __ldg(reinterpret_cast<const float4*>(row + to));
            const double2 *f = far[j / kEighth - j0 / kEighth] + c, *n = near[j % kEighth] + c;
            auto product = [&](uint32_t e) {
                return make_double2(f[e].x * n[e].x - f[e].y * n[e].y, f[e].x * n[e].y + f[e].y * n[e].x);
            };
            const Pair v[4] = {turned(x.x, w.x, second, product(0)), turned(x.y, w.y, second, product(1)),
                               turned(x.z, w.z, second, product(2)), turned(x.w, w.w, second, product(3))};
            y = store_block<true>(v, words_at(a.kv, at, j, d), scale_at(a.kv, at, j, d));
        } else {
            const Pair v[4] = {{x.x, 0.f}, {x.y, 0.f}, {x.z, 0.f}, {x.w, 0.f}};
            y = store_block<false>(v, words_at(a.kv, at, j, d), scale_at(a.kv, at, j, d));
        }
        lo = min4(lo, y);
        hi = max4(hi, y);
    }
    if (a.kv.bounds == nullptr) return;
    // the groups' extremes meet, by halves
    float4* mine = sums + tid * 2u;
    mine[0] = lo;
    mine[1] = hi;
    for (uint32_t n = min(groups, j1 - j0); n > 1u; n = (n + 1u) / 2u) {
        __syncthreads();
        const uint32_t from = g + (n + 1u) / 2u;
        if (from < n) {
            const float4* other = sums + (tid + (from - g) * 8u) * 2u;
            mine[0] = lo = min4(lo, other[0]);
            mine[1] = hi = max4(hi, other[1]);
        }
    }
    if (g == 0u) store_bounds(static_cast<__half*>(a.kv.bounds) + head * 2u * hd + d, hd, lo, hi, j0 == 0u);
}

// One piece of ROWS token rows per thread: pairs of pieces of the query heads, then, from a multiple
// of eight threads on, pieces of the keys (a.row_keys) and of the values.
template <uint32_t ROWS, bool KEYS>
__device__ __forceinline__ void append_rows4(const AppendArgs& a, float2 (*cs)[128], double2 (*cd)[128]) {
    __shared__ int row_pos[kMaxRows];
    __shared__ uint32_t row_page[kMaxRows];
    const uint32_t item = blockIdx.x - a.key_ctas, t0 = item / a.blocks * ROWS, tid = threadIdx.x, nt = blockDim.x;
    const uint32_t hd = a.kv.head_dim, half = hd / 2u, kvh = a.kv.kv_heads, quads = half / 4u;
    const uint32_t piece = item % a.blocks * nt + tid, q_pieces = a.heads * quads, from = (q_pieces + 7u) & ~7u;
    const bool query = piece < q_pieces, block = piece >= from && piece < a.pieces;
    // where the piece is in its row
    const uint32_t first = (KEYS ? a.heads : a.heads + kvh) * hd;  // channel of the first block
    const uint32_t h = query ? piece / quads : 0u;
    const uint32_t off = query ? h * hd + (piece - h * quads) * 4u : block ? first + (piece - from) * 4u : 0u;
    const bool key = KEYS && block && off < (a.heads + kvh) * hd;
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
            if constexpr (KEYS) {
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
            if (KEYS && key && a.rotate) {
                const double2* c = cd[r] + (second ? d - half : d);
                const Pair v[4] = {turned(x[r].x, y[r].x, second, c[0]), turned(x[r].y, y[r].y, second, c[1]),
                                   turned(x[r].z, y[r].z, second, c[2]), turned(x[r].w, y[r].w, second, c[3])};
                x[r] = store_block<true>(v, words_at(a.kv, at, slot, d), scale_at(a.kv, at, slot, d));
            } else {
                const Pair v[4] = {{x[r].x, 0.f}, {x[r].y, 0.f}, {x[r].z, 0.f}, {x[r].w, 0.f}};
                x[r] = store_block<false>(v, words_at(a.kv, at, slot, d), scale_at(a.kv, at, slot, d));
            }
            if (key && a.kv.bounds != nullptr) {
                const float4 none = make_float4(INFINITY, INFINITY, INFINITY, INFINITY);
                const float4 least = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                store_bounds(static_cast<__half*>(a.kv.bounds) + head * 2u * hd + d, hd, min4(none, x[r]), max4(least, x[r]), slot == 0u);
            }
        }
    }
}

// KEYS: keys with their rows (no sequence has several new tokens).
template <uint32_t ROWS, bool KEYS>
__global__ void __launch_bounds__(256) kv_append4_kernel(AppendArgs a) {
    // sines: of the rows' channel pairs; or of a block's channels for every eighth token of a page (at most 256)
    // and the eight in between, and behind them the threads' extremes
    constexpr uint32_t kFar = 256u / kEighth * 32u, kNear = kEighth * 32u;
    constexpr uint32_t kBytes = KEYS ? ROWS * 128u * 24u : (kFar + kNear) * 16u + 256u * 32u;
    __shared__ __align__(16) uint8_t sm[kBytes];
    if (!KEYS && blockIdx.x < a.key_ctas) {
        double2(*far)[32] = reinterpret_cast<double2(*)[32]>(sm);
        append_keys4(a, far, far + kFar / 32u, reinterpret_cast<float4*>(sm + (kFar + kNear) * 16u));
    } else {
        append_rows4<ROWS, KEYS>(a, reinterpret_cast<float2(*)[128]>(sm), reinterpret_cast<double2(*)[128]>(sm + ROWS * 128u * 8u));
    }
}

// ---- reading ------------------------------------------------------------------
struct ReadArgs {
    PagedKv kv;
    PagedBatch b;
    float *k, *v;
    uint32_t pieces, rows;  // pieces of eight channels of a row (keys, then values), rows of a CTA
    DeviceStatus* st;
};

constexpr uint32_t kReadRows = 8;
// Eight channels of a token's keys or values at a time.
__global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
    __shared__ uint32_t row_page[kReadRows], row_slot[kReadRows];
    __shared__ uint8_t row_there[kReadRows];
    const uint32_t t0 = blockIdx.x * a.rows, tid = threadIdx.x;
    if (tid < a.rows) {
        uint32_t page = kNone, slot = 0;
        bool there = false;
        const uint32_t s = t0 + tid < a.b.tokens ? seq_of_token(a.b, t0 + tid) : kNone;
        if (s != kNone) {
            const PagedSeq sq = load_seq(a.b, s, a.st);
            there = sq.n != 0u;
            const int p = there ? sq.pos(t0 + tid - sq.t0) : -1;
            if (p >= 0) {
                page = load_page(a.b, a.kv, s, static_cast<uint32_t>(p) >> a.kv.page_shift, a.st);
                slot = static_cast<uint32_t>(p) & (a.kv.page_size - 1u);
            }
        }
        row_page[tid] = page;
        row_slot[tid] = slot;
        row_there[tid] = there;
    }
    __syncthreads();
    const uint32_t hd = a.kv.head_dim, kvh = a.kv.kv_heads, row = kvh * hd;
#pragma unroll 4
    for (uint32_t x = tid; x < a.rows * a.pieces; x += blockDim.x) {
        const uint32_t r = x / a.pieces, piece = x - r * a.pieces;
        if (!row_there[r]) continue;
        const bool values = piece * 8u >= row;
        const uint32_t e = piece * 8u - (values ? row : 0u), kh = e / hd, d = e - kh * hd, page = row_page[r], slot = row_slot[r];
        float4 y[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        if (page != kNone) {
            const void* cache = values ? a.kv.v : a.kv.k;
            const size_t head = static_cast<size_t>(page) * kvh + kh, at = (head * a.kv.page_size + slot) * hd + d;
            if (a.kv.type == kF32) {
                y[0] = *reinterpret_cast<const float4*>(static_cast<const float*>(cache) + at);
                y[1] = *reinterpret_cast<const float4*>(static_cast<const float*>(cache) + at + 4u);
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
                y[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
                y[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
            }
        }
        float* to = (values ? a.v : a.k) + static_cast<size_t>(t0 + r) * row + e;
        *reinterpret_cast<float4*>(to) = y[0];
        *reinterpret_cast<float4*>(to + 4u) = y[1];
    }
}

}  // namespace

cudaError_t launch_kv_append4(const PagedKv& kv, const PagedBatch& b, uint32_t heads, const float* qkv, double theta,
                              float* q_out, DeviceStatus* st, cudaStream_t stream) {
    const uint32_t q_pieces = heads * (kv.head_dim / 8u);
    const AppendLaunch l = append_launch(kv, b, heads, qkv, theta, q_out, st, kv.kv_heads * (kv.head_dim / 4u), (8u - q_pieces % 8u) % 8u,
                                         kv.head_dim / 32u);
    if (l.grid > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    const bool four = l.a.rows == kMaxRows;
    void (*const kernel)(AppendArgs) = l.a.row_keys ? (four ? kv_append4_kernel<kMaxRows, true> : kv_append4_kernel<1, true>)
                                                    : (four ? kv_append4_kernel<kMaxRows, false> : kv_append4_kernel<1, false>);
    kernel<<<static_cast<uint32_t>(l.grid), l.threads, 0, stream>>>(l.a);
    return cudaGetLastError();
}

cudaError_t launch_kv_read(const PagedKv& kv, const PagedBatch& b, float* k, float* v, DeviceStatus* st, cudaStream_t stream) {
    ReadArgs a = {};
    a.kv = kv;
    a.b = b;
    a.k = k;
    a.v = v;
    a.pieces = 2u * kv.kv_heads * (kv.head_dim / 8u);
    // four pieces to a thread where there are CTAs enough
    a.rows = std::max(1u, std::min({1024u / a.pieces, kReadRows, b.tokens / 592u}));
    a.st = st;
    const uint32_t threads = std::min(256u, (a.pieces * a.rows + 31u) / 32u * 32u);
    kv_read_kernel<<<(b.tokens + a.rows - 1u) / a.rows, threads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace nedo_gpu

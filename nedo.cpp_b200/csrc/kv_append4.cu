// kv_append4.cu -- the new tokens' keys and values into a paged Q4_0 cache (paged_q4.cuh), with the
// position rotation of queries and keys on the way, and the tokens' keys and values out of a cache.
//
// A block of 32 channels becomes numbers n and a scale d:
//   d = -x / 8 for the number x of largest magnitude (the negative one where both signs reach it),
//       in eight significant bits, to the nearest (even) one, in steps of no less than 2^-24 and
//       with a magnitude of at most 8160 = 255 * 2^5;
//   n = floor(x / d + 8.5) within 0..15, 8 where d is 0;
// and the scale NaN where a number of it is not finite.  A rounding error in x moves n by a whole
// step where x is next to a border of two.  Values are compared with the borders d (n - 8.5), which are exact,
// as they come.  Keys are turned in 32 bits, with a bound on what that can be off; where a scale or a number is
// not certain, in one warp of some two hundred, the warp's keys are turned again, with angles, sines and cosines of 64
// bits and products as pairs of 32-bit numbers, x = hi + lo, exact to some 2^-46.  (Three prompts of 317 to 1025
// tokens 20.7 us; all keys turned so 37.6.)
//
// One launch with two kinds of CTAs, as over F16 and F32 caches.  Rows: one or four token rows, a thread a piece
// of each, a pair of pieces of a query head, or four channels of a value (or key, where no sequence has several
// new tokens), of which eight neighbouring threads have a block and agree on its extremes by shuffles.  Keys:
// a block of 32 channels of one page, for one or some KV heads, because the bounds need the page's new tokens in
// one place (keys with their rows and the bounds in a second launch: 37 us).  Sines and cosines are formed once
// for the heads of a CTA.
#include <algorithm>

#include "kv_append.cuh"
#include "paged_q4.cuh"

namespace nedo_gpu {
namespace {

// Turns per position of channel pair k; rate: -2 / head_dim log2(theta).
__device__ __forceinline__ double turns_of_rate(double rate, uint32_t k) {
    return exp2(k * rate) * 0.15915494309189535;  // 1 / (2 pi)
}
// Cosine and sine of position p's rotation in 64 bits.
__device__ __forceinline__ double2 rotation64(double p, double turns) {
    double turn = p * turns, c, s;
    turn -= rint(turn);
    sincospi(2.0 * turn, &s, &c);
    return make_double2(c, s);
}

// An eighth of a magnitude hi + lo as a scale: eight significant bits are the upper half of the number's.
__device__ __forceinline__ float scale_of(float hi, float lo) {
    const float x = hi * 0.125f;
    if (x < 0x1p-17f) return static_cast<float>(rint((static_cast<double>(hi) + lo) * 0x1p21) * 0x1p-24);
    uint32_t b = __float_as_uint(x);
    if ((b & 0xFFFFu) == 0x8000u && lo != 0.f) b += lo > 0.f ? 1u : ~0u;  // between two, but for what is left
    b += 0x7FFFu + ((b >> 16) & 1u);
    return fminf(__uint_as_float(b & 0xFFFF0000u), 8160.f);
}
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A number as hi + lo, hi the nearest of 32 bits.
struct Pair {
    float hi, lo;
};
__device__ __forceinline__ Pair pair_of(double x) {
    const float hi = static_cast<float>(x);
    return {hi, static_cast<float>(x - hi)};
}
// The smallest and largest of eight lanes' numbers.
__device__ __forceinline__ void extremes(float& low, float& high) {
#pragma unroll
    for (uint32_t o = 1; o < 8u; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xFFFFFFFFu, high, o));
    }
}
// Whether one of eight lanes says so.
__device__ __forceinline__ bool any_of_eight(bool x) {
    return (__ballot_sync(0xFFFFFFFFu, x) >> (threadIdx.x & 24u) & 0xFFu) != 0u;
}
// Four numbers of a block that eight neighbouring lanes have (all of a warp come here).
struct Quad {
    float d;         // the block's scale, its magnitude
    uint32_t sign;   // the bit that the numbers' signs are turned by: 0 where d is positive
    bool bad;        // a number of the block is not finite
    float m[4];      // n
};
// The block's scale and sign from the largest magnitude, of negative numbers or not, hi + lo.
__device__ __forceinline__ void set_scale(Quad& q, bool negative, float d, float odd) {
    q.bad = any_of_eight(odd != 0.f);  // (a sum of zeros times the numbers: NaN)
    q.d = q.bad ? 0.f : d;
    q.sign = negative ? 0u : 0x80000000u;
}
__device__ __forceinline__ float turn_sign(float x, uint32_t sign) { return __uint_as_float(__float_as_uint(x) ^ sign); }
// The largest whole number n with d (n - 8.5) <= v or the one below it (adding 1.5 2^23 rounds to a whole
// number), and the next one's border.
__device__ __forceinline__ float number_below(float v, float d, float inv, float* border) {
    const float t = fminf(fmaxf(v * inv, -9.f), 9.f) + (8.f - 1.f / 1024.f);
    const float n = (t + 12582912.f) - 12582912.f;
    *border = fmaf(n, d, -7.5f * d);
    return n;
}
__device__ __forceinline__ float number_of(const Quad& q, float n, bool up) {
    return q.d == 0.f ? 8.f : fminf(fmaxf(up ? n + 1.f : n, 0.f), 15.f);
}
// Numbers that are exact (values, keys that are not turned), or off by no more than off[e]: then whether the
// scale and the numbers are certain.
template <bool OFF>
__device__ __forceinline__ bool quantise(const float (&x)[4], const float (&off)[4], Quad& q) {
    float low = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), high = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    extremes(low, high);
    const bool negative = -low >= high;
    const float size = negative ? -low : high;
    float d = scale_of(size, 0.f);
    bool open = false;
    if constexpr (OFF) {
        float most = fmaxf(fmaxf(off[0], off[1]), fmaxf(off[2], off[3]));
#pragma unroll
        for (uint32_t o = 1; o < 8u; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
        open = scale_of(size + most, 0.f) != scale_of(fmaxf(size - most, 0.f), 0.f) || fabsf(-low - high) <= 2.f * most;
        open &= size + most >= 0x1p-22f;  // (nothing but zeros)
    }
    set_scale(q, negative, d, fmaf(x[0], 0.f, fmaf(x[1], 0.f, fmaf(x[2], 0.f, x[3] * 0.f))));
    const float inv = q.d == 0.f ? 0.f : reciprocal(q.d);
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
        const float v = turn_sign(x[e], q.sign);
        float border;
        const float n = number_below(v, q.d, inv, &border);
        q.m[e] = number_of(q, n, border <= v);
        if constexpr (OFF) open |= q.d != 0.f && (fabsf(v - border) <= off[e] || off[e] > q.d * (1.f / 4096.f));
    }
    return open;
}
// Numbers as pairs.
__device__ __forceinline__ void quantise(const Pair (&x)[4], Quad& q) {
    float low = fminf(fminf(x[0].hi, x[1].hi), fminf(x[2].hi, x[3].hi)), high = fmaxf(fmaxf(x[0].hi, x[1].hi), fmaxf(x[2].hi, x[3].hi));
    extremes(low, high);
    float low2 = INFINITY, high2 = -INFINITY;
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
        if (x[e].hi == low) low2 = fminf(low2, x[e].lo);
        if (x[e].hi == high) high2 = fmaxf(high2, x[e].lo);
    }
    extremes(low2, high2);
    const bool negative = -low > high || (-low == high && -low2 >= high2);
    set_scale(q, negative, negative ? scale_of(-low, -low2) : scale_of(high, high2),
              fmaf(x[0].hi, 0.f, fmaf(x[1].hi, 0.f, fmaf(x[2].hi, 0.f, x[3].hi * 0.f))));
    const float inv = q.d == 0.f ? 0.f : reciprocal(q.d);
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
        const float v = turn_sign(x[e].hi, q.sign);
        float border;
        const float n = number_below(v, q.d, inv, &border);
        q.m[e] = number_of(q, n, border < v || (border == v && turn_sign(x[e].lo, q.sign) >= 0.f));
    }
}
// The block's numbers to `words` and its scale to `scale`, where `store` says so, and what the cache then holds
// for the four.
__device__ __forceinline__ float4 store_block(const Quad& q, uint32_t* words, __half* scale, bool store) {
    const uint32_t lane = threadIdx.x & 31u;
    // channels 0 and 2 (or 4 and 6) to the low half, 1 and 3 to the high one
    uint32_t mine = static_cast<uint32_t>(fmaf(fmaf(q.m[3], 16.f, q.m[1]), 65536.f, fmaf(q.m[2], 16.f, q.m[0])));
    mine <<= (lane & 1u) * 8u;
    mine |= __shfl_xor_sync(0xFFFFFFFFu, mine, 1);
    if (store && (lane & 1u) == 0u) words[(lane & 7u) >> 1] = mine;
    if (store && (lane & 7u) == 0u) *scale = q.bad ? __ushort_as_half(0x7FFF) : __float2half_rn(turn_sign(q.d, q.sign));
    const float d = q.bad ? __int_as_float(0x7FFFFFFF) : turn_sign(q.d, q.sign);
    return make_float4(d * (q.m[0] - 8.f), d * (q.m[1] - 8.f), d * (q.m[2] - 8.f), d * (q.m[3] - 8.f));
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
// back): u cos -+ w sin, as a pair.
__device__ __forceinline__ Pair turned(float u, float w, bool second, double2 c) {
    const double t = second ? c.y : -c.y;
    if (fmaxf(fabsf(u), fabsf(w)) > 1e35f) {
        // what leaves 32 bits has the largest scale whatever it is: numbers above 10^36 come closer, in order
        const double x = u * c.x + w * t, size = fabs(x);
        return pair_of(size > 1e36 && size < static_cast<double>(INFINITY) ? copysign(1e36 + size * 0x1p-10, x) : x);
    }
    const Pair cos = pair_of(c.x), sin = pair_of(t);
    const float p = u * cos.hi, q = w * sin.hi;
    const float p2 = fmaf(u, cos.lo, fmaf(u, cos.hi, -p)), q2 = fmaf(w, sin.lo, fmaf(w, sin.hi, -q));
    const float s = p + q, r = s - p;
    const float low = ((p - (s - r)) + (q - r)) + (p2 + q2);
    const float hi = s + low;
    return {hi, low - (hi - s)};
}
// The numbers of a block of keys whose 32-bit ones are not certain: channels u, with w half a head on or back,
// of channel pairs k, k + 1, ... at position p.
__device__ __noinline__ Quad quantise_again(float4 u, float4 w, bool second, uint32_t k, int p, double rate) {
    Pair v[4];
    const float x[4] = {u.x, u.y, u.z, u.w}, y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll 1
    for (uint32_t e = 0; e < 4u; ++e) v[e] = turned(x[e], y[e], second, rotation64(p, turns_of_rate(rate, k + e)));
    Quad q;
    quantise(v, q);
    return q;
}

struct Append4Args {
    PagedKv kv;
    PagedBatch b;
    const float* qkv;
    float* q_out;
    double rate;              // -2 / head_dim log2(theta)
    uint32_t heads, rotate;
    uint32_t segs;            // pages that a sequence's new tokens can touch
    uint32_t keys_at, values_at, pieces;  // of a row: where those of the keys and values begin, and all
    uint32_t blocks;                      // CTAs that share them
    uint32_t key_ctas;        // CTAs of keys
    uint32_t key_heads;       // KV heads of one of them
    DeviceStatus* st;
};
constexpr uint32_t kMost = 256;  // threads of a CTA

// Four channels of a key, u, with w half a head on or back, turned by c at position p (channel pairs k, k + 1, ...),
// as a block's numbers.  A whole warp; `there`: not only along.
__device__ __forceinline__ Quad quantise_key(float4 u4, float4 w4, bool second, const float2* c, uint32_t k, int p, double rate,
                                             bool there) {
    const float u[4] = {u4.x, u4.y, u4.z, u4.w}, w[4] = {w4.x, w4.y, w4.z, w4.w};
    // 16 roundings of |u| + |w|: of the products, the sum, and four steps of sine and cosine
    float v[4], off[4];
    bool open = false;
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
        v[e] = fmaf(u[e], c[e].x, w[e] * (second ? c[e].y : -c[e].y));
        off[e] = (fabsf(u[e]) + fabsf(w[e])) * 0x1.01p-20f;
        open |= off[e] > 1e31f;
    }
    Quad q;
    open |= quantise<true>(v, off, q);
    if (__any_sync(0xFFFFFFFFu, open && there)) q = quantise_again(u4, w4, second, k, p, rate);
    return q;
}

constexpr uint32_t kAtOnce = 64;  // tokens whose sines are held
struct KeyShared {
    float2 sines[kAtOnce][32];
    float4 low[2][8][8], high[2][8][8];  // extremes [turn][warp][four channels]
};
// One block of 32 channels of the keys of one page and some KV heads, and its bounds (fminf / fmaxf leave
// NaN out).  A page whose first slot is written begins anew.
__device__ __forceinline__ void append_keys4(const Append4Args& a, KeyShared& sm) {
    const uint32_t blocks = a.kv.head_dim / 32u, parts = (a.kv.kv_heads + a.key_heads - 1u) / a.key_heads;
    uint32_t rest = blockIdx.x;
    const uint32_t block = rest % blocks;
    rest /= blocks;
    const uint32_t h0 = rest % parts * a.key_heads, h1 = min(h0 + a.key_heads, a.kv.kv_heads);
    rest /= parts;
    const uint32_t s = rest / a.segs, seg = rest % a.segs;
    const PagedSeq sq = load_seq(a.b, s, a.st);
    const uint32_t fresh = min(sq.n, sq.kv);  // rows that are tokens
    if (fresh == 0u) return;
    const uint32_t begin = sq.kv - fresh, lp = (begin >> a.kv.page_shift) + seg, first = lp << a.kv.page_shift;
    if (first >= sq.kv) return;
    const uint32_t page = load_page(a.b, a.kv, s, lp, a.st);
    if (page == kNone) return;
    const uint32_t j0 = first < begin ? begin - first : 0u, j1 = min(sq.kv - first, a.kv.page_size);
    const uint32_t hd = a.kv.head_dim, half = hd / 2u, tid = threadIdx.x, lane = tid & 31u, warp = tid / 32u;
    const uint32_t groups = blockDim.x / 8u, g = tid / 8u, warps = blockDim.x / 32u;
    const size_t width = static_cast<size_t>(a.heads + 2u * a.kv.kv_heads) * hd;
    const uint32_t c = (tid & 7u) * 4u, d = 32u * block + c;
    const bool second = d >= half;
    const int to = second ? -static_cast<int>(half) : static_cast<int>(half);
    const uint32_t ch = 32u * block + lane;
    const double turns = a.rotate ? turns_of_rate(a.rate, ch >= half ? ch - half : ch) : 0.0;
    uint32_t turn = 0;
    for (uint32_t b0 = j0; b0 < j1; b0 += kAtOnce) {
        const uint32_t b1 = min(j1, b0 + kAtOnce);
        if (a.rotate) {  // a warp: the 32 channels of one token
            if (b0 != j0) __syncthreads();
            for (uint32_t j = b0 + warp; j < b1; j += warps) sm.sines[j - b0][lane] = rotation(static_cast<int>(first + j), turns);
            __syncthreads();
        }
        for (uint32_t h = h0; h < h1; ++h) {
            const size_t head = static_cast<size_t>(page) * a.kv.kv_heads + h;
            uint8_t* const at = static_cast<uint8_t*>(a.kv.k) + head * q4_head_bytes(a.kv);
            const float* src = a.qkv + static_cast<size_t>(a.heads + h) * hd + d;
            float4 lo = make_float4(INFINITY, INFINITY, INFINITY, INFINITY), hi = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            // (whole warps, for the shuffles: a thread beyond the last token goes along with it; the next token's
            // channels are on their way.  A pair's other half is read only to turn with it: 0 times infinity is not 0)
            float4 x, w;
            auto load = [&](uint32_t jw) {
                const float* row = src + static_cast<size_t>(sq.t0 + sq.n - (sq.kv - (first + min(jw + (g & 3u), b1 - 1u)))) * width;
                x = __ldg(reinterpret_cast<const float4*>(row));
                if (a.rotate) w = __ldg(reinterpret_cast<const float4*>(row + to));
            };
            w = make_float4(0.f, 0.f, 0.f, 0.f);
            if (b0 + 4u * warp < b1) load(b0 + 4u * warp);
#pragma unroll 1
            for (uint32_t jw = b0 + 4u * warp; jw < b1; jw += groups) {
                const uint32_t j = min(jw + (g & 3u), b1 - 1u);
                const bool there = jw + (g & 3u) < b1;
                const float4 x0 = x, w0 = w;
                if (jw + groups < b1) load(jw + groups);
                Quad q;
                if (a.rotate) {
                    q = quantise_key(x0, w0, second, sm.sines[j - b0] + c, second ? d - half : d, static_cast<int>(first + j), a.rate, there);
                } else {
                    const float u[4] = {x0.x, x0.y, x0.z, x0.w};
                    quantise<false>(u, u, q);
                }
                const float4 y = store_block(q, words_at(a.kv, at, j, d), scale_at(a.kv, at, j, d), there);
                lo = min4(lo, y);
                hi = max4(hi, y);
            }
            if (a.kv.bounds == nullptr) continue;
            // the extremes of a warp's four tokens at once meet by shuffles, the warps' in shared memory
#pragma unroll
            for (uint32_t o = 8; o <= 16u; o <<= 1) {
                lo = min4(lo, make_float4(__shfl_xor_sync(0xFFFFFFFFu, lo.x, o), __shfl_xor_sync(0xFFFFFFFFu, lo.y, o),
                                          __shfl_xor_sync(0xFFFFFFFFu, lo.z, o), __shfl_xor_sync(0xFFFFFFFFu, lo.w, o)));
                hi = max4(hi, make_float4(__shfl_xor_sync(0xFFFFFFFFu, hi.x, o), __shfl_xor_sync(0xFFFFFFFFu, hi.y, o),
                                          __shfl_xor_sync(0xFFFFFFFFu, hi.z, o), __shfl_xor_sync(0xFFFFFFFFu, hi.w, o)));
            }
            turn ^= 1u;  // (in turns: one barrier a head)
            if (lane < 8u) {
                sm.low[turn][warp][lane] = lo;
                sm.high[turn][warp][lane] = hi;
            }
            __syncthreads();
            if (tid < 8u) {
                for (uint32_t w = 1; w < warps; ++w) {
                    lo = min4(lo, sm.low[turn][w][tid]);
                    hi = max4(hi, sm.high[turn][w][tid]);
                }
                store_bounds(static_cast<__half*>(a.kv.bounds) + head * 2u * hd + d, hd, lo, hi, b0 == 0u);
            }
        }
    }
}

// One piece of ROWS token rows per thread: pairs of pieces of the query heads, pieces of the keys (KEYS), pieces
// of the values, each of whole warps.
template <uint32_t ROWS, bool KEYS>
__device__ __forceinline__ void append_rows4(const Append4Args& a, float2 (*sines)[128]) {
    __shared__ int row_pos[ROWS];
    __shared__ uint32_t row_page[ROWS];
    const uint32_t item = blockIdx.x - a.key_ctas;
    const uint32_t t0 = item / a.blocks * ROWS, tid = threadIdx.x, nt = blockDim.x;
    const uint32_t hd = a.kv.head_dim, half = hd / 2u, kvh = a.kv.kv_heads, quads = half / 4u;
    const uint32_t piece = item % a.blocks * nt + tid, of_kind = kvh * (hd / 4u);
    // where the piece is in its row (a warp: one kind)
    const bool key = KEYS && piece >= a.keys_at && piece < a.values_at, value = piece >= a.values_at;
    const uint32_t at_kind = piece - (value ? a.values_at : key ? a.keys_at : 0u);
    const bool query = !key && !value, there = query ? piece < a.heads * quads : at_kind < of_kind;
    const uint32_t h = query ? at_kind / quads : at_kind / (hd / 4u);  // head, of its kind, and channel
    const uint32_t d = query ? (at_kind - h * quads) * 4u : (at_kind - h * (hd / 4u)) * 4u;
    const uint32_t off = there ? (h + (value ? a.heads + kvh : key ? a.heads : 0u)) * hd + d : 0u;
    const bool second = key && d >= half;
    const size_t width = static_cast<size_t>(a.heads + 2u * kvh) * hd;
    float4 x[ROWS], y[ROWS];
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        x[r] = y[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!there || t0 + r >= a.b.tokens) continue;
        const float* src = a.qkv + (t0 + r) * width + off;
        x[r] = __ldg(reinterpret_cast<const float4*>(src));
        // (a pair's other half is read only to turn with it: 0 times infinity is not 0)
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
        const double turns = tid < groups * half ? turns_of_rate(a.rate, k) : 0.0;
        __syncthreads();
        for (uint32_t r = tid / half; r < ROWS && tid < groups * half; r += groups)
            if (row_pos[r] >= 0) sines[r][k] = rotation(row_pos[r], turns);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        const int p = row_pos[r];
        if (p < 0) continue;
        const uint32_t k = !there ? 0u : second ? d - half : d;
        const float2* c = sines[r] + k;
        if (query) {
            if (!there) continue;
            if (a.rotate) rotate4(x[r], y[r], c);
            float* o = a.q_out + (static_cast<size_t>(t0 + r) * a.heads + h) * hd + d;
            *reinterpret_cast<float4*>(o) = x[r];
            *reinterpret_cast<float4*>(o + half) = y[r];
        } else if (row_page[r] != kNone) {
            const uint32_t slot = static_cast<uint32_t>(p) & (a.kv.page_size - 1u);
            const size_t head = static_cast<size_t>(row_page[r]) * kvh + h;
            uint8_t* const at = static_cast<uint8_t*>(key ? a.kv.k : a.kv.v) + (there ? head * q4_head_bytes(a.kv) : 0u);
            Quad q;
            if (key && a.rotate) {
                q = quantise_key(x[r], y[r], second, c, k, p, a.rate, there);
            } else {
                const float u[4] = {x[r].x, x[r].y, x[r].z, x[r].w};
                quantise<false>(u, u, q);
            }
            x[r] = store_block(q, words_at(a.kv, at, slot, d), scale_at(a.kv, at, slot, d), there);
            if (key && there && a.kv.bounds != nullptr) {
                const float4 none = make_float4(INFINITY, INFINITY, INFINITY, INFINITY);
                const float4 least = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                store_bounds(static_cast<__half*>(a.kv.bounds) + head * 2u * hd + d, hd, min4(none, x[r]), max4(least, x[r]), slot == 0u);
            }
        }
    }
}

// KEYS: keys with their rows (no sequence has several new tokens).
template <uint32_t ROWS, bool KEYS>
__global__ void __launch_bounds__(kMost, 4) kv_append4_kernel(Append4Args a) {
    constexpr uint32_t kSines = ROWS * 128u * 8u;
    __shared__ __align__(16) uint8_t sm[KEYS || kSines > sizeof(KeyShared) ? kSines : sizeof(KeyShared)];
    if (!KEYS && blockIdx.x < a.key_ctas) append_keys4(a, *reinterpret_cast<KeyShared*>(sm));
    else append_rows4<ROWS, KEYS>(a, reinterpret_cast<float2(*)[128]>(sm));
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
    Append4Args a = {};
    a.kv = kv;
    a.b = b;
    a.qkv = qkv;
    a.q_out = q_out;
    a.rotate = theta > 0.0;
    a.rate = a.rotate ? -2.0 / kv.head_dim * log2(theta) : 0.0;
    a.heads = heads;
    a.segs = (b.max_q_len + kv.page_size - 2u) / kv.page_size + 1u;
    a.st = st;
    const bool keys = b.max_q_len <= 1u;
    auto warps = [](uint32_t n) { return (n + 31u) / 32u * 32u; };
    a.keys_at = warps(heads * (kv.head_dim / 8u));
    a.values_at = a.keys_at + (keys ? warps(kv.kv_heads * (kv.head_dim / 4u)) : 0u);
    a.pieces = a.values_at + warps(kv.kv_heads * (kv.head_dim / 4u));
    a.blocks = (a.pieces + kMost - 1u) / kMost;
    const uint32_t rows = b.tokens >= 4u * 148u ? 4u : 1u;  // four rows share their sines where there are CTAs enough
    uint64_t key_ctas = 0;
    if (!keys) {
        // KV heads to a CTA of keys: several share their sines where there are CTAs enough
        const uint64_t pages = static_cast<uint64_t>(b.seqs) * a.segs * (kv.head_dim / 32u);
        a.key_heads = static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>(pages * kv.kv_heads / 592u, 1u), kv.kv_heads));
        key_ctas = pages * ((kv.kv_heads + a.key_heads - 1u) / a.key_heads);
    }
    const uint64_t grid = key_ctas + static_cast<uint64_t>((b.tokens + rows - 1u) / rows) * a.blocks;
    if (grid > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    a.key_ctas = static_cast<uint32_t>(key_ctas);
    // a thread for every piece, and for every channel pair; more for the tokens of a page, the more where there are
    // few pages (18 prompts of 35 to 106 tokens, 2 KV heads of 32 channels: 15 us; 26 with 64 threads)
    const uint32_t least = keys ? 32u : key_ctas < 592u ? kMost : 128u;
    const uint32_t threads = std::max(least, warps(std::max((a.pieces + a.blocks - 1u) / a.blocks, kv.head_dim / 2u)));
    void (*const kernel)(Append4Args) = keys ? (rows == 4u ? kv_append4_kernel<4, true> : kv_append4_kernel<1, true>)
                                             : (rows == 4u ? kv_append4_kernel<4, false> : kv_append4_kernel<1, false>);
    kernel<<<static_cast<uint32_t>(grid), threads, 0, stream>>>(a);
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

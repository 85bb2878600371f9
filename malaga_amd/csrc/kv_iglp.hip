// Attention of each sequence's rows over its tokens in the paged K/V cache (paged_kv.hpp):
//   s_j = scale q . k_j over the tokens that the row sees, o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m).
//
// One pass over the tokens with the running maximum m and sum l of the softmax, 32 tokens (a tile of
// the cache) at a time on v_mfma_f32_16x16x32_f16:
//   scores^T [32 tokens][16 rows] = K q^T,  out^T [dims][16 rows] += V^T p^T
// so that a lane keeps one row's statistics and p never leaves its registers. A row is one query head
// of one token; the heads that share a K/V head are rows of the same tile.
//
// Results are as exact as f32 arithmetic: K and V are exact operands (f16, or the whole numbers of a
// q8_0 block, whose scales are applied in f32), and q and p enter as two f16 each (hi = f16(x), lo =
// f16(x - hi): 22 bits), which doubles the matrix work. q is scaled by a power of two per row, and p's
// largest held between 2^7 and 2^15, so that what lo loses below f16's range is 2^-31 of the largest value.
// Sums are f32.
#include <type_traits>

#include "device.hpp"
#include "paged_kv.hpp"

namespace mlg {
namespace {

constexpr int kRows = 16;        // rows of a query tile (columns of the matrix products)
constexpr int kWaves = 4;        // waves of a workgroup
// p = 2^(s - m): m is the running maximum of the scores (log2 units) less kPShift, and follows a larger
// one only when it is kPSlack or more behind, which after the first tiles is rare: p stays below 2^15.
constexpr float kPShift = 7.f, kPSlack = 8.f;

constexpr int kLeastTiles = 8;  // of a split: a short sequence does not use all of a call's splits

// Partial result of a split: [m, l, -, -, out of HD dims] of one row, f32, as a Tile holds them.
constexpr int kPartHead = 4;

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ h8_t as_h8(const uint4 &v) { return __builtin_bit_cast(h8_t, v); }

// 8 int8 as f16, exactly: byte + 128 becomes the low byte of 1024 + u, minus 1152.
__device__ __forceinline__ h8_t i8_to_h8(uint32_t lo, uint32_t hi) {
    const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
    auto two = [](uint32_t v, uint32_t sel) __attribute__((always_inline)) {
        const h2_t h = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, v, sel));
        return __builtin_bit_cast(uint32_t, h - h2_t{_Float16(1152.f), _Float16(1152.f)});
    };
    return as_h8(make_uint4(two(a, 0x07010700u), two(a, 0x07030702u), two(b, 0x07010700u), two(b, 0x07030702u)));
}

// The maximum that keeps NaN: one v_maximum3_f32 for three values, where fmaxf first quiets what may
// be a signalling NaN. (No inline asm for it: the compiler does not see that such an instruction reads
// a matrix product's result or feeds a lane swap, and leaves out the waits that both need.)
__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float vmax3(float a, float b, float c) { return vmax(vmax(a, b), c); }

// v of lane l and of lane l ^ 32 (l ^ 16), in some order.
struct Pair {
    uint32_t a, b;
};
__device__ __forceinline__ Pair with_xor32(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return {uint32_t(r[0]), uint32_t(r[1])};
}
__device__ __forceinline__ Pair with_xor16(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return {uint32_t(r[0]), uint32_t(r[1])};
}
// Over the four k-groups' lanes of a row: l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float rows_max(float v) {
    Pair p = with_xor32(__float_as_uint(v));
    v = vmax(__uint_as_float(p.a), __uint_as_float(p.b));
    p = with_xor16(__float_as_uint(v));
    return vmax(__uint_as_float(p.a), __uint_as_float(p.b));
}
__device__ __forceinline__ float rows_sum(float v) {
    Pair p = with_xor32(__float_as_uint(v));
    v = __uint_as_float(p.a) + __uint_as_float(p.b);
    p = with_xor16(__float_as_uint(v));
    return __uint_as_float(p.a) + __uint_as_float(p.b);
}
__device__ __forceinline__ uint32_t rows_umax(uint32_t v) {
    Pair p = with_xor32(v);
    p = with_xor16(max(p.a, p.b));
    return max(p.a, p.b);
}

// One lane's part of a K or V tile, as it lies in the cache.
//
// BLOCKS (q8_0, 16 / (HD / 32) rows at most): column col of the products is one block of 32 dims, col %
// (HD / 32), of row col / (HD / 32) instead of a row. Its q is zero outside of its block and its p is
// times its block's scales, so that a lane applies the scales of its own block alone, once, where every
// row's lane applies all blocks' scales in turn otherwise.
template <int HD, bool Q8, bool BLOCKS>
struct RawTile {
    static constexpr int NC = HD / 32, NU = HD / 16, NP = Q8 ? NC : NU, ND = Q8 && !BLOCKS ? NC : 1;
    u4_t a[NP];
    u4_t d[ND];  // q8_0: the scales of the lane's tokens 8 g .. 8 g + 7, per block of 32 dims
    // ONCE: no other workgroup reads the tile, so it is not kept in the caches (non-temporal loads).
    template <bool ONCE>
    __device__ __forceinline__ void load(const uint8_t *tile, int lane) {
        auto at = [](const uint8_t *p) __attribute__((always_inline)) {
            const u4_t *q = reinterpret_cast<const u4_t *>(p);
            return ONCE ? __builtin_nontemporal_load(q) : *q;
        };
#pragma unroll
        for (int i = 0; i < NP; ++i) a[i] = at(tile + (i * 64 + lane) * 16);
        if constexpr (Q8) {
#pragma unroll
            for (int c = 0; c < ND; ++c)
                d[c] = at(tile + kv_scale_byte(HD, 8 * (lane >> 4), BLOCKS ? (lane & 15) % NC : c));
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NP; ++i) a[i] = u4_t{0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < ND; ++i) d[i] = u4_t{0u, 0u, 0u, 0u};
    }
    // As a matrix operand: K's product b of dims 32 c .. at 2 c + b, V's dims 16 u .. at u.
    __device__ __forceinline__ h8_t frag(int i) const {
        if constexpr (Q8) return i8_to_h8(a[i >> 1][2 * (i & 1)], a[i >> 1][2 * (i & 1) + 1]);
        else return __builtin_bit_cast(h8_t, a[i]);
    }
    __device__ __forceinline__ float scale(int c, int n) const {
        return float(__builtin_bit_cast(h2_t, uint32_t(d[c][n >> 1]))[n & 1]);
    }
    // V's tokens past the first `keep` of the lane's eight as zeros (of q8_0, their scales): they are
    // whatever the page held before. f16: what is left of inf and NaN as zeros too, which 0 would turn
    // into NaN for the rows that do not see its token; whether there was any (see not_finite).
    __device__ __forceinline__ bool cut(int keep) {
        bool odd = false;
        constexpr int N = Q8 ? ND : NU;
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                uint32_t w = Q8 ? d[Q8 ? i : 0][n] : a[Q8 ? 0 : i][n];
                w = keep > 2 * n + 1 ? w : keep > 2 * n ? w & 0xffffu : 0u;
                if constexpr (Q8) {
                    d[i][n] = w;
                } else {
                    const bool lo = (w & 0x7c00u) == 0x7c00u, hi = (w & 0x7c000000u) == 0x7c000000u;
                    odd |= lo || hi;
                    a[i][n] = w & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
                }
            }
        }
        return odd;
    }
    // q8_0, V: the exponent of the largest scale of the tile's tokens (INT_MIN: all zeros), of the lane's
    // block where it has one, inf and NaN left out; subnormals count as the smallest normal one.
    __device__ __forceinline__ int top_exponent() const {
        // f16 bit patterns of scales, which are not negative, are ordered; two at once
        typedef uint16_t u2_t __attribute__((ext_vector_type(2)));
        u2_t t2 = {0, 0};
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int n = 0; n < 4; ++n) t2 = __builtin_elementwise_max(t2, __builtin_bit_cast(u2_t, uint32_t(d[c][n])));
        uint32_t top = rows_umax(max(uint32_t(t2[0]), uint32_t(t2[1])));
        if (__any(top >= 0x7c00u)) {
            top = 0u;
#pragma unroll
            for (int c = 0; c < ND; ++c)
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const uint32_t b = d[c][n >> 1] >> (16 * (n & 1)) & 0xffffu;
                    top = max(top, b >= 0x7c00u ? 0u : b);
                }
            top = rows_umax(top);
        }
        return top ? max(int(top >> 10), 1) - 15 : int(0x80000000);
    }
};

// Two f16 operands of 8 f32 values: hi truncated, lo the rest, truncated too: less than 2^-20 of x is
// lost, 2^-22 on average. (Truncating, a pair of values takes 4 operations; rounded to nearest, 8.)
__device__ __forceinline__ void split8(const float (&p)[8], h8_t &hi, h8_t &lo) {
    uint32_t h[4], l[4];
    float minus = -1.f;  // not a constant to the compiler, which keeps x - hi one operation (v_fma_mix)
    asm("" : "+s"(minus));
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        // p as finished f32 values: hi's and lo's uses of a product are otherwise rounded apart
        float x = p[2 * n], y = p[2 * n + 1];
        asm("" : "+v"(x), "+v"(y));
        const h2_t t = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(x, y));
        h[n] = __builtin_bit_cast(uint32_t, t);
        l[n] = __builtin_bit_cast(
            uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf(float(t[0]), minus, x), fmaf(float(t[1]), minus, y)));
    }
    hi = as_h8(make_uint4(h[0], h[1], h[2], h[3]));
    lo = as_h8(make_uint4(l[0], l[1], l[2], l[3]));
}

__device__ __forceinline__ f4_t mfma(const h8_t &a, const h8_t &b, const f4_t &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Sum over the columns of a row: N = 1, 2, 4 or 8 neighbouring lanes, the same in each of them.
template <int N>
__device__ __forceinline__ float over_columns(float v) {
    if constexpr (N >= 2) v += dpp_mov<kDppXor1>(v);
    if constexpr (N >= 4) v += dpp_mov<kDppXor2>(v);
    if constexpr (N >= 8) v += dpp_mov<kDppHalfMirror>(v);
    return v;
}

// A tile of 16 columns (rows, or blocks of rows), and the softmax and sums of what it has seen.
template <int HD, bool Q8, bool BLOCKS>
struct Tile {
    static constexpr int NC = HD / 32, NU = HD / 16;
    h8_t qh[NC], ql[NC];
    float qf;    // scores in log2 units: qf (above 0) times the product of the scaled q
    int vis;     // tokens that this lane's row sees
    float m;     // the running maximum (log2 units) less kPShift, as rounded: p = 2^(s - m)
    f4_t l;      // f16: sum of p over all tokens so far, in each element; q8_0: l[0] over the lane's
    f4_t o[NU];
    // q8_0: the largest exponent of V's scales so far (none is below -14); p, l and out are held times 2^-e
    int e = -15;

    // q: the row's HD values (null: a row past the last, as zeros)
    __device__ __forceinline__ void load_q(const float *q, float scale, int lane) {
        float x[NC][8], amax = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
            if (q) {
                a = ld4(q + 32 * c + 8 * (lane >> 4), 0);
                b = ld4(q + 32 * c + 8 * (lane >> 4), 1);
            }
            x[c][0] = a.x, x[c][1] = a.y, x[c][2] = a.z, x[c][3] = a.w;
            x[c][4] = b.x, x[c][5] = b.y, x[c][6] = b.z, x[c][7] = b.w;
#pragma unroll
            for (int n = 0; n < 8; ++n) amax = fmaxf(amax, fabsf(x[c][n]));
            if (BLOCKS && c != (lane & 15) % NC) {
#pragma unroll
                for (int n = 0; n < 8; ++n) x[c][n] = 0.f;
            }
        }
        amax = rows_max(amax);
        // the row's largest value to [2^14, 2^15); not for 0, inf (NaN is not seen by the maximum)
        const int up = amax > 0.f && amax < INFINITY ? 14 - ilogbf(amax) : 0;
        const float sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
        // not 0: what a row does not see scores -inf, also at a scale of 0
        qf = fmaxf(ldexpf(scale == 0.f ? 1.f : fabsf(scale), -up) * 1.44269504088896340736f, 1.17549435e-38f);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                float v = ldexpf(x[c][n] * sign, up);
                asm("" : "+v"(v));
                const _Float16 h = _Float16(v);
                qh[c][n] = h;
                ql[c][n] = _Float16(v - float(h));
            }
        m = -INFINITY;
        l = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; ++u) o[u] = f4_t{0.f, 0.f, 0.f, 0.f};
    }

    // The largest score of the lane's row in a tile, as m holds it.
    __device__ __forceinline__ float top(const float (&s)[8]) const {
        const float t = vmax3(vmax3(s[0], s[1], s[2]), vmax3(s[3], s[4], s[5]), vmax(s[6], s[7]));
        return fmaf(rows_max(t), qf, -kPShift);
    }
    // Whether it takes a row's p past 2^15.
    __device__ __forceinline__ bool behind(float t) const { return t > m + kPSlack; }
    // m, l and out follow it, and (q8_0) the exponent x.
    __device__ __forceinline__ void follow(float t, int x) {
        const float mn = fmaxf(m, t);
        float al = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        if constexpr (Q8) {
            const int en = max(e, x);
            al = ldexpf(al, e - en);
            e = en;
        }
        l *= al;
#pragma unroll
        for (int u = 0; u < NU; ++u) o[u] *= al;
        m = mn;
    }
    // s becomes p.
    __device__ __forceinline__ void probs(float (&s)[8]) {
        const float base = (m == -INFINITY ? 0.f : m) + (Q8 ? float(e) : 0.f);  // -inf: every score is -inf
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = __builtin_amdgcn_exp2f(fmaf(s[n], qf, -base));
        if constexpr (Q8) l[0] += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    }

    // f16, after the last tile: the inf and NaN that cut() took out of one tile's V, to the rows that
    // see their tokens (tile: V of tokens tok0 .. in the cache). Not met by ordinary caches.
    __device__ __forceinline__ void not_finite(const uint8_t *tile, int tok0, int ctx) {
        const int g = int(threadIdx.x & 63) >> 4;
#pragma unroll 1
        for (int tk = 0; tk < min(kKvTile, ctx - tok0); ++tk) {
            const bool sees = tok0 + tk < vis;
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = kv_v_elem(false, tk, 16 * u + 4 * g + i);
                    const uint32_t x = reinterpret_cast<const uint16_t *>(tile)[e];
                    if (sees && (x & 0x7c00u) == 0x7c00u) o[u][i] += h2f(x);
                }
        }
    }

    __device__ __forceinline__ void hide(float (&s)[8], int tok0) const {
        const int at = tok0 + 8 * (int(threadIdx.x & 63) >> 4);
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = at + n < vis ? s[n] : -INFINITY;
    }
};

// A wave's QT tiles of rows: the matrix products, a K or V operand at a time for all of them.
template <int HD, bool Q8, bool BLOCKS, int QT>
struct Rows {
    static constexpr int NC = HD / 32, NU = HD / 16;
    typedef RawTile<HD, Q8, BLOCKS> Raw;
    Tile<HD, Q8, BLOCKS> t[QT];

    // The lane's 8 products (tokens 8 g .. 8 g + 7 of the tile) for its row of each tile, not yet times qf.
    __device__ __forceinline__ void scores(const Raw &k, float (&s)[QT][8]) const {
        // lo of q first; products that wait for each other lie 2 QT apart
        const f4_t zero = {0.f, 0.f, 0.f, 0.f};
        f4_t acc[QT][2];
        static_for<0, NC>([&](auto c_) __attribute__((always_inline)) {
            constexpr int c = decltype(c_)::value;
            constexpr bool kOwn = Q8 && !BLOCKS;  // a sum of its own for each block, for its scales
            const h8_t kf[2] = {k.frag(2 * c), k.frag(2 * c + 1)};
            f4_t x[QT][2];
#pragma unroll
            for (int i = 0; i < 2 * QT; ++i)
                x[i >> 1][i & 1] = mfma(kf[i & 1], t[i >> 1].ql[c], kOwn || c == 0 ? zero : acc[i >> 1][i & 1]);
#pragma unroll
            for (int i = 0; i < 2 * QT; ++i) x[i >> 1][i & 1] = mfma(kf[i & 1], t[i >> 1].qh[c], x[i >> 1][i & 1]);
#pragma unroll
            for (int q = 0; q < QT; ++q)
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const float z = x[q][n >> 2][n & 3];
                    acc[q][n >> 2][n & 3] = !kOwn ? z : fmaf(z, k.scale(c, n), c == 0 ? 0.f : acc[q][n >> 2][n & 3]);
                }
        });
#pragma unroll
        for (int q = 0; q < QT; ++q)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                s[q][n] = acc[q][n >> 2][n & 3];
                if constexpr (BLOCKS) s[q][n] = over_columns<NC>(fmaf(s[q][n], k.scale(0, n), 0.f));
            }
    }

    // m follows the tile's scores where a row's p would grow too large. q8_0: e likewise a larger scale of
    // V than any before, so that p times a scale stays within f16's range (below 2^16) and keeps its bits
    // whatever the scales' size.
    __device__ __forceinline__ void follow(const float (&s)[QT][8], const Raw &v) {
        float top[QT];
        int x = 0;
        bool behind = false;
        if constexpr (Q8) {
            x = v.top_exponent();
            behind = x > t[0].e;
        }
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            top[q] = t[q].top(s[q]);
            behind |= t[q].behind(top[q]);
        }
        if (__any(behind)) {  // wave-uniform
#pragma unroll
            for (int q = 0; q < QT; ++q) t[q].follow(top[q], x);
        }
    }

    // s becomes p, out += p V. MASKED: tokens whose p is 0 here may hold anything, inf and NaN among it.
    template <bool MASKED>
    __device__ __forceinline__ void values(const Raw &v, float (&s)[QT][8]) {
        if constexpr (Q8) {
#pragma unroll
            for (int q = 0; q < QT; ++q) t[q].probs(s[q]);
            auto scaled = [&](int q, int c, h8_t &ph, h8_t &pl) __attribute__((always_inline)) {
                float pd[8];
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    pd[n] = fmaf(s[q][n], v.scale(c, n), 0.f);
                    if (MASKED && s[q][n] == 0.f) pd[n] = 0.f;
                }
                split8(pd, ph, pl);
            };
            h8_t ph, pl;
            if constexpr (BLOCKS) scaled(0, 0, ph, pl);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const h8_t vf[2] = {v.frag(2 * c), v.frag(2 * c + 1)};
#pragma unroll
                for (int q = 0; q < QT; ++q) {
                    if constexpr (!BLOCKS) scaled(q, c, ph, pl);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        t[q].o[2 * c + u] = mfma(vf[u], ph, mfma(vf[u], pl, t[q].o[2 * c + u]));
                }
            }
        } else {
            const _Float16 w = _Float16(1.f);
            const h8_t one = {w, w, w, w, w, w, w, w};
#pragma unroll
            for (int q = 0; q < QT; ++q) {
                t[q].probs(s[q]);
                h8_t ph, pl;
                split8(s[q], ph, pl);
                t[q].l = mfma(one, pl, t[q].l);
#pragma unroll
                for (int u = 0; u < NU; ++u) t[q].o[u] = mfma(v.frag(u), pl, t[q].o[u]);
                t[q].l = mfma(one, ph, t[q].l);
#pragma unroll
                for (int u = 0; u < NU; ++u) t[q].o[u] = mfma(v.frag(u), ph, t[q].o[u]);
            }
        }
    }

    // After the last tile: a row's l as one sum, its out as it is.
    __device__ __forceinline__ float finish(int q) {
        if constexpr (Q8) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int n = 0; n < 4; ++n) t[q].o[u][n] = ldexpf(t[q].o[u][n], t[q].e);
            return ldexpf(rows_sum(t[q].l[0]), t[q].e);
        }
        return t[q].l[0];
    }
};

// What a workgroup works on: rows row0 .. of one sequence and K/V head, over a
// share of its tokens.
struct Work {
    KvSeq s;
    int i, head, split, group;
    __device__ __forceinline__ int sees(const KvAttn &a, int row) const {
        return a.causal ? max(0, s.ctx - s.n + row / group + 1) : s.ctx;
    }
    __device__ __forceinline__ size_t qrow(int row) const { return size_t(s.r0 + row / group); }
    __device__ __forceinline__ int qhead(int row) const { return head * group + row % group; }
};

// One row's result, or its part of one: lane 16 g + r holds dims 16 u + 4 g .. of the row.
template <int HD>
__device__ __forceinline__ void put_row(const KvAttn &a, const Work &w, int splits, int row, int u, int lane,
                                        const f4_t &o, float m, float l) {
    // m and l of a row are written once, with its dims 0 .. 3
    const int dim = 16 * u + 4 * (lane >> 4);
    if (splits == 1) {
        const f4_t y = l == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : o / l;
        *reinterpret_cast<f4_t *>(a.out + w.qrow(row) * a.ldo + size_t(w.qhead(row)) * HD + dim) = y;
    } else {
        float *part = a.scratch + ((w.qrow(row) * size_t(a.heads) + size_t(w.qhead(row))) * size_t(splits) +
                                   size_t(w.split)) * size_t(HD + kPartHead);
        if (l != 0.f) *reinterpret_cast<f4_t *>(part + kPartHead + dim) = o;
        if (dim == 0) {
            part[0] = m;
            part[1] = l;
        }
    }
}

// Many rows to a K/V head: two groups of many_qt tiles by two waves each.
constexpr int many_qt(int hd) { return hd <= 128 ? 2 : 1; }
constexpr int many_rows(int hd) { return 2 * many_qt(hd) * kRows; }

// RG groups of QT tiles of rows, by TG waves each that take every TG-th tile of tokens. Every wave
// reads its tiles straight into the registers that the matrix products take them from: K of the next
// tile is asked for once this one's is used, V likewise, so that one of them is always on its way.
//
// Few rows (single tokens) are bound by the cache's bytes: 3 contexts of 60002 .. 100003 tokens, 8 K/V
// heads of 128, f16, 961 MB in 150 us = 6.4 TB/s (a plain read of 1 GB: 7.1 TB/s with non-temporal loads,
// 6.4 without, which is why theirs are); 64 sequences of 91 .. 2301 tokens, 16 heads of 128, q8_0,
// 345 MB in 70 us = 4.9 TB/s: ragged ends, and the conversion of int8 to f16 beside the reads.
//
// Many rows (chunks) are bound by arithmetic, two matrix products for each of q k and p v and about as
// long again in the softmax and the splitting of p: 4001 rows over 8000 tokens, 16 heads of 64, f16, in
// 208 us = 472 TFLOP/s (944 of the products as made; a large f16 product of the library reaches 1115),
// q8_0 in 298 us. Waves of other rows read the same lines at about the same time, out of L1 and L2. Eight
// waves that shared tiles through LDS, a stage ahead, took 376 us against 241 us so at that time: a
// stage is worked on in less time than the next takes to come. Two groups by two waves: 236 us at that
// time, one by four 243, four by one 246; four tiles of rows to a wave 213 us against 208.
//
// Sequences of up to `skip` rows, or more than `limit`, are another shape's.
template <int HD, bool Q8, int QT, int RG, int TG, bool BLOCKS>
struct Shape {
    static constexpr int NC = BLOCKS ? HD / 32 : 1, NU = HD / 16;  // columns of a row
    static constexpr int kRowsWg = RG * QT * kRows / NC, kThreads = 64 * RG * TG;
    // waves of a SIMD: what the registers of a wave leave room for
    static constexpr int kWavesSimd =
        QT == 1 ? (HD <= 64 ? 4 : HD <= 128 ? (BLOCKS ? 3 : 2) : 1) : HD <= 64 && QT == 2 ? 3 : 2;
    // few rows: a K/V head's tiles are read by one workgroup alone, and not again soon
    static constexpr bool kOnce = RG == 1;
    struct Lds {
        f4_t o[TG][RG][QT][NU][64];
        float m[TG][RG][QT][kRows], l[TG][RG][QT][kRows];
    };
};

// Workgroup b of a launch of this shape.
template <int HD, bool Q8, int QT, int RG, int TG, bool BLOCKS>
__device__ __forceinline__ void attn(const KvPool &pool, const KvAttn &a, const KvRows &r, int group, int row_tiles,
                                     int splits, int skip, int limit, uint32_t b, void *lds) {
    typedef Shape<HD, Q8, QT, RG, TG, BLOCKS> S;
    static_assert(!BLOCKS || (Q8 && QT == 1 && RG == 1), "blocks as columns: one tile of few rows");
    constexpr int TB = kv_tile_bytes(Q8, HD), NU = HD / 16;
    auto &so = static_cast<typename S::Lds *>(lds)->o;
    auto &sm = static_cast<typename S::Lds *>(lds)->m;
    auto &sl = static_cast<typename S::Lds *>(lds)->l;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = w % RG, tg = w / RG;
    Work job;
    job.group = group;
    job.split = int(b % uint32_t(splits));
    b /= uint32_t(splits);
    // A K/V head's workgroups are as many apart as there are heads (with 8 or 16 of them all on one of
    // the 8 XCDs, whose L2 then reads the head's tiles once); the longest row tiles come first, so that
    // the short ones fill what is left at the end.
    const uint32_t pairs = uint32_t(pool.seqs) * uint32_t(pool.heads), pair = b % pairs;
    const int rt = row_tiles - 1 - int(b / pairs);
    job.head = int(pair % uint32_t(pool.heads));
    job.i = int(pair / uint32_t(pool.heads));
    const KvSeq s = job.s = kv_seq(pool, r, job.i);
    if (!s.ok && r.bad && threadIdx.x == 0) *r.bad = 1u;
    const int rows = s.n * group, first = rt * S::kRowsWg;
    if (first >= rows || rows <= skip || rows > limit) return;
    const int row0 = first + rg * QT * kRows;  // the wave's first row
    const bool busy = row0 < rows;
    const int lr = lane & 15, lrow = lr / S::NC;  // the lane's column, and its row in a tile
    // what the wave's first and last row see
    const int least = job.sees(a, min(row0, rows - 1)), most = busy ? job.sees(a, min(row0 + QT * kRows, rows) - 1) : 0;
    Rows<HD, Q8, BLOCKS, QT> wave;
    auto &t = wave.t;
#pragma unroll
    for (int j = 0; j < QT; ++j) {
        const int mine = row0 + j * kRows + lrow, row = min(mine, rows - 1);
        t[j].load_q(mine < rows ? a.q + job.qrow(row) * a.ldq + size_t(job.qhead(row)) * HD : nullptr, a.scale, lane);
        t[j].vis = job.sees(a, row);
    }
    // the split's tiles: the same for all of a workgroup's rows
    const int all = (job.sees(a, min(first + S::kRowsWg, rows) - 1) + kKvTile - 1) / kKvTile;
    const int per = max((all + splits - 1) / splits, kLeastTiles);
    const int end = min((most + kKvTile - 1) / kKvTile, (job.split + 1) * per);
    const uint32_t *table = pool.table + size_t(job.i) * size_t(pool.table_len);
    RawTile<HD, Q8, BLOCKS> kr, vr;
    auto page_of = [&](int kt) __attribute__((always_inline)) {
        return kt < end ? table[kt * kKvTile >> pool.shift] : 0xffffffffu;
    };
    // Always loads: where there is no such tile, or its page does not exist, from the pool's first one,
    // and the result is not used. (Loads that may not happen would have to be waited for at once.)
    const uint32_t in_page = (1u << (pool.shift - 5)) - 1u, to_v = (in_page + 1u) * TB;
    const uint32_t head_at = uint32_t(job.head) * 2u * to_v, page_bytes = uint32_t(pool.heads) * 2u * to_v;
    auto tile_of = [&](uint32_t page, int kt) __attribute__((always_inline)) {
        const bool there = page < uint32_t(pool.pages);
        const uint32_t in = there ? head_at + (uint32_t(kt) & in_page) * TB : 0u;
        return pool.pool + size_t(there ? page : 0u) * page_bytes + in;
    };
    int kt = job.split * per + tg;
    bool odd = false;
    uint32_t page = page_of(kt), next = page_of(kt + TG);
    constexpr bool kOnce = S::kOnce;
    const uint8_t *at = tile_of(page, kt);
    kr.template load<kOnce>(at, lane);
    vr.template load<kOnce>(at + to_v, lane);
    auto step = [&](auto masked) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        const int tok0 = kt * kKvTile;
        float p[QT][8];
        wave.scores(kr, p);
        at = tile_of(next, kt + TG);
        kr.template load<kOnce>(at, lane);
        if (page >= uint32_t(pool.pages)) {  // its tokens are not there
            if (r.bad && lane == 0) *r.bad = 1u;
#pragma unroll
            for (int q = 0; q < QT; ++q) t[q].hide(p[q], 0x7fffffe0);
            vr.clear();
        }
        if constexpr (kMasked) {
#pragma unroll
            for (int q = 0; q < QT; ++q) t[q].hide(p[q], tok0);
            odd |= vr.cut(s.ctx - tok0 - 8 * (lane >> 4));
        }
        wave.follow(p, vr);
        __builtin_amdgcn_iglp_opt(1);
        wave.template values<kMasked>(vr, p);
        vr.template load<kOnce>(at + to_v, lane);
        page = next;
        next = page_of(kt + 2 * TG);
    };
    const int whole = min(end, least / kKvTile);
    for (; kt < whole; kt += TG) step(std::false_type{});
    const int masked0 = kt;
    for (; kt < end; kt += TG) step(std::true_type{});
    if (__any(odd))  // wave-uniform
        for (kt = masked0; kt < end; kt += TG)
            if (const uint32_t id = page_of(kt); id < uint32_t(pool.pages))
#pragma unroll
                for (int q = 0; q < QT; ++q)
                    t[q].not_finite(tile_of(id, kt) + to_v, kt * kKvTile, s.ctx);
    // the results of the waves with the same rows meet in LDS
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        const float l = wave.finish(q);
        if (lane < kRows) {
            sm[tg][rg][q][lane] = t[q].m;
            sl[tg][rg][q][lane] = l;
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) so[tg][rg][q][u][lane] = t[q].o[u];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        const int row = row0 + q * kRows + lrow;
        float m = -INFINITY, l = 0.f, f[TG];
#pragma unroll
        for (int k = 0; k < TG; ++k) m = fmaxf(m, sm[k][rg][q][lr]);
#pragma unroll
        for (int k = 0; k < TG; ++k) {
            // a wave that saw no token adds nothing, whatever its zeros would be multiplied by
            const float lk = sl[k][rg][q][lr], mk = sm[k][rg][q][lr];
            f[k] = lk == 0.f ? 0.f : mk == m ? 1.f : __builtin_amdgcn_exp2f(mk - m);
            l += lk == 0.f ? 0.f : f[k] * lk;
        }
        if (row >= rows) continue;
        for (int u = tg; u < NU; u += TG) {
            if (BLOCKS && u >> 1 != lr % S::NC) continue;  // another column's
            f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < TG; ++k)
                if (sl[k][rg][q][lr] != 0.f) o += so[k][rg][q][u][lane] * f[k];
            put_row<HD>(a, job, splits, row, u, lane, o, m, l);
        }
    }
}

// The launches: few rows, many rows, and both at once (the first `few` workgroups are the few rows'),
// where the few rows' reads run beside the many rows' arithmetic.
template <int HD, bool Q8, bool BLOCKS>
using FewShape = Shape<HD, Q8, 1, 1, kWaves, BLOCKS>;
template <int HD, bool Q8>
using ManyShape = Shape<HD, Q8, many_qt(HD), 2, 2, false>;

template <int HD, bool Q8, bool BLOCKS>
__global__ __launch_bounds__(64 * kWaves, (FewShape<HD, Q8, BLOCKS>::kWavesSimd)) void k_attn_few(
    KvPool pool, KvAttn a, KvRows r, int group, int splits, int limit) {
    __shared__ typename FewShape<HD, Q8, BLOCKS>::Lds lds;
    attn<HD, Q8, 1, 1, kWaves, BLOCKS>(pool, a, r, group, 1, splits, 0, limit, blockIdx.x, &lds);
}
template <int HD, bool Q8>
__global__ __launch_bounds__(64 * kWaves, (ManyShape<HD, Q8>::kWavesSimd)) void k_attn_many(
    KvPool pool, KvAttn a, KvRows r, int group, int row_tiles, int splits) {
    __shared__ typename ManyShape<HD, Q8>::Lds lds;
    attn<HD, Q8, many_qt(HD), 2, 2, false>(pool, a, r, group, row_tiles, splits, 0, 0x7fffffff, blockIdx.x, &lds);
}
template <int HD, bool Q8>
__global__ __launch_bounds__(64 * kWaves, (ManyShape<HD, Q8>::kWavesSimd)) void k_attn_both(
    KvPool pool, KvAttn a, KvRows r, int group, int row_tiles, int splits, int limit, uint32_t few) {
    constexpr bool BLOCKS = Q8 && HD > 32;
    __shared__ union {
        typename FewShape<HD, Q8, BLOCKS>::Lds few;
        typename ManyShape<HD, Q8>::Lds many;
    } lds;
    if (blockIdx.x < few)
        attn<HD, Q8, 1, 1, kWaves, BLOCKS>(pool, a, r, group, 1, splits, 0, limit, blockIdx.x, &lds);
    else
        attn<HD, Q8, many_qt(HD), 2, 2, false>(pool, a, r, group, row_tiles, splits, limit, 0x7fffffff,
                                               blockIdx.x - few, &lds);
}

// Whether some sequence has the row, for the 64 / LANES rows of a wave at once (each the same in its
// LANES neighbouring lanes): a row that is none's, or past max_new of its own, is left alone.
template <int LANES>
__device__ __forceinline__ bool is_a_row(const KvPool &pool, const KvRows &r, size_t qrow) {
    const int lane = threadIdx.x & 63;
    if (!r.row_off) return qrow < size_t(pool.seqs) * size_t(r.max_new);
    const uint64_t mine = (LANES == 64 ? ~0ull : (1ull << LANES) - 1ull) << (lane / LANES * LANES);
    bool found = false;
    for (int i0 = 0; i0 < pool.seqs; i0 += LANES) {  // wave-uniform
        const int i = i0 + lane % LANES;
        bool in = false;
        if (i < pool.seqs) {
            const KvSeq s = kv_seq(pool, r, i);
            in = qrow >= size_t(s.r0) && qrow < size_t(s.r0) + size_t(s.n);
        }
        found |= (__ballot(in) & mine) != 0ull;
    }
    return found;
}

// The splits of a row joined in their order, a few of them: HD / 4 lanes to a (row, head). Bytes and one
// chain of reads: 2 shares of 1024 rows of 128 in 4.4 us.
template <int HD>
__global__ __launch_bounds__(256) void k_attn_join_few(KvPool pool, KvAttn a, KvRows r, int splits) {
    constexpr int LANES = HD / 4, PART = HD + kPartHead;
    const size_t job = (size_t(blockIdx.x) * 256 + threadIdx.x) / LANES, qrow = job / size_t(a.heads);
    const int head = int(job % size_t(a.heads)), lane = threadIdx.x % LANES;
    if (!is_a_row<LANES>(pool, r, qrow) || qrow >= size_t(r.rows)) return;
    const float *part = a.scratch + job * size_t(splits) * size_t(PART);
    float m = -INFINITY, l = 0.f;
    f4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < splits; k0 += 4) {
        float mk[4], lk[4];
        f4_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float *pk = part + size_t(min(k0 + j, splits - 1)) * PART;
            mk[j] = k0 + j < splits ? pk[0] : -INFINITY;
            lk[j] = k0 + j < splits ? pk[1] : 0.f;
            x[j] = *reinterpret_cast<const f4_t *>(pk + kPartHead + 4 * lane);  // not used where there is none
        }
        const float mn = fmaxf(fmaxf(fmaxf(mk[0], mk[1]), fmaxf(mk[2], mk[3])), m);
        const float down = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l = l == 0.f ? 0.f : l * down;
        o *= down;
        m = mn;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (lk[j] == 0.f) continue;  // a split that saw no token adds nothing (and has no out)
            const float f = mk[j] == m ? 1.f : __builtin_amdgcn_exp2f(mk[j] - m);
            l += f * lk[j];
            o += x[j] * f;
        }
    }
    const f4_t y = l == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : o / l;
    *reinterpret_cast<f4_t *>(a.out + qrow * a.ldo + size_t(head) * HD + 4 * lane) = y;
}

// The same for many: a workgroup to a (row, head), each wave a quarter of the splits. Lane k weighs the
// quarter's split k, all of their m and l read at once; then the outs, 16 bytes a lane, as many splits at
// a time as a wave has lanes for. The waves meet in LDS. (85 shares of 96 rows of 128: 11 us by one wave.)
template <int HD>
__global__ __launch_bounds__(256) void k_attn_join(KvPool pool, KvAttn a, KvRows r, int splits) {
    constexpr int LANES = HD / 4, AT = 64 / LANES, PART = HD + kPartHead;  // lanes of an out; outs at a time
    __shared__ float sm[kWaves], sl[kWaves];
    __shared__ f4_t so[kWaves][LANES];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const size_t job = blockIdx.x, qrow = job / size_t(a.heads);
    const int head = int(job % size_t(a.heads));
    if (!is_a_row<64>(pool, r, qrow) || qrow >= size_t(r.rows)) return;  // the workgroup's alike
    const float *part = a.scratch + job * size_t(splits) * size_t(PART);
    const int quarter = (splits + kWaves - 1) / kWaves, first = w * quarter, end = min(splits, first + quarter);
    float m = -INFINITY, l = 0.f;
    f4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = first; k0 < end; k0 += 64) {
        const int n = min(64, end - k0);
        const float *pk = part + size_t(k0) * PART;
        float mk = -INFINITY, lk = 0.f;
        if (lane < n) {
            mk = pk[size_t(lane) * PART];
            lk = pk[size_t(lane) * PART + 1];
        }
        const float mn = fmaxf(m, wave_max(mk)), down = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        // a split that saw no token adds nothing (and has no out)
        const float f = lk == 0.f ? 0.f : mk == mn ? 1.f : __builtin_amdgcn_exp2f(mk - mn);
        l = (l == 0.f ? 0.f : l * down) + wave_sum(lk == 0.f ? 0.f : f * lk);
        o *= down;
        m = mn;
        const int last = 64 - __builtin_clzll(__ballot(lk != 0.f) | 1ull);  // splits that have an out: below
        for (int k = 0; k < last; k += 4 * AT) {
            f4_t x[4];
            float fk[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int z = k + j * AT + lane / LANES;
                fk[j] = __shfl(f, z & 63);
                const float lz = __shfl(lk, z & 63);  // all lanes
                x[j] = f4_t{0.f, 0.f, 0.f, 0.f};
                if (z < last && lz != 0.f)
                    x[j] = *reinterpret_cast<const f4_t *>(pk + size_t(z) * PART + kPartHead + 4 * (lane % LANES));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) o += x[j] * fk[j];
        }
    }
#pragma unroll
    for (int d = LANES; d < 64; d *= 2)
#pragma unroll
        for (int n = 0; n < 4; ++n) o[n] += __shfl_xor(o[n], d);
    if (lane < LANES) so[w][lane] = o;
    if (lane == 0) {
        sm[w] = m;
        sl[w] = l;
    }
    __syncthreads();
    if (w > 0 || lane >= LANES) return;
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    l = 0.f;
    o = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        if (sl[k] == 0.f) continue;
        const float f = sm[k] == m ? 1.f : __builtin_amdgcn_exp2f(sm[k] - m);
        l += f * sl[k];
        o += so[k][lane] * f;
    }
    const f4_t y = l == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : o / l;
    *reinterpret_cast<f4_t *>(a.out + qrow * a.ldo + size_t(head) * HD + 4 * lane) = y;
}

// How a call is cut: sequences of up to `limit` rows to a K/V head (group * rows) to the few rows' shape,
// the others to the many rows', and the tokens of both into `splits` shares, none under 256 tokens.
struct Plan {
    int splits, tiles;        // shares; row tiles of the many rows' shape
    bool few, many, blocks;   // blocks: the few rows' columns are blocks (q8_0)
    int limit;
};
constexpr int kFewSplits = 8;  // above, a row's shares are more than its lanes read at once
Plan plan(const KvPool &p, bool q8, int hd, int heads, int rows, int max_new, int max_ctx, bool uniform) {
    Plan c;
    const long long most = (long long)max_new * (heads / p.heads);
    c.many = most > kRows;
    c.few = !c.many || !uniform;
    const int by_block = kRows / (hd / 32);
    c.blocks = q8 && hd > 32 && (c.many || most <= by_block);
    c.limit = c.blocks ? by_block : kRows;
    const int wg = many_rows(hd);
    c.tiles = int((most + wg - 1) / wg);
    // Workgroups without splits, of the shape that has the most of the work, and how many the GPU holds.
    const long long of_rows = ((long long)rows * (heads / p.heads) + wg - 1) / wg;
    const long long jobs = (long long)p.heads * (c.many ? of_rows : p.seqs);
    const int of_cu = c.many ? (hd <= 64 ? 3 : hd <= 128 ? 2 : 1) : hd <= 64 ? 4 : hd > 128 ? 1 : c.blocks ? 3 : 2;
    const int held = 256 * of_cu;
    // Many rows: as many as it holds; twice that for ragged sequences, whose longest would run alone at
    // the end otherwise (q8_0 mix of single tokens and chunks of 33 .. 517 rows: 90 us so, 100 us with three
    // times, 113 us unsplit; a chunk of 4001 rows: 208 us unsplit, 231 us in two).
    // Few rows: half as many again where the heads are too few to fill it (3 contexts of 60000 .. 100002
    // tokens, 8 heads: 150 us, 156 us with twice, 159 us with three times as many); else two shares for
    // up to 1024 heads, against ragged lengths (64 sequences of 91 .. 2301 tokens, 16 heads: 70 us, 73 us unsplit).
    const bool ragged = (long long)rows * 2 < (long long)p.seqs * max_new;
    const long long most_jobs = c.many ? (ragged ? 2 : 1) * held : jobs < held ? held + held / 2 : 2048;
    long long s = most_jobs / jobs;
    s = s < max_ctx / 256 ? s : max_ctx / 256;
    c.splits = s < 1 ? 1 : int(s);
    return c;
}

}  // namespace

size_t attn_paged_scratch(const KvPool &p, bool q8, int hd, int heads, int rows, int max_new, int max_ctx) {
    if (p.seqs <= 0 || rows <= 0) return 0;
    const int s = plan(p, q8, hd, heads, rows, max_new, max_ctx, false).splits;
    return s == 1 ? 0 : size_t(rows) * size_t(heads) * size_t(s) * size_t(hd + kPartHead) * sizeof(float);
}

namespace {
template <int HD, bool Q8>
hipError_t launch(const KvPool &p, const KvAttn &a, const KvRows &r, int max_ctx, hipStream_t st) {
    const int group = a.heads / p.heads;
    const Plan c = plan(p, Q8, HD, a.heads, r.rows, r.max_new, max_ctx, !r.row_off);
    if ((long long)r.max_new * group > 0x7fffffffll) return hipErrorInvalidValue;
    const long long pairs = (long long)p.seqs * p.heads * c.splits, many = pairs * c.tiles;
    const bool few = c.splits <= kFewSplits;
    const int per = few ? 256 / (HD / 4) : 1;  // (row, head)s of a workgroup of the join
    const long long joins = ((long long)r.rows * a.heads + per - 1) / per;
    if (pairs + many > 0x7fffffffll || joins > 0x7fffffffll) return hipErrorInvalidValue;
    constexpr bool kByBlock = Q8 && HD > 32;
    const dim3 threads(64 * kWaves);
    if (c.many && c.few)
        hipLaunchKernelGGL((k_attn_both<HD, Q8>), dim3(unsigned(pairs + many)), threads, 0, st, p, a, r, group, c.tiles,
                           c.splits, c.limit, unsigned(pairs));
    else if (c.many)
        hipLaunchKernelGGL((k_attn_many<HD, Q8>), dim3(unsigned(many)), threads, 0, st, p, a, r, group, c.tiles,
                           c.splits);
    else if (c.blocks)
        hipLaunchKernelGGL((k_attn_few<HD, Q8, kByBlock>), dim3(unsigned(pairs)), threads, 0, st, p, a, r, group,
                           c.splits, c.limit);
    else
        hipLaunchKernelGGL((k_attn_few<HD, Q8, false>), dim3(unsigned(pairs)), threads, 0, st, p, a, r, group, c.splits,
                           c.limit);
    if (c.splits > 1 && few)
        hipLaunchKernelGGL((k_attn_join_few<HD>), dim3(unsigned(joins)), dim3(256), 0, st, p, a, r, c.splits);
    if (c.splits > 1 && !few)
        hipLaunchKernelGGL((k_attn_join<HD>), dim3(unsigned(joins)), dim3(256), 0, st, p, a, r, c.splits);
    return hipGetLastError();
}
}  // namespace

hipError_t attn_paged(const KvPool &p, bool q8, int hd, const KvAttn &a, const KvRows &r, int max_ctx, hipStream_t st) {
    if (p.seqs <= 0 || r.rows <= 0) return hipSuccess;
    switch (hd) {
    case 32: return q8 ? launch<32, true>(p, a, r, max_ctx, st) : launch<32, false>(p, a, r, max_ctx, st);
    case 64: return q8 ? launch<64, true>(p, a, r, max_ctx, st) : launch<64, false>(p, a, r, max_ctx, st);
    case 128: return q8 ? launch<128, true>(p, a, r, max_ctx, st) : launch<128, false>(p, a, r, max_ctx, st);
    case 256: return q8 ? launch<256, true>(p, a, r, max_ctx, st) : launch<256, false>(p, a, r, max_ctx, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace mlg

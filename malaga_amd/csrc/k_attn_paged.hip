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
// f16(x - hi): 22 bits), which doubles the matrix work. q is scaled by a power of two per row and p by
// 2^15 (its maximum is 1) so that what lo loses below f16's range is 2^-29 of the largest value. Sums
// are f32.
#include <type_traits>

#include "device.hpp"
#include "paged_kv.hpp"

namespace mlg {
namespace {

constexpr int kRows = 16;        // rows of a query tile (columns of the matrix products)
constexpr int kWaves = 4;        // waves of a workgroup
constexpr float kPShift = 15.f;  // p is held times 2^15

// Partial result of a split: [m, l, -, -, out of HD dims] of one row, f32, as a Tile holds them.
constexpr int kPartHead = 4;

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ h8_t as_h8(const uint4 &v) { return __builtin_bit_cast(h8_t, v); }

// 8 int8 as f16, exactly: byte + 128 becomes the low byte of 1024 + u, minus 1152.
__device__ __forceinline__ h8_t i8_to_h8(uint32_t lo, uint32_t hi) {
    const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
    const h2_t off = {_Float16(1152.f), _Float16(1152.f)};
    const uint4 w = make_uint4(
        __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, a, 0x07010700u)) - off),
        __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, a, 0x07030702u)) - off),
        __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, b, 0x07010700u)) - off),
        __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, b, 0x07030702u)) - off));
    return as_h8(w);
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
template <int HD, bool Q8>
struct RawTile {
    static constexpr int NC = HD / 32, NP = Q8 ? NC : 2 * NC, ND = Q8 ? NC : 1;
    uint4 a[NP];
    uint4 d[ND];  // q8_0: the scales of the lane's tokens 8 g .. 8 g + 7, per block of 32 dims
    __device__ __forceinline__ void load(const uint8_t *tile, int lane) {
#pragma unroll
        for (int i = 0; i < NP; ++i) a[i] = *reinterpret_cast<const uint4 *>(tile + (i * 64 + lane) * 16);
        if constexpr (Q8) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
                d[c] = *reinterpret_cast<const uint4 *>(tile + kv_scale_byte(HD, 8 * (lane >> 4), c));
        }
    }
};

// The same as matrix operands: K's product b of dims 32 c .. at 2 c + b, V's dims 16 u .. at u.
template <int HD, bool Q8>
struct Frags {
    static constexpr int NC = HD / 32, NU = HD / 16;
    h8_t a[NU];
    uint4 d[Q8 ? NC : 1];
    __device__ __forceinline__ void from(const RawTile<HD, Q8> &r) {
        if constexpr (Q8) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                a[2 * c] = i8_to_h8(r.a[c].x, r.a[c].y);
                a[2 * c + 1] = i8_to_h8(r.a[c].z, r.a[c].w);
                d[c] = r.d[c];
            }
        } else {
#pragma unroll
            for (int u = 0; u < NU; ++u) a[u] = as_h8(r.a[u]);
        }
    }
    __device__ __forceinline__ float scale(int c, int n) const {
        const uint32_t w[4] = {d[c].x, d[c].y, d[c].z, d[c].w};
        return float(__builtin_bit_cast(h2_t, w[n >> 1])[n & 1]);
    }
    // V's tokens past the first `keep` of the lane's eight as zeros (of q8_0, their scales): they are
    // whatever the page held before. f16: what is left of inf and NaN as zeros too, which 0 would turn
    // into NaN for the rows that do not see its token; whether there was any (see not_finite).
    __device__ __forceinline__ bool cut(int keep) {
        bool odd = false;
        constexpr int N = Q8 ? NC : NU;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint4 v = Q8 ? d[Q8 ? i : 0] : __builtin_bit_cast(uint4, a[i]);
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                w[n] = keep > 2 * n + 1 ? w[n] : keep > 2 * n ? w[n] & 0xffffu : 0u;
                if constexpr (!Q8) {
                    const bool lo = (w[n] & 0x7c00u) == 0x7c00u, hi = (w[n] & 0x7c000000u) == 0x7c000000u;
                    odd |= lo || hi;
                    w[n] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                }
            }
            if constexpr (Q8) d[i] = make_uint4(w[0], w[1], w[2], w[3]);
            else a[i] = as_h8(make_uint4(w[0], w[1], w[2], w[3]));
        }
        return odd;
    }
};

// Two f16 operands of 8 f32 values: hi truncated, lo the rest, truncated too (2^-20 of x at most,
// 2^-22 on average; rounding lo to nearest measured 4 more operations per pair of values).
__device__ __forceinline__ void split8(const float (&p)[8], h8_t &hi, h8_t &lo) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        // p as finished f32 values: hi's and lo's uses of a product are otherwise rounded apart
        float x = p[2 * n], y = p[2 * n + 1];
        asm("" : "+v"(x), "+v"(y));
        const h2_t t = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(x, y));
        h[n] = __builtin_bit_cast(uint32_t, t);
        l[n] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf(float(t[0]), -1.f, x), fmaf(float(t[1]), -1.f, y)));
    }
    hi = as_h8(make_uint4(h[0], h[1], h[2], h[3]));
    lo = as_h8(make_uint4(l[0], l[1], l[2], l[3]));
}

__device__ __forceinline__ f4_t mfma(const h8_t &a, const h8_t &b, const f4_t &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A tile of 16 rows, and the softmax and sums of what it has seen.
template <int HD, bool Q8>
struct Tile {
    static constexpr int NC = HD / 32, NU = HD / 16;
    h8_t qh[NC], ql[NC];
    float qf;    // scores in log2 units: qf (above 0) times the product of the scaled q
    int vis;     // tokens that this lane's row sees
    float m;     // the running maximum (log2 units) less kPShift, as rounded: p = 2^(s - m)
    f4_t l;      // f16: sum of p over all tokens so far, in each element; q8_0: l[0] over the lane's
    f4_t o[NU];
    int e;       // q8_0: out is held times 2^-e (e: the largest exponent of V's scales so far)

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
        }
        amax = rows_max(amax);
        // the row's largest value to [2^14, 2^15); not for 0, inf (NaN is not seen by the maximum)
        const int up = amax > 0.f && amax < INFINITY ? 14 - ilogbf(amax) : 0;
        const float sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
        // not 0: what a row does not see scores -inf, also at a scale of 0
        qf = fmaxf(ldexpf(scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896340736f, -up), 1.17549435e-38f);
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
        e = -100;
#pragma unroll
        for (int u = 0; u < NU; ++u) o[u] = f4_t{0.f, 0.f, 0.f, 0.f};
    }

    // The lane's 8 products (tokens 8 g .. 8 g + 7 of the tile, its row), not yet times qf.
    __device__ __forceinline__ void scores(const Frags<HD, Q8> &k, float (&s)[8]) const {
        f4_t acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if constexpr (Q8) {
                    f4_t t = mfma(k.a[2 * c + b], qh[c], mfma(k.a[2 * c + b], ql[c], f4_t{0.f, 0.f, 0.f, 0.f}));
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[b][i] = fmaf(t[i], k.scale(c, 4 * b + i), acc[b][i]);
                } else {
                    acc[b] = mfma(k.a[2 * c + b], qh[c], mfma(k.a[2 * c + b], ql[c], acc[b]));
                }
            }
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = acc[n >> 2][n & 3];
    }

    // s becomes p (times 2^15); m, l and out follow a larger maximum.
    __device__ __forceinline__ void softmax(float (&s)[8]) {
        float t = vmax3(vmax3(s[0], s[1], s[2]), vmax3(s[3], s[4], s[5]), vmax(s[6], s[7]));
        t = fmaf(rows_max(t), qf, -kPShift);
        if (__any(t > m)) {  // wave-uniform
            const float mn = fmaxf(m, t), al = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int u = 0; u < NU; ++u) o[u] *= al;
            m = mn;
        }
        const float base = m == -INFINITY ? 0.f : m;  // nothing seen: every score is -inf
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = __builtin_amdgcn_exp2f(fmaf(s[n], qf, -base));
        if constexpr (Q8) l[0] += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    }

    // q8_0: out follows a larger scale of V than any before, so that p times a scale stays within
    // f16's range (below 2^16) and keeps its bits whatever the scales' size.
    __device__ __forceinline__ void fit(const Frags<HD, Q8> &v) {
        // f16 bit patterns of scales that are not negative are ordered; two at once
        typedef uint16_t u2_t __attribute__((ext_vector_type(2)));
        u2_t t2 = {0, 0};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const uint32_t w[4] = {v.d[c].x, v.d[c].y, v.d[c].z, v.d[c].w};
#pragma unroll
            for (int n = 0; n < 4; ++n) t2 = __builtin_elementwise_max(t2, __builtin_bit_cast(u2_t, w[n]));
        }
        uint32_t top = rows_umax(max(uint32_t(t2[0]), uint32_t(t2[1])));
        if (__any(top >= 0x7c00u)) {  // inf, NaN (no scale is negative): the other tokens' rows go on
            top = 0u;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const uint32_t w[4] = {v.d[c].x, v.d[c].y, v.d[c].z, v.d[c].w};
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const uint32_t b = w[n >> 1] >> (16 * (n & 1)) & 0xffffu;
                    top = max(top, b >= 0x7c00u ? 0u : b);
                }
            }
            top = rows_umax(top);
        }
        // the exponent of an f16; subnormals count as the smallest normal one
        const int x = top ? max(int(top >> 10), 1) - 15 : e;
        if (__any(x > e)) {
            const int en = max(e, x);
            const float f = ldexpf(1.f, max(e - en, -126));
#pragma unroll
            for (int u = 0; u < NU; ++u) o[u] *= f;
            e = en;
        }
    }

    // out += p V. MASKED: tokens whose p is 0 here may hold anything, inf and NaN among it.
    template <bool MASKED>
    __device__ __forceinline__ void values(const Frags<HD, Q8> &v, const float (&p)[8]) {
        h8_t ph, pl;
        if constexpr (Q8) {
            fit(v);
            const float down = ldexpf(1.f, -e);
            float pe[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) pe[n] = p[n] * down;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float pd[8];
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    pd[n] = fmaf(pe[n], v.scale(c, n), 0.f);
                    if (MASKED && p[n] == 0.f) pd[n] = 0.f;
                }
                split8(pd, ph, pl);
#pragma unroll
                for (int u = 2 * c; u < 2 * c + 2; ++u) o[u] = mfma(v.a[u], ph, mfma(v.a[u], pl, o[u]));
            }
        } else {
            split8(p, ph, pl);
            const _Float16 w = _Float16(1.f);
            const h8_t one = {w, w, w, w, w, w, w, w};
            l = mfma(one, ph, mfma(one, pl, l));
#pragma unroll
            for (int u = 0; u < NU; ++u) o[u] = mfma(v.a[u], ph, mfma(v.a[u], pl, o[u]));
        }
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
                    const uint32_t x = reinterpret_cast<const uint16_t *>(tile)[kv_v_elem(false, tk, 16 * u + 4 * g + i)];
                    if (sees && (x & 0x7c00u) == 0x7c00u) o[u][i] += h2f(x);
                }
        }
    }

    __device__ __forceinline__ void hide(float (&s)[8], int tok0) const {
        const int at = tok0 + 8 * (int(threadIdx.x & 63) >> 4);
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = at + n < vis ? s[n] : -INFINITY;
    }

    // After the last tile: l as one sum of the row, out as it is.
    __device__ __forceinline__ float finish() {
        if constexpr (Q8) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int n = 0; n < 4; ++n) o[u][n] = ldexpf(o[u][n], e);
            return rows_sum(l[0]);
        }
        return l[0];
    }
};

// What a workgroup of either kernel works on: rows row0 .. of one sequence and K/V head, over a
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
    const int dim = 16 * u + 4 * (lane >> 4);
    if (splits == 1) {
        const f4_t y = l == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : o / l;
        *reinterpret_cast<f4_t *>(a.out + w.qrow(row) * a.ldo + size_t(w.qhead(row)) * HD + dim) = y;
    } else {
        float *part = a.scratch + ((w.qrow(row) * size_t(a.heads) + size_t(w.qhead(row))) * size_t(splits) +
                                   size_t(w.split)) * size_t(HD + kPartHead);
        *reinterpret_cast<f4_t *>(part + kPartHead + dim) = o;
        if (u == 0 && lane < kRows) {
            part[0] = m;
            part[1] = l;
        }
    }
}

// ---- few rows to a K/V head: each wave reads its own tiles straight into registers ----
template <int HD, bool Q8>
__global__ __launch_bounds__(256, HD <= 64 ? 3 : HD <= 128 ? 2 : 1) void k_attn_rows(KvPool pool, KvAttn a, KvRows r,
                                                                                     int group, int splits) {
    constexpr int TB = kv_tile_bytes(Q8, HD), NU = HD / 16;
    __shared__ float sm[kWaves][kRows], sl[kWaves][kRows];
    __shared__ f4_t so[kWaves][NU][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t b = blockIdx.x;
    Work job;
    job.group = group;
    job.split = int(b % uint32_t(splits));
    b /= uint32_t(splits);
    job.head = int(b % uint32_t(pool.heads));
    job.i = int(b / uint32_t(pool.heads));
    const KvSeq s = job.s = kv_seq(pool, r, job.i);
    if (!s.ok && r.bad && threadIdx.x == 0) *r.bad = 1u;
    const int rows = s.n * group;
    if (rows == 0 || rows > kRows) return;  // more: k_attn_chunk's
    // this lane's row, and the tokens that it and the tile's first and last row see
    const int row = min(lane & 15, rows - 1);
    const int least = job.sees(a, 0), most = job.sees(a, rows - 1);
    const bool have = (lane & 15) < rows;
    Tile<HD, Q8> t;
    t.load_q(have ? a.q + job.qrow(row) * a.ldq + size_t(job.qhead(row)) * HD : nullptr, a.scale, lane);
    t.vis = job.sees(a, row);
    const int tiles = (most + kKvTile - 1) / kKvTile, per = (tiles + splits - 1) / splits;
    const int end = min(tiles, (job.split + 1) * per);
    const uint32_t *table = pool.table + size_t(job.i) * size_t(pool.table_len);
    // K of the next tile is asked for once this one's is used, V likewise: one of them is always on its way
    RawTile<HD, Q8> kr, vr;
    auto page_of = [&](int kt) { return kt < end ? table[kt * kKvTile >> pool.shift] : 0xffffffffu; };
    auto load = [&](RawTile<HD, Q8> &x, int which, uint32_t page, int kt) __attribute__((always_inline)) {
        if (page < uint32_t(pool.pages))
            x.load(pool.pool + pool.tile_at(page, job.head, which, kt * kKvTile, TB), lane);
    };
    int kt = job.split * per + w;
    bool odd = false;
    uint32_t page = page_of(kt), next = page_of(kt + kWaves);
    load(kr, 0, page, kt);
    load(vr, 1, page, kt);
    auto step = [&](auto masked) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        const int tok0 = kt * kKvTile;
        const bool there = page < uint32_t(pool.pages);
        float p[8];
        Frags<HD, Q8> f;
        if (there) {
            f.from(kr);
            t.scores(f, p);
        } else if (r.bad && lane == 0) {  // its tokens are not there
            *r.bad = 1u;
        }
        load(kr, 0, next, kt + kWaves);
        if (there) {
            if constexpr (kMasked) t.hide(p, tok0);
            t.softmax(p);
            f.from(vr);
        }
        load(vr, 1, next, kt + kWaves);
        if (there) {
            if constexpr (kMasked) odd |= f.cut(s.ctx - tok0 - 8 * (lane >> 4));
            t.template values<kMasked>(f, p);
        }
        page = next;
        next = page_of(kt + 2 * kWaves);
    };
    const int whole = min(end, least / kKvTile);
    for (; kt < whole; kt += kWaves) step(std::false_type{});
    const int masked0 = kt;
    for (; kt < end; kt += kWaves) step(std::true_type{});
    if (__any(odd))  // wave-uniform
        for (kt = masked0; kt < end; kt += kWaves)
            if (const uint32_t id = page_of(kt); id < uint32_t(pool.pages))
                t.not_finite(pool.pool + pool.tile_at(id, job.head, 1, kt * kKvTile, TB), kt * kKvTile, s.ctx);
    // the waves' results meet in LDS
    const float lw = t.finish();
    if (lane < kRows) {
        sm[w][lane] = t.m;
        sl[w][lane] = lw;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) so[w][u][lane] = t.o[u];
    __syncthreads();
    float m = -INFINITY, l = 0.f, f[kWaves];
    const int lr = lane & 15;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) m = fmaxf(m, sm[k][lr]);
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        // a wave without tokens adds nothing, whatever its zeros would be multiplied by
        f[k] = sl[k][lr] == 0.f ? 0.f : sm[k][lr] == m ? 1.f : __builtin_amdgcn_exp2f(sm[k][lr] - m);
        l += sl[k][lr] == 0.f ? 0.f : f[k] * sl[k][lr];
    }
    if (!have) return;
    for (int u = w; u < NU; u += kWaves) {
        f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kWaves; ++k)
            if (sl[k][lr] != 0.f) o += so[k][u][lane] * f[k];
        put_row<HD>(a, job, splits, row, u, lane, o, m, l);
    }
}

// ---- many rows to a K/V head: the workgroup's waves share the tiles through LDS ----
// Eight waves: four groups of QT tiles of rows, twice, one for each of the two tiles of tokens that a
// stage holds (four waves alone left the SIMDs with two waves each, and neither the matrix unit nor
// the VALU busy). A stage is fetched into registers while the one before it is worked on, then
// (q8_0: as f16) put into the other half of LDS: one barrier a stage, and each line of the cache is
// read once for 64 QT rows. The two halves' results meet in LDS at the end.
template <int HD, bool Q8>
struct Chunk {
    static constexpr int QT = HD <= 128 ? 2 : 1, ST = 2, kWavesWg = 8;
    static constexpr int kRowsWg = 4 * QT * kRows;
    static constexpr int NU = HD / 16, NC = HD / 32;
    static constexpr int kFragBytes = NU * 1024, kScaleBytes = Q8 ? NC * 64 : 0;
    static constexpr int kTileLds = kFragBytes + kScaleBytes;  // of K or V
    static_assert(4 * QT * NU * 1024 <= 2 * ST * 2 * kTileLds, "half of the waves' out fits the stages' LDS");
};

template <int HD, bool Q8>
__global__ __launch_bounds__(512, HD <= 64 ? 4 : 2) void k_attn_chunk(KvPool pool, KvAttn a, KvRows r, int group,
                                                                      int row_tiles, int splits, int skip) {
    typedef Chunk<HD, Q8> C;
    constexpr int TB = kv_tile_bytes(Q8, HD), NU = HD / 16, QT = C::QT, ST = C::ST;
    __shared__ uint8_t lds[2][ST][2][C::kTileLds] __attribute__((aligned(16)));
    __shared__ float sml[2][4][QT][kRows];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = w & 3, kg = w >> 2;
    uint32_t b = blockIdx.x;
    Work job;
    job.group = group;
    job.split = int(b % uint32_t(splits));
    b /= uint32_t(splits);
    // A K/V head's workgroups are as many apart as there are heads (with 8 or 16 of them all on one of
    // the 8 XCDs, whose L2 then reads the head's tiles once); the longest row tiles come first, and
    // every other 256 workgroups in reverse, so that a CU's long ones meet short ones.
    const uint32_t pairs = uint32_t(pool.seqs) * uint32_t(pool.heads), pair = b % pairs;
    int rank = int(b / pairs);
    const int turn = max(1, int(256u / pairs)), fold = rank / turn;
    if ((fold & 1) && (fold + 1) * turn <= row_tiles) rank = fold * turn + (turn - 1 - rank % turn);
    const int rt = row_tiles - 1 - rank;
    job.head = int(pair % uint32_t(pool.heads));
    job.i = int(pair / uint32_t(pool.heads));
    const KvSeq s = job.s = kv_seq(pool, r, job.i);
    if (!s.ok && r.bad && threadIdx.x == 0) *r.bad = 1u;
    const int rows = s.n * group, first = rt * C::kRowsWg;
    if (first >= rows || rows <= skip) return;  // skip: k_attn_rows' sequences
    const int wg_most = job.sees(a, min(first + C::kRowsWg, rows) - 1);
    const int row0 = first + rg * QT * kRows;  // the wave's first row
    const bool busy = row0 < rows;
    const int most = job.sees(a, min(row0 + QT * kRows, rows) - 1);
    Tile<HD, Q8> t[QT];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
        const int mine = row0 + j * kRows + (lane & 15), row = min(mine, rows - 1);
        t[j].load_q(mine < rows ? a.q + job.qrow(row) * a.ldq + size_t(job.qhead(row)) * HD : nullptr, a.scale, lane);
        t[j].vis = job.sees(a, row);
    }
    const int tiles = (wg_most + kKvTile - 1) / kKvTile;
    const int per = ((tiles + splits - 1) / splits + ST - 1) / ST * ST;
    const int begin = job.split * per, end = min(tiles, begin + per);
    const uint32_t *table = pool.table + size_t(job.i) * size_t(pool.table_len);

    // a thread's share of a stage: 16-byte pieces of the tiles' K and V, and of q8_0's scales
    constexpr int NP = Q8 ? HD / 32 : HD / 16;  // 1 KB pieces of a tile
    constexpr int ALL = ST * 2 * NP, NPER = ALL > C::kWavesWg ? ALL / C::kWavesWg : 1;  // pieces; of a wave
    static_assert(ALL <= C::kWavesWg || ALL % C::kWavesWg == 0, "pieces to waves");
    constexpr int NS = C::NC * 4;  // 16-byte pieces of a tile's scales
    u4_t raw[NPER], rsc = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int n = 0; n < NPER; ++n) raw[n] = rsc;
    uint32_t pages[ST], coming[ST];
    auto pages_of = [&](int kt, uint32_t (&p)[ST]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < ST; ++j) p[j] = kt + j < end ? table[(kt + j) * kKvTile >> pool.shift] : 0xffffffffu;
    };
    auto fetch = [&](int kt, const uint32_t (&p)[ST]) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NPER; ++n) {
            const int pc = w * NPER + n, j = pc / (2 * NP), which = pc / NP % 2, q = pc % NP;
            const uint32_t page = j ? p[1] : p[0];
            if (pc < ALL && page < uint32_t(pool.pages))
                raw[n] = *reinterpret_cast<const u4_t *>(
                    pool.pool + pool.tile_at(page, job.head, which, (kt + j) * kKvTile, TB) + (q * 64 + lane) * 16);
        }
        if constexpr (Q8) {
            const int pc = int(threadIdx.x), j = pc / (2 * NS), which = pc / NS % 2, q = pc % NS;
            const uint32_t page = j ? p[1] : p[0];
            if (pc < ST * 2 * NS && page < uint32_t(pool.pages))
                rsc = *reinterpret_cast<const u4_t *>(
                    pool.pool + pool.tile_at(page, job.head, which, (kt + j) * kKvTile, TB) + 32 * HD + q * 16);
        }
    };
    auto keep = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NPER; ++n) {
            const int pc = w * NPER + n, j = pc / (2 * NP), which = pc / NP % 2, q = pc % NP;
            if (pc >= ALL) continue;
            uint8_t *at = lds[buf][j][which];
            if constexpr (Q8) {
                *reinterpret_cast<h8_t *>(at + ((2 * q) * 64 + lane) * 16) = i8_to_h8(raw[n][0], raw[n][1]);
                *reinterpret_cast<h8_t *>(at + ((2 * q + 1) * 64 + lane) * 16) = i8_to_h8(raw[n][2], raw[n][3]);
            } else {
                *reinterpret_cast<u4_t *>(at + (q * 64 + lane) * 16) = raw[n];
            }
        }
        if constexpr (Q8) {
            const int pc = int(threadIdx.x), j = pc / (2 * NS), which = pc / NS % 2, q = pc % NS;
            if (pc < ST * 2 * NS) *reinterpret_cast<u4_t *>(lds[buf][j][which] + C::kFragBytes + q * 16) = rsc;
        }
    };
    auto read = [&](Frags<HD, Q8> &f, const uint8_t *at) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NU; ++u) f.a[u] = *reinterpret_cast<const h8_t *>(at + (u * 64 + lane) * 16);
        if constexpr (Q8) {
#pragma unroll
            for (int c = 0; c < C::NC; ++c)
                f.d[c] = *reinterpret_cast<const uint4 *>(at + C::kFragBytes + c * 64 + (lane >> 4) * 16);
        }
    };

    if (begin < end) {
        pages_of(begin, pages);
        fetch(begin, pages);
        pages_of(begin + ST, coming);
        keep(0);
    }
    int buf = 0, kt = begin;
    bool odd = false;
    auto stage = [&](auto masked) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        __syncthreads();  // this stage is in LDS, and the other half is no longer read
        if (kt + ST < end) fetch(kt + ST, coming);
        const int tok0 = (kt + kg) * kKvTile;
        const uint32_t page = kg ? pages[1] : pages[0];
        const bool there = page < uint32_t(pool.pages);
        if (!there && kt + kg < end && r.bad && lane == 0) *r.bad = 1u;  // its tokens are not there
        if (busy && there && (!kMasked || tok0 < most)) {
            float p[QT][8];
            Frags<HD, Q8> f;
            read(f, lds[buf][kg][0]);
#pragma unroll
            for (int q = 0; q < QT; ++q) t[q].scores(f, p[q]);
            if constexpr (kMasked) {
#pragma unroll
                for (int q = 0; q < QT; ++q) t[q].hide(p[q], tok0);
            }
#pragma unroll
            for (int q = 0; q < QT; ++q) t[q].softmax(p[q]);
            read(f, lds[buf][kg][1]);
            if constexpr (kMasked) odd |= f.cut(s.ctx - tok0 - 8 * (lane >> 4));
#pragma unroll
            for (int q = 0; q < QT; ++q) t[q].template values<kMasked>(f, p[q]);
        }
        if (kt + ST < end) keep(buf ^ 1);
#pragma unroll
        for (int j = 0; j < ST; ++j) pages[j] = coming[j];
        pages_of(kt + 2 * ST, coming);
        buf ^= 1;
    };
    // the same for every wave: stages that the workgroup's first row sees whole, then the others
    const int whole = min(end, job.sees(a, first) / kKvTile) - (ST - 1);
    for (; kt < whole; kt += ST) stage(std::false_type{});
    const int masked0 = kt;
    for (; kt < end; kt += ST) stage(std::true_type{});
    if (__any(odd))  // wave-uniform
        for (kt = masked0 + kg; kt < end; kt += ST)
            if (const uint32_t id = table[kt * kKvTile >> pool.shift]; id < uint32_t(pool.pages) && kt * kKvTile < most)
#pragma unroll
                for (int q = 0; q < QT; ++q)
                    t[q].not_finite(pool.pool + pool.tile_at(id, job.head, 1, kt * kKvTile, TB), kt * kKvTile, s.ctx);

    // the halves meet: the second one's out in LDS, [row group][QT][NU][lane]
    f4_t *const so = reinterpret_cast<f4_t *>(&lds[0][0][0][0]) + rg * QT * NU * 64 + lane;
    __syncthreads();
    float l[QT];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        l[q] = t[q].finish();
        if (kg == 1 && lane < kRows) {
            sml[0][rg][q][lane] = t[q].m;
            sml[1][rg][q][lane] = l[q];
        }
        if (kg == 1) {
#pragma unroll
            for (int u = 0; u < NU; ++u) so[(q * NU + u) * 64] = t[q].o[u];
        }
    }
    __syncthreads();
    if (!busy || kg == 1) return;
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        const int mine = row0 + q * kRows + (lane & 15);
        const float m1 = sml[0][rg][q][lane & 15], l1 = sml[1][rg][q][lane & 15], m = fmaxf(t[q].m, m1);
        // a half that saw no token adds nothing, whatever its zeros would be multiplied by
        const bool h0 = l[q] != 0.f, h1 = l1 != 0.f;
        const float f0 = t[q].m == m ? 1.f : __builtin_amdgcn_exp2f(t[q].m - m);
        const float f1 = m1 == m ? 1.f : __builtin_amdgcn_exp2f(m1 - m);
        const float sum = (h0 ? l[q] * f0 : 0.f) + (h1 ? l1 * f1 : 0.f);
        if (mine < rows) {
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                f4_t o = {0.f, 0.f, 0.f, 0.f};
                if (h0) o += t[q].o[u] * f0;
                if (h1) o += so[(q * NU + u) * 64] * f1;
                put_row<HD>(a, job, splits, mine, u, lane, o, m, sum);
            }
        }
    }
}

// The splits of a row joined in their order: a wave per (row, head).
template <int HD>
__global__ __launch_bounds__(256) void k_attn_join(KvPool pool, KvAttn a, KvRows r, int splits) {
    const int lane = threadIdx.x & 63;
    const size_t job = size_t(blockIdx.x) * kWaves + (threadIdx.x >> 6);
    const size_t per = size_t(r.max_new) * size_t(a.heads);
    const int i = int(job / per);
    if (i >= pool.seqs) return;
    const KvSeq s = kv_seq(pool, r, i);
    const int row = int(job % per / size_t(a.heads)), head = int(job % size_t(a.heads));
    if (row >= s.n) return;
    const size_t qrow = size_t(s.r0 + row);
    const float *part = a.scratch + (qrow * size_t(a.heads) + size_t(head)) * size_t(splits) * size_t(HD + kPartHead);
    float m = -INFINITY, l = 0.f;
    for (int k = 0; k < splits; ++k) m = fmaxf(m, part[size_t(k) * (HD + kPartHead)]);
    constexpr int ND = (HD + 63) / 64;
    float o[ND];
#pragma unroll
    for (int n = 0; n < ND; ++n) o[n] = 0.f;
    for (int k = 0; k < splits; ++k) {
        const float *pk = part + size_t(k) * (HD + kPartHead);
        const float mk = pk[0], lk = pk[1];
        if (lk == 0.f) continue;  // no token of this split seen
        const float f = mk == m ? 1.f : __builtin_amdgcn_exp2f(mk - m);
        l += f * lk;
#pragma unroll
        for (int n = 0; n < ND; ++n)
            if (HD >= 64 || lane < HD) o[n] += f * pk[kPartHead + 64 * n + lane];
    }
    float *out = a.out + qrow * a.ldo + size_t(head) * HD;
#pragma unroll
    for (int n = 0; n < ND; ++n)
        if (HD >= 64 || lane < HD) out[64 * n + lane] = l == 0.f ? 0.f : o[n] / l;
}

// How a call is cut: sequences of up to kRows rows to a K/V head (group * rows) to k_attn_rows, the
// others to k_attn_chunk, and the tokens of both into `splits` shares: enough workgroups to fill the
// GPU, and none with fewer than 256 tokens.
struct Plan {
    int splits, chunk_tiles;
    bool rows, chunk;
};
Plan plan(const KvPool &p, int hd, int heads, int max_new, int max_ctx, bool uniform) {
    Plan c;
    const int group = heads / p.heads;
    const long long most = (long long)max_new * group, wg = hd <= 128 ? 128 : 64;
    c.chunk = most > kRows;
    c.rows = !c.chunk || !uniform;
    c.chunk_tiles = int((most + wg - 1) / wg);
    const long long jobs = (long long)p.seqs * p.heads * (c.chunk ? c.chunk_tiles : 1);
    // workgroups that the 256 CUs hold at once, and of k_attn_rows twice as many, so that sequences of
    // different lengths even out
    const int fit = c.chunk ? (hd <= 64 ? 2 : 1) : 2 * (hd <= 64 ? 3 : hd <= 128 ? 2 : 1);
    long long s = 256 * fit / jobs;
    s = s < max_ctx / 256 ? s : max_ctx / 256;
    c.splits = s < 1 ? 1 : int(s);
    return c;
}

}  // namespace

size_t attn_paged_scratch(const KvPool &p, int hd, int heads, int rows, int max_new, int max_ctx) {
    if (p.seqs <= 0 || rows <= 0) return 0;
    const int s = plan(p, hd, heads, max_new, max_ctx, false).splits;
    return s == 1 ? 0 : size_t(rows) * size_t(heads) * size_t(s) * size_t(hd + kPartHead) * sizeof(float);
}

namespace {
template <int HD, bool Q8>
hipError_t launch(const KvPool &p, const KvAttn &a, const KvRows &r, int max_ctx, hipStream_t st) {
    const int group = a.heads / p.heads;
    const Plan c = plan(p, HD, a.heads, r.max_new, max_ctx, !r.row_off);
    const long long pairs = (long long)p.seqs * p.heads * c.splits, chunks = pairs * c.chunk_tiles;
    const long long joins = ((long long)p.seqs * r.max_new * a.heads + kWaves - 1) / kWaves;
    if (pairs > 0x7fffffffll || chunks > 0x7fffffffll || joins > 0x7fffffffll) return hipErrorInvalidValue;
    if (c.chunk)
        hipLaunchKernelGGL((k_attn_chunk<HD, Q8>), dim3(unsigned(chunks)), dim3(512), 0, st, p, a, r, group,
                           c.chunk_tiles, c.splits, c.rows ? kRows : 0);
    if (c.rows)
        hipLaunchKernelGGL((k_attn_rows<HD, Q8>), dim3(unsigned(pairs)), dim3(64 * kWaves), 0, st, p, a, r, group,
                           c.splits);
    if (c.splits > 1)
        hipLaunchKernelGGL((k_attn_join<HD>), dim3(unsigned(joins)), dim3(64 * kWaves), 0, st, p, a, r, c.splits);
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

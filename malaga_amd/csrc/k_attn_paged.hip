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
#include "device.hpp"
#include "paged_kv.hpp"

namespace mlg {
namespace {

constexpr int kRows = 16;       // rows of a wave's query tile (columns of the matrix products)
constexpr int kWaves = 4;       // waves of a workgroup
constexpr float kPShift = 15.f;  // p is held times 2^15

// Partial result of a split: [m, l, -, -, out of HD dims] of one row, f32, as a Tile holds them.
constexpr int kPartHead = 4;

__device__ __forceinline__ h8_t as_h8(const uint4 &v) { return __builtin_bit_cast(h8_t, v); }

// 8 int8 as f16, exactly: byte + 128 becomes the low byte of 1024 + u, minus 1152.
__device__ __forceinline__ h8_t i8_to_h8(uint32_t lo, uint32_t hi) {
    const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
    const uint32_t w[4] = {__builtin_amdgcn_perm(0x64646464u, a, 0x07010700u),
                           __builtin_amdgcn_perm(0x64646464u, a, 0x07030702u),
                           __builtin_amdgcn_perm(0x64646464u, b, 0x07010700u),
                           __builtin_amdgcn_perm(0x64646464u, b, 0x07030702u)};
    h8_t r;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        h2_t h = __builtin_bit_cast(h2_t, w[n]) - h2_t{_Float16(1152.f), _Float16(1152.f)};
        r[2 * n] = h[0];
        r[2 * n + 1] = h[1];
    }
    return r;
}

// The four k-groups' lanes of a row: l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float rows_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float rows_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
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
    __device__ __forceinline__ float scale(int c, int n) const {
        const uint32_t w[4] = {d[c].x, d[c].y, d[c].z, d[c].w};
        return h2f(w[n >> 1] >> (16 * (n & 1)));
    }
};

// A wave's query tile: 16 rows, and the softmax and sums of what it has seen.
template <int HD, bool Q8>
struct Tile {
    static constexpr int NC = HD / 32, NU = HD / 16;
    h8_t qh[NC], ql[NC];
    float qf;  // scores in log2 units: qf times the product of the scaled q
    int vis;   // tokens that this lane's row sees
    float m, l;  // the running maximum (log2 units) less kPShift, as rounded; sum of p = 2^(s - m)
    f4_t o[NU];
    int e;  // q8_0: out is held times 2^-e (e: the largest exponent of V's scales so far)

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
        qf = ldexpf(scale * 1.44269504088896340736f, -up);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const float v = ldexpf(x[c][n], up);
                const _Float16 h = _Float16(v);
                qh[c][n] = h;
                ql[c][n] = _Float16(v - float(h));
            }
        m = -INFINITY;
        l = 0.f;
        e = -100;
#pragma unroll
        for (int u = 0; u < NU; ++u) o[u] = f4_t{0.f, 0.f, 0.f, 0.f};
    }

    // The lane's 8 scores (tokens 8 g .. 8 g + 7 of the tile, its row), log2 units.
    __device__ __forceinline__ void scores(const RawTile<HD, Q8> &k, float (&s)[8]) const {
        f4_t acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        if constexpr (Q8) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const h8_t kf[2] = {i8_to_h8(k.a[c].x, k.a[c].y), i8_to_h8(k.a[c].z, k.a[c].w)};
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    f4_t t = {0.f, 0.f, 0.f, 0.f};
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b], ql[c], t, 0, 0, 0);
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b], qh[c], t, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[b][i] = fmaf(t[i], k.scale(c, 4 * b + i), acc[b][i]);
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const h8_t kf = as_h8(k.a[2 * c + b]);
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[c], acc[b], 0, 0, 0);
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[c], acc[b], 0, 0, 0);
                }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = acc[n >> 2][n & 3] * qf;
    }

    // s becomes p (times 2^15); m, l and out follow a larger maximum.
    __device__ __forceinline__ void softmax(float (&s)[8]) {
        float t = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        t = rows_max(t) - kPShift;
        if (__any(t > m)) {  // wave-uniform
            const float mn = fmaxf(m, t), al = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int u = 0; u < NU; ++u) o[u] *= al;
            m = mn;
        }
        const float base = m == -INFINITY ? 0.f : m;  // nothing seen: every score is -inf
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = __builtin_amdgcn_exp2f(s[n] - base);
        l += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    }

    __device__ __forceinline__ static void split(const float (&p)[8], h8_t &hi, h8_t &lo) {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            // p as a finished f32 value: where it is a product, the compiler may otherwise round the
            // product to f16 in one step for hi and in two for lo's difference, and near a tie the
            // two are a unit of f16 apart (seen as 2^-11 of one p missing)
            float x = p[n];
            asm("" : "+v"(x));
            hi[n] = _Float16(x);
            lo[n] = _Float16(x - float(hi[n]));
        }
    }

    // q8_0: out follows a larger scale of V than any before, so that p times a scale stays within
    // f16's range (below 2^15 * 2) and keeps its bits whatever the scales' size.
    __device__ __forceinline__ void fit(const RawTile<HD, Q8> &v) {
        auto largest = [&](bool finite) {  // f16 bit patterns of scales that are not negative are ordered
            uint32_t top = 0u;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const uint32_t w[4] = {v.d[c].x, v.d[c].y, v.d[c].z, v.d[c].w};
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const uint32_t b = w[n >> 1] >> (16 * (n & 1)) & 0x7fffu;
                    top = max(top, finite && b >= 0x7c00u ? 0u : b);
                }
            }
            top = max(top, uint32_t(__shfl_xor(int(top), 16)));
            return max(top, uint32_t(__shfl_xor(int(top), 32)));
        };
        uint32_t top = largest(false);
        if (__any(top >= 0x7c00u)) top = largest(true);  // inf, NaN: the other tokens' rows go on
        const int x = top ? ilogbf(h2f(top)) : e;
        if (__any(x > e)) {
            const int en = max(e, x);
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[u][i] = ldexpf(o[u][i], e - en);
            e = en;
        }
    }

    // out += p V. MASKED: tokens whose p is 0 here may hold anything, inf and NaN among it.
    template <bool MASKED>
    __device__ __forceinline__ void values(const RawTile<HD, Q8> &v, const float (&p)[8]) {
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
                    pd[n] = pe[n] * v.scale(c, n);
                    if (MASKED && p[n] == 0.f) pd[n] = 0.f;
                }
                h8_t ph, pl;
                split(pd, ph, pl);
                const h8_t vf[2] = {i8_to_h8(v.a[c].x, v.a[c].y), i8_to_h8(v.a[c].z, v.a[c].w)};
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    o[2 * c + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], pl, o[2 * c + b], 0, 0, 0);
                    o[2 * c + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], ph, o[2 * c + b], 0, 0, 0);
                }
            }
        } else {
            h8_t ph, pl;
            split(p, ph, pl);
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const h8_t vf = as_h8(v.a[u]);
                o[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o[u], 0, 0, 0);
                o[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, o[u], 0, 0, 0);
            }
        }
    }

    // V's values that are inf or NaN, where some row does not see their token and 0 times them would be
    // NaN: added token by token, each row keeping what it had where it does not see the token.
    __device__ __forceinline__ void not_finite(const RawTile<HD, Q8> &v, const float (&p)[8], int tok0) {
        const int g = int(threadIdx.x & 63) >> 4;
#pragma unroll 1
        for (int t = 0; t < kKvTile; ++t) {  // wave-uniform
            float p1[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) p1[n] = 8 * g + n == t ? p[n] : 0.f;
            h8_t ph, pl;
            split(p1, ph, pl);
            const bool sees = tok0 + t < vis;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                uint32_t w[4] = {v.a[u].x, v.a[u].y, v.a[u].z, v.a[u].w};
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    if (8 * g + n != t || (w[n >> 1] >> (16 * (n & 1)) & 0x7c00u) != 0x7c00u)
                        w[n >> 1] &= n & 1 ? 0xffffu : 0xffff0000u;
                const h8_t vf = as_h8(make_uint4(w[0], w[1], w[2], w[3]));
                f4_t s = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o[u], 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, s, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[u][i] = sees ? s[i] : o[u][i];
            }
        }
    }

    // One tile of tokens tok0 .. tok0 + 31, of which the cache holds those below ctx.
    template <bool MASKED>
    __device__ __forceinline__ void step(const RawTile<HD, Q8> &k, RawTile<HD, Q8> &v, int tok0, int ctx) {
        const int at = tok0 + 8 * (int(threadIdx.x & 63) >> 4);
        float s[8];
        scores(k, s);
        if constexpr (MASKED) {
#pragma unroll
            for (int n = 0; n < 8; ++n) s[n] = at + n < vis ? s[n] : -INFINITY;
        }
        softmax(s);
        const int keep = ctx - at;  // of the lane's 8 tokens; those past the last are whatever the page held before
        if constexpr (MASKED && Q8) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                uint32_t w[4] = {v.d[c].x, v.d[c].y, v.d[c].z, v.d[c].w};
#pragma unroll
                for (int n = 0; n < 4; ++n) w[n] = keep > 2 * n + 1 ? w[n] : keep > 2 * n ? w[n] & 0xffffu : 0u;
                v.d[c] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        if constexpr (MASKED && !Q8) {
            bool odd = false;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                uint32_t w[4] = {v.a[u].x, v.a[u].y, v.a[u].z, v.a[u].w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    w[n] = keep > 2 * n + 1 ? w[n] : keep > 2 * n ? w[n] & 0xffffu : 0u;
                    odd |= (w[n] & 0x7c00u) == 0x7c00u || (w[n] & 0x7c000000u) == 0x7c000000u;
                }
                v.a[u] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (__any(odd)) {  // wave-uniform, and not met by ordinary caches
                not_finite(v, s, tok0);
#pragma unroll
                for (int u = 0; u < NU; ++u) {
                    uint32_t w[4] = {v.a[u].x, v.a[u].y, v.a[u].z, v.a[u].w};
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        if ((w[n] & 0x7c00u) == 0x7c00u) w[n] &= 0xffff0000u;
                        if ((w[n] & 0x7c000000u) == 0x7c000000u) w[n] &= 0xffffu;
                    }
                    v.a[u] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        values<MASKED>(v, s);
    }
};

// ---- few rows to a K/V head: each wave reads its own tiles straight into registers ----
template <int HD, bool Q8>
__global__ __launch_bounds__(256) void k_attn_rows(KvPool pool, KvAttn a, KvRows r, int group, int row_tiles,
                                                   int splits) {
    constexpr int TB = kv_tile_bytes(Q8, HD), NU = HD / 16;
    __shared__ float sm[kWaves][kRows], sl[kWaves][kRows];
    __shared__ f4_t so[kWaves][NU][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t b = blockIdx.x;
    const int split = int(b % uint32_t(splits));
    b /= uint32_t(splits);
    const int rt = int(b % uint32_t(row_tiles));
    b /= uint32_t(row_tiles);
    const int head = int(b % uint32_t(pool.heads)), i = int(b / uint32_t(pool.heads));
    const KvSeq s = kv_seq(pool, r, i);
    if (!s.ok && r.bad && threadIdx.x == 0) *r.bad = 1u;
    const int rows = s.n * group, row0 = rt * kRows;
    if (row0 >= rows) return;
    // this lane's row, and the tokens that it and the tile's first and last row see
    auto sees = [&](int row) { return a.causal ? max(0, s.ctx - s.n + row / group + 1) : s.ctx; };
    const int row = row0 + (lane & 15), last = min(row0 + kRows, rows) - 1;
    const int least = sees(row0), most = sees(last);
    const bool have = row < rows;
    const size_t qrow = size_t(s.r0 + (have ? row : last) / group);
    const int qhead = head * group + (have ? row : last) % group;
    Tile<HD, Q8> t;
    t.load_q(have ? a.q + qrow * a.ldq + size_t(qhead) * HD : nullptr, a.scale, lane);
    t.vis = have ? sees(row) : most;
    const int tiles = (most + kKvTile - 1) / kKvTile, per = (tiles + splits - 1) / splits;
    const int end = min(tiles, (split + 1) * per);
    const uint32_t *table = pool.table + size_t(i) * size_t(pool.table_len);
    for (int kt = split * per + w; kt < end; kt += kWaves) {
        const int tok0 = kt * kKvTile;
        const uint32_t page = table[tok0 >> pool.shift];
        if (page >= uint32_t(pool.pages)) {  // its tokens are not there
            if (r.bad && lane == 0) *r.bad = 1u;
            continue;
        }
        RawTile<HD, Q8> k, v;
        k.load(pool.pool + pool.tile_at(page, head, 0, tok0, TB), lane);
        v.load(pool.pool + pool.tile_at(page, head, 1, tok0, TB), lane);
        if (tok0 + kKvTile <= least) t.template step<false>(k, v, tok0, s.ctx);
        else t.template step<true>(k, v, tok0, s.ctx);
    }
    // the waves' results meet in LDS
    t.l = rows_sum(t.l);
    if (lane < kRows) {
        sm[w][lane] = t.m;
        sl[w][lane] = t.l;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        if constexpr (Q8) {
#pragma unroll
            for (int n = 0; n < 4; ++n) t.o[u][n] = ldexpf(t.o[u][n], t.e);
        }
        so[w][u][lane] = t.o[u];
    }
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
        const int dim = 16 * u + 4 * (lane >> 4);
        if (splits == 1) {
            const f4_t y = l == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : o / l;
            *reinterpret_cast<f4_t *>(a.out + qrow * a.ldo + size_t(qhead) * HD + dim) = y;
        } else {
            float *part = a.scratch + ((qrow * size_t(a.heads) + size_t(qhead)) * size_t(splits) + size_t(split)) *
                                          size_t(HD + kPartHead);
            *reinterpret_cast<f4_t *>(part + kPartHead + dim) = o;
            if (u == 0 && lane < kRows) {
                part[0] = m;
                part[1] = l;
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

// How many splits of the tokens a call makes: enough workgroups to fill the GPU, and none with
// fewer than 256 tokens.
int plan_splits(const KvPool &p, int heads, int max_new, int max_ctx) {
    const int group = heads / p.heads;
    const long long jobs = (long long)p.seqs * p.heads * (((long long)max_new * group + kRows - 1) / kRows);
    long long s = (1024 + jobs - 1) / jobs;
    s = s < max_ctx / 256 ? s : max_ctx / 256;
    return s < 1 ? 1 : int(s);
}

}  // namespace

size_t attn_paged_scratch(const KvPool &p, int hd, int heads, int rows, int max_new, int max_ctx) {
    if (p.seqs <= 0 || rows <= 0) return 0;
    const int s = plan_splits(p, heads, max_new, max_ctx);
    return s == 1 ? 0 : size_t(rows) * size_t(heads) * size_t(s) * size_t(hd + kPartHead) * sizeof(float);
}

namespace {
template <int HD, bool Q8>
hipError_t launch(const KvPool &p, const KvAttn &a, const KvRows &r, int max_ctx, hipStream_t st) {
    const int group = a.heads / p.heads, splits = plan_splits(p, a.heads, r.max_new, max_ctx);
    const long long row_tiles = ((long long)r.max_new * group + kRows - 1) / kRows;
    const long long blocks = (long long)p.seqs * p.heads * row_tiles * splits;
    const long long joins = ((long long)p.seqs * r.max_new * a.heads + kWaves - 1) / kWaves;
    if (blocks > 0x7fffffffll || joins > 0x7fffffffll) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_attn_rows<HD, Q8>), dim3(unsigned(blocks)), dim3(64 * kWaves), 0, st, p, a, r, group,
                       int(row_tiles), splits);
    if (splits > 1)
        hipLaunchKernelGGL((k_attn_join<HD>), dim3(unsigned(joins)), dim3(64 * kWaves), 0, st, p, a, r, splits);
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

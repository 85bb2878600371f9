// Writing and reading the paged K/V cache (paged_kv.hpp has the layout).
//
// Both are copies: bytes alone bound them. A workgroup of 4 waves takes a tile's K and V of one head, a
// wave a block of 32 dims of either: 4 KB of f32 rows in runs of 128 bytes, and of the cache the 2 KB
// (f16) or 1 KB (q8_0) that lie together. K: a lane has 8 dims of two tokens, V: two dims of 8 tokens,
// the operands that the attention reads. The f32 rows pass the caches by (non-temporal): nothing reads
// them again from there soon, and what the cache takes may stay. 32001 tokens, 8 heads of 128, q8_0 (339
// MB each way): written in 74 us = 4.6 TB/s, read back in 74 us; a copy of 2 GB reaches 5.0 TB/s. (V a dim
// to a lane in runs of 64 bytes, and K in every other 16 bytes: 95 us each.)
#include "device.hpp"
#include "paged_kv.hpp"

namespace mlg {
namespace {

struct TileJob {
    KvSeq s;
    int first, base;  // position of the first new token; of the tile's first token
    int head;
    uint32_t page;
    bool have;  // false: no new token in this tile
};

// Block -> (sequence, head, 32-token tile that holds some of its new tokens).
__device__ __forceinline__ TileJob tile_job(const KvPool &p, const KvRows &r, int tiles) {
    TileJob j;
    const uint32_t b = blockIdx.x, t = b % uint32_t(tiles), sh = b / uint32_t(tiles);
    j.head = int(sh % uint32_t(p.heads));
    const int i = int(sh / uint32_t(p.heads));
    j.s = kv_seq(p, r, i);
    j.first = j.s.ctx - j.s.n;
    j.base = (j.first & ~(kKvTile - 1)) + kKvTile * int(t);
    // more rows than tokens: none of them has a place in the cache
    const bool usable = j.s.ok && j.first >= 0;
    if ((!j.s.ok || (!usable && j.s.n > 0)) && r.bad && threadIdx.x == 0) *r.bad = 1u;
    j.have = usable && j.s.n > 0 && j.base < j.s.ctx;
    j.page = j.have ? p.table[size_t(i) * size_t(p.table_len) + size_t(j.base >> p.shift)] : 0u;
    if (j.have && j.page >= uint32_t(p.pages)) {
        if (r.bad && threadIdx.x == 0) *r.bad = 1u;
        j.page = 0xffffffffu;
    }
    return j;
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    return uint32_t(__half_as_ushort(__float2half_rn(a))) | uint32_t(__half_as_ushort(__float2half_rn(b))) << 16;
}

typedef float f2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));

// A q8_0 block's scale and its inverse from max |x| of its 32 values, inf where one of them is not
// finite: d = amax / 127 and 1 / d in f32, as the GGUF codec computes them. A block with a value that
// is not finite is stored as NaN (d), so that it reads back as NaN instead of a wrong number.
struct Q8Scale {
    float inv;
    uint32_t d;  // f16 bits
};
__device__ __forceinline__ Q8Scale q8_scale(float amax) {
    Q8Scale s;
    const bool finite = amax < INFINITY;
    const float d = __fdiv_rn(amax, 127.f);
    s.inv = d > 0.f && finite ? __fdiv_rn(1.f, d) : 0.f;
    if (!(s.inv < INFINITY)) s.inv = 0.f;  // d below 2^-128: it is stored as 0 whatever q says
    s.d = finite ? __half_as_ushort(__float2half_rn(d)) : 0x7e00u;
    return s;
}
// Four values as int8: x / d rounded half away from zero, |x| inv <= 127 + 2^-16. The largest number
// below 0.5 added with x's sign rounds to the next integer exactly where the half does (at y + 0.5 - 2^-25
// a tie goes to the even number, which is the integer), and leaves all that is below the half below it.
// inf times inv = 0 is NaN, which converts to 0.
__device__ __forceinline__ uint32_t q8_four(float a, float b, float c, float d, float ia, float ib, float ic,
                                            float id) {
    auto one = [](float x, float inv) __attribute__((always_inline)) {
        float y = x * inv;
        asm("" : "+v"(y));  // rounded here: the compiler would make one operation of the product and the sum
        return uint32_t(int(y + copysignf(0x1.fffffep-2f, y)));
    };
    const uint32_t lo = __builtin_amdgcn_perm(one(b, ib), one(a, ia), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(one(d, id), one(c, ic), 0x04000c0cu);
    return lo | hi;
}
__device__ __forceinline__ float largest(float m, float x) {  // inf for a value that is not finite
    return fabsf(x) < INFINITY ? fmaxf(m, fabsf(x)) : INFINITY;
}
// v of lane N of the lane's 16.
template <int N>
__device__ __forceinline__ float of_lane16(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x150 + N, 0xf, 0xf, true));
}

// K rows: lane 16 g + r has dims 8 g .. 8 g + 7 of a token's 32, in memory 16-byte chunks 2 g and 2 g + 1.
// A load or store of chunk 2 g alone would take every other 16 bytes; instead the first of the two takes
// chunks 0 .. 3, lane g's at chunk_of(g), the second 4 .. 7, and the halves of the wave trade places.
__device__ __forceinline__ int chunk_of(int g) { return (g & 1) * 2 + (g >> 1); }
__device__ __forceinline__ void trade(f4_t &a, f4_t &b) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a[n]), __float_as_uint(b[n]), false, false);
        a[n] = __uint_as_float(r[0]);
        b[n] = __uint_as_float(r[1]);
    }
}

__device__ __forceinline__ float i8_of(uint32_t w, int n) { return float(int(w << (24 - 8 * n)) >> 24); }

template <int HD, bool Q8>
__global__ __launch_bounds__(256) void k_kv_write(KvPool p, const float *k, size_t ldk, const float *v, size_t ldv,
                                                  KvRows r, int tiles) {
    const TileJob j = tile_job(p, r, tiles);
    if (!j.have || j.page == 0xffffffffu) return;
    constexpr int TB = kv_tile_bytes(Q8, HD), NC = HD / 32;
    const int lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    for (int w = int(threadIdx.x >> 6); w < 2 * NC; w += 4) {  // wave-uniform
        const int which = w >= NC, c = which ? w - NC : w;
        uint8_t *tile = p.pool + p.tile_at(j.page, j.head, which, j.base, TB);
        if (!which) {
            // row of the token at position pos: j.s.r0 + pos - j.first
            f4_t x[2][2];
            bool in[2];
            const int t0 = 8 * (lr >> 2) + (lr & 3);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int pos = j.base + t0 + 4 * b;
                in[b] = pos >= j.first && pos < j.s.ctx;
                const f4_t *src = reinterpret_cast<const f4_t *>(k + size_t(j.s.r0 + (in[b] ? pos - j.first : 0)) * ldk +
                                                                 size_t(j.head) * HD + 32 * c) + chunk_of(g);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    x[b][h] = in[b] ? __builtin_nontemporal_load(src + 4 * h) : f4_t{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) trade(x[b][0], x[b][1]);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if constexpr (!Q8) {
                    if (in[b])
                        *reinterpret_cast<u4_t *>(tile + ((2 * c + b) * 64 + lane) * 16) =
                            u4_t{pack_h2(x[b][0][0], x[b][0][1]), pack_h2(x[b][0][2], x[b][0][3]),
                                 pack_h2(x[b][1][0], x[b][1][1]), pack_h2(x[b][1][2], x[b][1][3])};
                } else {
                    float amax = 0.f;
#pragma unroll
                    for (int n = 0; n < 8; ++n) amax = largest(amax, x[b][n >> 2][n & 3]);
                    // the block's four k-groups: lanes lr, 16 + lr, 32 + lr, 48 + lr
                    amax = fmaxf(amax, __shfl_xor(amax, 16));
                    amax = fmaxf(amax, __shfl_xor(amax, 32));
                    const Q8Scale sc = q8_scale(amax);
                    u2_t q;
#pragma unroll
                    for (int h = 0; h < 2; ++h) q[h] = q8_four(x[b][h][0], x[b][h][1], x[b][h][2], x[b][h][3], sc.inv, sc.inv, sc.inv, sc.inv);
                    if (in[b]) {
                        *reinterpret_cast<u2_t *>(tile + (c * 64 + lane) * 16 + 8 * b) = q;
                        if (g == 0) *reinterpret_cast<uint16_t *>(tile + kv_scale_byte(HD, t0 + 4 * b, c)) = uint16_t(sc.d);
                    }
                }
            }
        } else {
            // dims 32 c + 2 lr + 0, 1 of tokens 8 g .. 8 g + 7: which are new, lo <= n < hi
            const int lo = max(0, j.first - j.base - 8 * g), hi = min(8, j.s.ctx - j.base - 8 * g);
            f2_t x[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const bool in = n >= lo && n < hi;
                const f2_t *src = reinterpret_cast<const f2_t *>(
                    v + size_t(in ? j.s.r0 + j.base + 8 * g + n - j.first : j.s.r0) * ldv + size_t(j.head) * HD +
                    32 * c + 2 * lr);
                x[n] = in ? __builtin_nontemporal_load(src) : f2_t{0.f, 0.f};
            }
            const bool all = lo == 0 && hi == 8;
            if constexpr (!Q8) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    u4_t h;
#pragma unroll
                    for (int n = 0; n < 4; ++n) h[n] = pack_h2(x[2 * n][e], x[2 * n + 1][e]);
                    uint8_t *at = tile + ((2 * c + (lr >> 3)) * 64 + g * 16 + (2 * lr & 15) + e) * 16;
                    if (all) {
                        *reinterpret_cast<u4_t *>(at) = h;
                    } else {
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                            if (n >= lo && n < hi)
                                reinterpret_cast<uint16_t *>(at)[n] = uint16_t(h[n >> 1] >> (16 * (n & 1)));
                    }
                }
            } else {
                // lane n of the 16 (and n + 8) computes the scale of token n, the others take it from there
                float own = 0.f;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    // the block's 32 dims: 16 lanes
                    const float amax = group_reduce(largest(largest(0.f, x[n][0]), x[n][1]), 4, OpMax{});
                    own = (lr & 7) == n ? amax : own;
                }
                const Q8Scale sc = q8_scale(own);
                float inv[8];
                static_for<0, 8>([&](auto n) __attribute__((always_inline)) {
                    inv[decltype(n)::value] = of_lane16<decltype(n)::value>(sc.inv);
                });
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    u2_t q;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const f4_t y = {x[4 * h][e], x[4 * h + 1][e], x[4 * h + 2][e], x[4 * h + 3][e]};
                        q[h] = q8_four(y[0], y[1], y[2], y[3], inv[4 * h], inv[4 * h + 1], inv[4 * h + 2], inv[4 * h + 3]);
                    }
                    uint8_t *at = tile + (c * 64 + g * 16 + (2 * lr & 15) + e) * 16 + 8 * (lr >> 3);
                    if (all) {
                        *reinterpret_cast<u2_t *>(at) = q;
                    } else {
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                            if (n >= lo && n < hi) at[n] = uint8_t(q[n >> 2] >> (8 * (n & 3)));
                    }
                }
                if (lr >= lo && lr < hi)
                    *reinterpret_cast<uint16_t *>(tile + kv_scale_byte(HD, 8 * g + lr, c)) = uint16_t(sc.d);
            }
        }
    }
}

template <int HD, bool Q8>
__global__ __launch_bounds__(256) void k_kv_read(KvPool p, float *k, size_t ldk, float *v, size_t ldv, KvRows r,
                                                 int tiles) {
    const TileJob j = tile_job(p, r, tiles);
    constexpr int TB = kv_tile_bytes(Q8, HD), NC = HD / 32;
    const int lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    if (!j.have || j.page == 0xffffffffu) {  // no place to read: rows of zeros
        const bool lost = j.have || !j.s.ok || j.first < 0;
        if (!lost || j.s.n == 0) return;
        // of an unusable sequence, tile t clears rows 32 t ..; of a bad page, the tile's rows
        const int t = int(blockIdx.x % uint32_t(tiles));
        const int a = j.have ? max(j.base, j.first) - j.first : kKvTile * t;
        const int b = j.have ? min(j.base + kKvTile, j.s.ctx) - j.first : min(a + kKvTile, j.s.n);
        for (int e = int(threadIdx.x); e < (b - a) * HD; e += 256) {
            const size_t row = size_t(j.s.r0 + a + e / HD), c = size_t(j.head) * HD + size_t(e % HD);
            k[row * ldk + c] = 0.f;
            v[row * ldv + c] = 0.f;
        }
        return;
    }
    for (int w = int(threadIdx.x >> 6); w < 2 * NC; w += 4) {
        const int which = w >= NC, c = which ? w - NC : w;
        const uint8_t *tile = p.pool + p.tile_at(j.page, j.head, which, j.base, TB);
        if (!which) {
            const int t0 = 8 * (lr >> 2) + (lr & 3);
            u4_t raw[2];
            if constexpr (Q8) {
                raw[0] = *reinterpret_cast<const u4_t *>(tile + (c * 64 + lane) * 16);
            } else {
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    raw[b] = *reinterpret_cast<const u4_t *>(tile + ((2 * c + b) * 64 + lane) * 16);
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int pos = j.base + t0 + 4 * b;
                f4_t x[2];
                if constexpr (Q8) {
                    const float d = h2f(*reinterpret_cast<const uint16_t *>(tile + kv_scale_byte(HD, t0 + 4 * b, c)));
#pragma unroll
                    for (int n = 0; n < 8; ++n) x[n >> 2][n & 3] = i8_of(raw[0][2 * b + (n >> 2)], n & 3) * d;
                } else {
#pragma unroll
                    for (int n = 0; n < 8; ++n) x[n >> 2][n & 3] = h2f(raw[b][n >> 1] >> (16 * (n & 1)));
                }
                trade(x[0], x[1]);
                if (pos < j.first || pos >= j.s.ctx) continue;
                f4_t *dst = reinterpret_cast<f4_t *>(k + size_t(j.s.r0 + pos - j.first) * ldk + size_t(j.head) * HD +
                                                     32 * c) + chunk_of(g);
                __builtin_nontemporal_store(x[0], dst);
                __builtin_nontemporal_store(x[1], dst + 4);
            }
        } else {
            u4_t raw[2], dd = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if constexpr (Q8) {
                    const u2_t q = *reinterpret_cast<const u2_t *>(tile + (c * 64 + g * 16 + (2 * lr & 15) + e) * 16 +
                                                                   8 * (lr >> 3));
                    raw[e] = u4_t{q[0], q[1], 0u, 0u};
                } else {
                    raw[e] = *reinterpret_cast<const u4_t *>(
                        tile + ((2 * c + (lr >> 3)) * 64 + g * 16 + (2 * lr & 15) + e) * 16);
                }
            }
            if constexpr (Q8) dd = *reinterpret_cast<const u4_t *>(tile + kv_scale_byte(HD, 8 * g, c));
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int pos = j.base + 8 * g + n;
                f2_t x;
                if constexpr (Q8) {
                    const float d = h2f(dd[n >> 1] >> (16 * (n & 1)));
                    x = f2_t{i8_of(raw[0][n >> 2], n & 3) * d, i8_of(raw[1][n >> 2], n & 3) * d};
                } else {
                    x = f2_t{h2f(raw[0][n >> 1] >> (16 * (n & 1))), h2f(raw[1][n >> 1] >> (16 * (n & 1)))};
                }
                if (pos < j.first || pos >= j.s.ctx) continue;
                __builtin_nontemporal_store(x, reinterpret_cast<f2_t *>(v + size_t(j.s.r0 + pos - j.first) * ldv +
                                                                        size_t(j.head) * HD + 32 * c + 2 * lr));
            }
        }
    }
}

// Blocks of a write or read: every tile that max_new tokens in a row may touch.
bool tile_grid(const KvPool &p, const KvRows &r, int *tiles, unsigned *blocks) {
    const long long t = ((long long)r.max_new + kKvTile - 2) / kKvTile + 1;
    *tiles = int(t);
    const unsigned long long n = (unsigned long long)p.seqs * (unsigned long long)p.heads * (unsigned long long)*tiles;
    *blocks = unsigned(n);
    return n <= 0x7fffffffull;
}

}  // namespace

#define MLG_KV_DISPATCH(KERNEL, ...)                                                                                \
    switch (hd * 2 + int(q8)) {                                                                                     \
    case 64: hipLaunchKernelGGL((KERNEL<32, false>), dim3(blocks), dim3(256), 0, st, __VA_ARGS__); break;           \
    case 65: hipLaunchKernelGGL((KERNEL<32, true>), dim3(blocks), dim3(256), 0, st, __VA_ARGS__); break;            \
    case 128: hipLaunchKernelGGL((KERNEL<64, false>), dim3(blocks), dim3(256), 0, st, __VA_ARGS__); break;          \
    case 129: hipLaunchKernelGGL((KERNEL<64, true>), dim3(blocks), dim3(256), 0, st, __VA_ARGS__); break;           \
    case 256: hipLaunchKernelGGL((KERNEL<128, false>), dim3(blocks), dim3(256), 0, st, __VA_ARGS__); break;         \
    case 257: hipLaunchKernelGGL((KERNEL<128, true>), dim3(blocks), dim3(256), 0, st, __VA_ARGS__); break;          \
    case 512: hipLaunchKernelGGL((KERNEL<256, false>), dim3(blocks), dim3(256), 0, st, __VA_ARGS__); break;         \
    case 513: hipLaunchKernelGGL((KERNEL<256, true>), dim3(blocks), dim3(256), 0, st, __VA_ARGS__); break;          \
    default: return hipErrorInvalidValue;                                                                           \
    }

hipError_t kv_write(const KvPool &p, bool q8, int hd, const float *k, size_t ldk, const float *v, size_t ldv,
                    const KvRows &r, hipStream_t st) {
    int tiles;
    unsigned blocks;
    if (p.seqs <= 0 || r.rows <= 0) return hipSuccess;
    if (!tile_grid(p, r, &tiles, &blocks)) return hipErrorInvalidValue;
    MLG_KV_DISPATCH(k_kv_write, p, k, ldk, v, ldv, r, tiles)
    return hipGetLastError();
}

hipError_t kv_read(const KvPool &p, bool q8, int hd, float *k, size_t ldk, float *v, size_t ldv, const KvRows &r,
                   hipStream_t st) {
    int tiles;
    unsigned blocks;
    if (p.seqs <= 0 || r.rows <= 0) return hipSuccess;
    if (!tile_grid(p, r, &tiles, &blocks)) return hipErrorInvalidValue;
    MLG_KV_DISPATCH(k_kv_read, p, k, ldk, v, ldv, r, tiles)
    return hipGetLastError();
}

}  // namespace mlg

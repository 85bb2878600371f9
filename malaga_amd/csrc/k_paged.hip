// Writing and reading the paged K/V cache (paged_kv.hpp has the layout).
//
// Both kernels give a wave one 1 KB piece of a tile (q8_0: with its two halves), lane l to the
// piece's bytes 16 l .. 16 l + 15, so the cache's side of the copy is whole lines: 4 KB per tile
// at hd 64 f16. The f32 side is then 128-byte runs of 16 rows for K (a lane's 8 dims of one token)
// and 64-byte runs for V (a lane's one dim of 8 tokens). A workgroup of 4 waves takes a tile's K and
// V of one head.
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

// A q8_0 block's scale and its inverse from max |x| of its 32 values, and whether every one of them
// is finite: d = amax / 127 and 1 / d in f32, as the GGUF codec computes them. A block with a value
// that is not finite is stored as NaN (d), so that it reads back as NaN instead of a wrong number.
struct Q8Scale {
    float inv;
    uint16_t d;
};
__device__ __forceinline__ Q8Scale q8_scale(float amax, bool finite) {
    Q8Scale s;
    const float d = __fdiv_rn(amax, 127.f);
    s.inv = d > 0.f && finite ? __fdiv_rn(1.f, d) : 0.f;
    if (!(s.inv < INFINITY)) s.inv = 0.f;  // d below 2^-128: it is stored as 0 whatever q says
    s.d = finite ? __half_as_ushort(__float2half_rn(d)) : uint16_t(0x7e00u);
    return s;
}
__device__ __forceinline__ uint32_t q8_value(float x, const Q8Scale &s) {
    // round half away from zero; a value that is not finite has inv = 0 and its product dropped
    const float y = s.inv > 0.f ? roundf(__fmul_rn(x, s.inv)) : 0.f;
    return uint32_t(int(fminf(fmaxf(y, -127.f), 127.f))) & 0xffu;
}

template <int HD, bool Q8>
__global__ __launch_bounds__(256) void k_kv_write(KvPool p, const float *k, size_t ldk, const float *v, size_t ldv,
                                                  KvRows r, int tiles) {
    const TileJob j = tile_job(p, r, tiles);
    if (!j.have || j.page == 0xffffffffu) return;
    constexpr int TB = kv_tile_bytes(Q8, HD), NC = HD / 32, NP = Q8 ? NC : 2 * NC;
    const int lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    for (int w = int(threadIdx.x >> 6); w < 2 * NP; w += 4) {  // wave-uniform
        const int which = w >= NP, pc = which ? w - NP : w;
        uint8_t *tile = p.pool + p.tile_at(j.page, j.head, which, j.base, TB);
        // row of the token at position pos: j.s.r0 + pos - j.first
        if (!which) {
            constexpr int NB = Q8 ? 2 : 1;  // tokens of this lane
            const int c = Q8 ? pc : pc >> 1;
            float x[NB][8];
            bool in[NB];
#pragma unroll
            for (int e = 0; e < NB; ++e) {
                const int t = 8 * (lr >> 2) + 4 * (Q8 ? e : pc & 1) + (lr & 3), pos = j.base + t;
                in[e] = pos >= j.first && pos < j.s.ctx;
                if (in[e]) {
                    const float *src = k + size_t(j.s.r0 + pos - j.first) * ldk + size_t(j.head) * HD + 32 * c + 8 * g;
                    const float4 a = ld4(src, 0), b = ld4(src, 1);
                    x[e][0] = a.x, x[e][1] = a.y, x[e][2] = a.z, x[e][3] = a.w;
                    x[e][4] = b.x, x[e][5] = b.y, x[e][6] = b.z, x[e][7] = b.w;
                } else {
#pragma unroll
                    for (int n = 0; n < 8; ++n) x[e][n] = 0.f;
                }
            }
            if constexpr (!Q8) {
                if (in[0])
                    *reinterpret_cast<uint4 *>(tile + (pc * 64 + lane) * 16) =
                        make_uint4(pack_h2(x[0][0], x[0][1]), pack_h2(x[0][2], x[0][3]), pack_h2(x[0][4], x[0][5]),
                                   pack_h2(x[0][6], x[0][7]));
            } else {
#pragma unroll
                for (int e = 0; e < NB; ++e) {
                    float amax = 0.f;
                    bool bad = false;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        amax = fmaxf(amax, fabsf(x[e][n]));
                        bad |= !(fabsf(x[e][n]) < INFINITY);
                    }
                    // the block's four k-groups: lanes lr, 16 + lr, 32 + lr, 48 + lr
                    if (bad) amax = INFINITY;
                    amax = fmaxf(amax, __shfl_xor(amax, 16));
                    amax = fmaxf(amax, __shfl_xor(amax, 32));
                    const Q8Scale sc = q8_scale(amax, amax < INFINITY);
                    uint32_t q[2] = {0u, 0u};
#pragma unroll
                    for (int n = 0; n < 8; ++n) q[n >> 2] |= q8_value(x[e][n], sc) << (8 * (n & 3));
                    if (in[e]) {
                        *reinterpret_cast<uint2 *>(tile + (pc * 64 + lane) * 16 + 8 * e) = make_uint2(q[0], q[1]);
                        const int t = 8 * (lr >> 2) + 4 * e + (lr & 3);
                        if (g == 0) *reinterpret_cast<uint16_t *>(tile + kv_scale_byte(HD, t, c)) = sc.d;
                    }
                }
            }
        } else {
            constexpr int NU = Q8 ? 2 : 1;  // dims of this lane
            // its 8 tokens 8 g .. 8 g + 7: which are new, lo <= n < hi
            const int lo = max(0, j.first - j.base - 8 * g), hi = min(8, j.s.ctx - j.base - 8 * g);
            float x[NU][8];
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const bool in = n >= lo && n < hi;
                const float *src = v + size_t(in ? j.s.r0 + j.base + 8 * g + n - j.first : j.s.r0) * ldv +
                                   size_t(j.head) * HD + 16 * NU * pc + lr;
#pragma unroll
                for (int u = 0; u < NU; ++u) x[u][n] = in ? src[16 * u] : 0.f;
            }
            if constexpr (!Q8) {
                uint32_t h[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) h[n] = pack_h2(x[0][2 * n], x[0][2 * n + 1]);
                uint8_t *at = tile + (pc * 64 + lane) * 16;
                if (lo == 0 && hi == 8) {
                    *reinterpret_cast<uint4 *>(at) = make_uint4(h[0], h[1], h[2], h[3]);
                } else {
#pragma unroll
                    for (int n = 0; n < 8; ++n)
                        if (n >= lo && n < hi)
                            reinterpret_cast<uint16_t *>(at)[n] = uint16_t(h[n >> 1] >> (16 * (n & 1)));
                }
            } else {
                uint32_t q[2][2] = {{0u, 0u}, {0u, 0u}};
                uint16_t d[8];
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    float amax = fmaxf(fabsf(x[0][n]), fabsf(x[1][n]));
                    if (!(fabsf(x[0][n]) < INFINITY) || !(fabsf(x[1][n]) < INFINITY)) amax = INFINITY;
                    amax = group_reduce(amax, 4, OpMax{});  // the block's 32 dims: 16 lanes
                    const Q8Scale sc = q8_scale(amax, amax < INFINITY);
                    d[n] = sc.d;
#pragma unroll
                    for (int u = 0; u < 2; ++u) q[u][n >> 2] |= q8_value(x[u][n], sc) << (8 * (n & 3));
                }
                uint8_t *at = tile + (pc * 64 + lane) * 16, *sd = tile + kv_scale_byte(HD, 8 * g, pc);
                if (lo == 0 && hi == 8) {
                    *reinterpret_cast<uint4 *>(at) = make_uint4(q[0][0], q[0][1], q[1][0], q[1][1]);
                    if (lr == 0)
                        *reinterpret_cast<uint4 *>(sd) =
                            make_uint4(d[0] | uint32_t(d[1]) << 16, d[2] | uint32_t(d[3]) << 16,
                                       d[4] | uint32_t(d[5]) << 16, d[6] | uint32_t(d[7]) << 16);
                } else {
#pragma unroll
                    for (int n = 0; n < 8; ++n)
                        if (n >= lo && n < hi) {
                            at[n] = uint8_t(q[0][n >> 2] >> (8 * (n & 3)));
                            at[8 + n] = uint8_t(q[1][n >> 2] >> (8 * (n & 3)));
                            if (lr == 0) reinterpret_cast<uint16_t *>(sd)[n] = d[n];
                        }
                }
            }
        }
    }
}

template <int HD, bool Q8>
__global__ __launch_bounds__(256) void k_kv_read(KvPool p, float *k, size_t ldk, float *v, size_t ldv, KvRows r,
                                                 int tiles) {
    const TileJob j = tile_job(p, r, tiles);
    constexpr int TB = kv_tile_bytes(Q8, HD), NC = HD / 32, NP = Q8 ? NC : 2 * NC;
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
    for (int w = int(threadIdx.x >> 6); w < 2 * NP; w += 4) {
        const int which = w >= NP, pc = which ? w - NP : w;
        const uint8_t *tile = p.pool + p.tile_at(j.page, j.head, which, j.base, TB);
        const uint4 raw = *reinterpret_cast<const uint4 *>(tile + (pc * 64 + lane) * 16);
        const uint32_t a[4] = {raw.x, raw.y, raw.z, raw.w};
        if (!which) {
            constexpr int NB = Q8 ? 2 : 1;
            const int c = Q8 ? pc : pc >> 1;
#pragma unroll
            for (int e = 0; e < NB; ++e) {
                const int t = 8 * (lr >> 2) + 4 * (Q8 ? e : pc & 1) + (lr & 3), pos = j.base + t;
                if (pos < j.first || pos >= j.s.ctx) continue;
                float x[8];
                if constexpr (Q8) {
                    const float d = h2f(*reinterpret_cast<const uint16_t *>(tile + kv_scale_byte(HD, t, c)));
#pragma unroll
                    for (int n = 0; n < 8; ++n) x[n] = float(int(a[2 * e + (n >> 2)] << (24 - 8 * (n & 3))) >> 24) * d;
                } else {
#pragma unroll
                    for (int n = 0; n < 8; ++n) x[n] = h2f(a[n >> 1] >> (16 * (n & 1)));
                }
                float4 *dst = reinterpret_cast<float4 *>(k + size_t(j.s.r0 + pos - j.first) * ldk +
                                                         size_t(j.head) * HD + 32 * c + 8 * g);
                dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            }
        } else {
            constexpr int NU = Q8 ? 2 : 1;
            uint4 draw = make_uint4(0, 0, 0, 0);
            if constexpr (Q8) draw = *reinterpret_cast<const uint4 *>(tile + kv_scale_byte(HD, 8 * g, pc));
            const uint32_t dd[4] = {draw.x, draw.y, draw.z, draw.w};
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int pos = j.base + 8 * g + n;
                if (pos < j.first || pos >= j.s.ctx) continue;
                float *dst = v + size_t(j.s.r0 + pos - j.first) * ldv + size_t(j.head) * HD + 16 * NU * pc + lr;
                if constexpr (Q8) {
                    const float d = h2f(dd[n >> 1] >> (16 * (n & 1)));
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        dst[16 * u] = float(int(a[2 * u + (n >> 2)] << (24 - 8 * (n & 3))) >> 24) * d;
                } else {
                    dst[0] = h2f(a[n >> 1] >> (16 * (n & 1)));
                }
            }
        }
    }
}

// Blocks of a write or read: every tile that max_new tokens in a row may touch.
bool tile_grid(const KvPool &p, const KvRows &r, int *tiles, unsigned *blocks) {
    *tiles = (r.max_new + kKvTile - 2) / kKvTile + 1;
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

// The paged K/V cache: where a token's values lie in the pool, and the launchers of the kernels
// that write, read and attend it (k_paged.hip, k_attn_paged.hip).
//
// A page holds `page` tokens of every K/V head, K and V apart, in tiles of 32 tokens:
//   [page][head][K, V][page / 32 tiles].
// A tile is laid out as the operands of v_mfma_f32_16x16x32_f16 are read, lane l = 16 g + r of a
// wave taking 16 bytes at 16 l of each 1 KB piece, so that every load is one run of whole lines
// and no value crosses lanes between the score product and the value product:
//   K (scores^T = K q^T: the A operand's row r of product b is token 8 (r / 4) + 4 b + r % 4, its
//     k-group g the dims 8 g .. 8 g + 7 of a block of 32): the result then leaves lane 16 g + r
//     with the scores of tokens 8 g .. 8 g + 7 for query r, which is
//   V (out^T = V^T p^T: row r is dim 16 u + r, k-group g tokens 8 g .. 8 g + 7): what its B operand
//     takes from that lane.
// f16: piece 2 c + b of K (c: the block of 32 dims), piece u of V. q8_0: int8, piece c of K holds
// b = 0, 1 (8 bytes each), piece c of V u = 2 c, 2 c + 1; then one f16 scale per token and block of
// 32 dims, [block][32 tokens] (a q8_0 block is 32 dims of one token, as in the GGUF codec).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mlg {

constexpr int kKvTile = 32;  // tokens of a tile

__host__ __device__ constexpr int kv_tile_bytes(bool q8, int hd) { return (q8 ? 34 : 64) * hd; }

// Index of (token t of the tile, dim) in a K or V tile, in elements (f16 or int8).
__host__ __device__ constexpr int kv_k_elem(bool q8, int t, int dim) {
    const int lane = (dim >> 3 & 3) * 16 + (t >> 3) * 4 + (t & 3), b = t >> 2 & 1, c = dim >> 5;
    return (q8 ? (c * 64 + lane) * 2 + b : (c * 2 + b) * 64 + lane) * 8 + (dim & 7);
}
__host__ __device__ constexpr int kv_v_elem(bool q8, int t, int dim) {
    const int lane = (t >> 3) * 16 + (dim & 15), u = dim >> 4;
    return (q8 ? ((u >> 1) * 64 + lane) * 2 + (u & 1) : u * 64 + lane) * 8 + (t & 7);
}
// Byte of the f16 scale of (token t, dims 32 c ..) in a q8_0 tile.
__host__ __device__ constexpr int kv_scale_byte(int hd, int t, int c) { return 32 * hd + (c * kKvTile + t) * 2; }

struct KvPool {
    uint8_t *pool;
    const uint32_t *table;  // [seqs][table_len] page ids
    int seqs, table_len, heads, pages;
    int shift;  // page = 1 << shift tokens, 32 .. 256
    // Byte of the tile that holds position pos's token in page `id`, K (which = 0) or V (1).
    __host__ __device__ size_t tile_at(uint32_t id, int head, int which, int pos, int tile_bytes) const {
        const int per = shift - 5, in = (pos & ((1 << shift) - 1)) >> 5;
        return (((((size_t(id) * size_t(heads) + size_t(head)) * 2 + size_t(which)) << per) + size_t(in))) *
               size_t(tile_bytes);
    }
};

// Which rows and positions a call is about. Sequence i's rows are row_off[i] .. row_off[i + 1] - 1
// (row_off null: max_new rows each), and the cache holds ctx[i] of its tokens.
struct KvRows {
    const uint32_t *row_off, *ctx;
    int rows, max_new;
    uint32_t *bad;  // set to 1 where a sequence or page is not usable (may be null)
};

struct KvSeq {
    int r0, n;  // its rows; n = 0: none, or not usable
    int ctx;    // its tokens
    bool ok;    // false: more tokens than its table row holds, more than max_new rows, or falling offsets
};

// The rows and tokens of sequence i, with every bound checked.
__host__ __device__ inline KvSeq kv_seq(const KvPool &p, const KvRows &r, int i) {
    KvSeq s;
    long long a, b;
    if (r.row_off) {
        a = r.row_off[i];
        b = r.row_off[i + 1];
    } else {
        a = (long long)i * r.max_new;
        b = a + r.max_new;
    }
    const long long ctx = r.ctx[i];
    s.ok = a <= b && b <= r.rows && b - a <= r.max_new && ctx <= ((long long)p.table_len << p.shift);
    // a sequence that is not usable keeps the rows that a call may still clear
    a = a < r.rows ? a : r.rows;
    b = b < r.rows ? b : r.rows;
    const long long n = b > a ? b - a : 0;
    s.r0 = int(a);
    s.n = int(n < r.max_new ? n : r.max_new);
    s.ctx = s.ok ? int(ctx) : 0;
    return s;
}

// f32 rows k, v (row r at k + r ldk, head h at h hd) into the cache, and back out of it. A
// sequence's rows are its last n tokens. hd: 32, 64, 128 or 256.
hipError_t kv_write(const KvPool &p, bool q8, int hd, const float *k, size_t ldk, const float *v, size_t ldv,
                    const KvRows &r, hipStream_t st);
hipError_t kv_read(const KvPool &p, bool q8, int hd, float *k, size_t ldk, float *v, size_t ldv, const KvRows &r,
                   hipStream_t st);

// Attention of the rows over their sequence's tokens; heads = p.heads * group query heads.
struct KvAttn {
    const float *q;
    float *out;
    size_t ldq, ldo;
    int heads, causal;
    float scale;
    float *scratch;
};
size_t attn_paged_scratch(const KvPool &p, bool q8, int hd, int heads, int rows, int max_new, int max_ctx);
hipError_t attn_paged(const KvPool &p, bool q8, int hd, const KvAttn &a, const KvRows &r, int max_ctx, hipStream_t st);

}  // namespace mlg

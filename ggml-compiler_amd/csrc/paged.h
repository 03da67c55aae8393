// paged.h - the paged 4-bit cache's device layout and the batch's lookups (include/gcq_paged.h).
//
// Bytes: [page][KV head][tile of 32 tokens][36 D]. A tile is what a wavefront of the attention kernels takes at a
// time, one contiguous piece, laid out so that a lane's 16-byte loads are its MFMA operands. Byte i of a token's D / 2
// code bytes holds dim i (low nibble) and dim i + D / 2 (high):
//   K codes  16 D  [token][g 4][b D/64][j 8], i = 32 b + 8 g + j: lane group g's 8 dims of every block side by side
//   V codes  16 D  [t D/64][g 4][c 16][u 2][m 8], token 8 g + m, i = 16 (2 t + u) + c: 8 tokens of one dim pair per
//            8 bytes, as P V's operand needs them
//   K scales, V scales  2 D each, f16 [block D/32][32], token t at 8 (t / 8) + order(t % 8)
// order() swaps 1, 2 and 5, 6: masking a word's nibbles with 0x000f000f leaves bytes (0, 2) and (1, 3) as f16 pairs.
#pragma once

#include "gcq_common.h"

namespace gcq {

constexpr int kPagedTile = 32;
constexpr float kPagedMax = 65504.0f;  // the largest f16: every value d (c - 8) is within it

struct Paged {
    uint8_t * data;
    const int32_t * pages, * starts, * past;
    int64_t ld;
    int n_pages, shift, Hkv, n_seq, max_pages, n_rows;  // page_size == 1 << shift
};

__device__ __forceinline__ int paged_order(int m) { return (m & 4) | (m & 1) << 1 | (m >> 1 & 1); }

// The sequence that owns row r, -1 if none does (all lanes together; r uniform).
__device__ __forceinline__ int paged_seq(const Paged & a, int r) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 64)
        n += __popcll(__ballot(s0 + lane < a.n_seq && a.starts[min(s0 + lane, a.n_seq - 1) + 1] <= r));
    return n < a.n_seq && a.starts[n] <= r && r < a.starts[n + 1] ? n : -1;
}

// Byte offset of the tile that holds position pos of sequence s for KV head h, -1 if the token is not there.
__device__ __forceinline__ int64_t paged_tile(const Paged & a, int s, int64_t pos, int h, int D) {
    if (pos < 0 || pos >> a.shift >= a.max_pages) return -1;
    const int e = a.pages[s * a.ld + (pos >> a.shift)];
    if ((unsigned) e >= (unsigned) a.n_pages) return -1;
    return ((((int64_t) e * a.Hkv + h) << (a.shift - 5)) + ((pos & ((1 << a.shift) - 1)) >> 5)) * (36 * D);
}

// Inclusive prefix sum over the wavefront.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15 into the next row, then 31 into the upper half
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// Eight `id` (8 positions, a quarter of a tile) of those that the batch's new rows touch, a sequence's after the one's before:
// the sequence, its rows and the eight's number in it (uniform; all lanes together).
struct PagedSpan {
    int s, r0, rows;
    int64_t past, eight;
};
__device__ __forceinline__ bool paged_find(const Paged & a, int id, PagedSpan & w) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
        int r0 = 0, rows = 0, past = 0, n = 0;
        if (s0 + lane < a.n_seq) {
            r0 = a.starts[s0 + lane];
            rows = r0 < 0 ? 0 : max(min(a.starts[s0 + lane + 1], a.n_rows) - r0, 0);
            past = a.past[s0 + lane];
            n = rows ? (int) ((((int64_t) past + rows - 1) >> 3) - (past >> 3)) + 1 : 0;
        }
        const int sum = wave_scan(n);
        const uint64_t at = __ballot(base + sum > id);
        if (at) {
            const int l = __builtin_ctzll(at);
            w.s = s0 + l;
            w.r0 = __builtin_amdgcn_readlane(r0, l);
            w.rows = __builtin_amdgcn_readlane(rows, l);
            w.past = __builtin_amdgcn_readlane(past, l);
            w.eight = (w.past >> 3) + id - base - __builtin_amdgcn_readlane(sum - n, l);
            return true;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// Within a tile: code byte i of token slot t, and the f16 scale of block b (byte offsets).
template <int D> __device__ __forceinline__ int paged_k_byte(int t, int i) {
    return t * (D / 2) + (i >> 3 & 3) * (D / 8) + (i >> 5) * 8 + (i & 7);
}
template <int D> __device__ __forceinline__ int paged_v_byte(int t, int i) {
    return 16 * D + ((i >> 5) * 4 + (t >> 3)) * 256 + (i & 15) * 16 + (i >> 4 & 1) * 8 + (t & 7);
}
template <int D> __device__ __forceinline__ int paged_k_scale(int t, int b) {
    return 32 * D + 2 * (b * 32 + (t & 24) + paged_order(t & 7));
}
template <int D> __device__ __forceinline__ int paged_v_scale(int t, int b) { return paged_k_scale<D>(t, b) + 2 * D; }

// A launch's grid: it may hold fewer than 2^32 threads.
inline unsigned paged_grid(int64_t blocks, int threads) {
    if (blocks * threads > (int64_t) UINT32_MAX) fail("paged: too many rows and heads");
    return (unsigned) blocks;
}

size_t paged_attn_workspace(const Paged & p, int D, int H, int64_t max_rows);
void launch_paged_attn(const Paged & p, int D, const void * q, int64_t q_r, int64_t q_h, int H, int64_t max_rows, int window,
                       float scale, float * out, void * ws, hipStream_t s);

}  // namespace gcq

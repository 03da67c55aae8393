// paged.hip - the paged 4-bit key / value cache: append with rotation, read back, and the C ABI
// (include/gcq_paged.h; layout in paged.h).
#include "paged.h"

#include <algorithm>
#include <cmath>

#include "../../include/gcq_paged.h"

namespace gcq {

namespace {

struct AppendArgs {
    Paged p;
    const float * k, * v, * q;
    int64_t k_r, k_h, v_r, v_h, q_r, q_h;
    _Float16 * q_out;
    const float * freqs;
    float attn_factor;
    int H, n_dims, per, parts;  // heads (of H + 2 Hkv) per wavefront, wavefronts per row
};

// ---------------------------------------------------------------------------------- append

// One element of a turned pair: x c + p s, p its partner (s negated for the pair's first).
__device__ __forceinline__ float turned(float x, double c, float p, double s) { return (float) fma((double) x, c, (double) p * s); }

// What is held of a value: NaN as 0, the rest within f16.
__device__ __forceinline__ float held(float w) { return w == w ? fminf(fmaxf(w, -kPagedMax), kPagedMax) : 0.0f; }

// A block's scale from its largest value (ggml's Q4_0: the first of the largest becomes code 0), and a value's code.
__device__ __forceinline__ float block_scale(float m, bool minus) { return (minus ? m : -m) * 0.125f; }
__device__ __forceinline__ float block_inverse(float d) { return d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f; }
__device__ __forceinline__ int code_of(float w, float inverse) {
#pragma clang fp contract(off)
    return max(min((int) (w * inverse + 8.5f), 15), 0);
}

// One row at a time: a wavefront takes `per` heads of it. Lane i holds dims i and i + D / 2 (D = 64: a head per half wavefront; 256: two
// such pairs), so a NEOX pair, a code byte and, per register and half wavefront, a whole block are at hand without an
// exchange but the block's maximum. The row's sines are computed once per wavefront, in 64 bits: a 32-bit angle is off by
// 2^-24 of itself, 0.006 radians at position 10^5, and codes would follow the error. Latency: 3.9 us for a row of 32 heads,
// 8 + 8 KV heads of 128, 5.8 us for 64 sequences' rows.
template <int D, bool FULL>
__global__ __launch_bounds__(256) void k_paged_append(const AppendArgs a) {
    constexpr int NP = D == 256 ? 2 : 1, HS = D == 64 ? 2 : 1;
    const int lane = threadIdx.x & 63, il = D == 64 ? lane & 31 : lane;
    const int64_t unit = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    const int r = (int) (unit / a.parts);
    if (r >= a.p.n_rows) return;  // whole wavefronts
    const int s = paged_seq(a.p, r);
    if (s < 0) return;
    const int64_t pos = (int64_t) a.p.past[s] + (r - a.p.starts[s]);
    const int h0 = (int) (unit % a.parts) * a.per, h1 = min(h0 + a.per, a.H + 2 * a.p.Hkv);
    const int slot = (int) pos & 31;

    // cos and sin of each element's pair (FULL: an element and its partner share them)
    constexpr int NC = FULL ? NP : 2 * NP;
    double cs[NC], sn[NC];
    const int half = a.n_dims / 2;
    const bool turn = a.freqs && h0 < a.H + a.p.Hkv;
    if (turn) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int e = FULL ? il + 64 * c : il + 64 * (c >> 1) + (c & 1) * (D / 2);
            cs[c] = 1.0;
            sn[c] = 0.0;
            if (FULL || e < a.n_dims) {
                sincos((double) pos * (double) a.freqs[!FULL && e >= half ? e - half : e], &sn[c], &cs[c]);
                cs[c] *= (double) a.attn_factor;
                sn[c] *= (double) a.attn_factor;
            }
        }
    }
    for (int hb = h0; hb < h1; hb += HS) {
        const int h = D == 64 ? hb + (lane >> 5) : hb;
        const bool on = h < h1, is_q = h < a.H, is_k = !is_q && h < a.H + a.p.Hkv;
        const int hk = is_k ? h - a.H : h - a.H - a.p.Hkv;
        const float * x = is_q ? a.q + r * a.q_r + h * a.q_h : is_k ? a.k + r * a.k_r + hk * a.k_h : a.v + r * a.v_r + hk * a.v_h;
        float y[NP][2];
#pragma unroll
        for (int n = 0; n < NP; n++) {
            const int i = il + 64 * n;
            y[n][0] = on ? x[i] : 0.0f;
            y[n][1] = on ? x[i + D / 2] : 0.0f;
            if (turn && (is_q || is_k) && on) {
                if constexpr (FULL) {
                    const float u = y[n][0], w = y[n][1];
                    y[n][0] = turned(u, cs[n], w, -sn[n]);
                    y[n][1] = turned(w, cs[n], u, sn[n]);
                } else {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int d = i + e * (D / 2), c = 2 * n + e;
                        if (d < half) y[n][e] = turned(y[n][e], cs[c], x[d + half], -sn[c]);
                        else if (d < a.n_dims) y[n][e] = turned(y[n][e], cs[c], x[d - half], sn[c]);
                    }
                }
            }
        }
        if (on && is_q) {
            _Float16 * o = a.q_out + ((int64_t) r * a.H + h) * D;
#pragma unroll
            for (int n = 0; n < NP; n++) {
                o[il + 64 * n] = (_Float16) y[n][0];
                o[il + 64 * n + D / 2] = (_Float16) y[n][1];
            }
        }
        if (hb + HS <= a.H) continue;
        const int64_t tile = on && !is_q ? paged_tile(a.p, s, pos, hk, D) : -1;
#pragma unroll
        for (int n = 0; n < NP; n++) {
            int code[2];
            float d[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float w = held(y[n][e]);
                const float m = wave_max<32>(fabsf(w));
                const uint64_t at = __ballot(fabsf(w) == m), neg = __ballot(w < 0.0f);
                const uint32_t at32 = (uint32_t) (lane < 32 ? at : at >> 32), neg32 = (uint32_t) (lane < 32 ? neg : neg >> 32);
                const bool minus = neg32 >> __builtin_ctz(at32) & 1;  // the first of the largest
                d[e] = block_scale(m, minus);
                code[e] = code_of(w, block_inverse(d[e]));
            }
            if (tile >= 0) {
                const int i = il + 64 * n;
                uint8_t * t = a.p.data + tile;
                t[is_k ? paged_k_byte<D>(slot, i) : paged_v_byte<D>(slot, i)] = (uint8_t) (code[0] | code[1] << 4);
                if ((lane & 31) == 0)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int b = i / 32 + e * (D / 64);
                        *(uint16_t *) (t + (is_k ? paged_k_scale<D>(slot, b) : paged_v_scale<D>(slot, b))) = f2h_exact(d[e]);
                    }
            }
        }
    }
}

// Eight tokens of a tile (one of its four parts) put side by side: 9 D bytes, and where their 16-byte pieces belong in the tile.
template <int D>
struct Eight {
    static constexpr int kPieces = 9 * D / 16;  // D / 4 of K's codes (D / 32 to a token), D / 4 of V's, one of scales for each block
    static __device__ __forceinline__ int k_byte(int m, int i) { return paged_k_byte<D>(m, i); }
    static __device__ __forceinline__ int v_byte(int m, int i) { return 4 * D + (i >> 5) * 256 + (i & 15) * 16 + (i >> 4 & 1) * 8 + m; }
    static __device__ __forceinline__ int scale(int m, int b, int v) { return 8 * D + 16 * (b + v * (D / 32)) + 2 * paged_order(m); }
    static __device__ __forceinline__ int piece(int c, int g) {
        if (c < D / 4) return 4 * D * g + 16 * c;
        if (c < D / 2) return 16 * D + ((c - D / 4) >> 4) * 1024 + g * 256 + (c & 15) * 16;
        return 32 * D + (c - D / 2) * 64 + g * 16;
    }
};

// Many rows of a sequence: a workgroup takes eight positions of a tile for one KV head, and their rows of q heads hk,
// hk + Hkv, .. A thread has four pairs of one row for all of those heads, their sines in registers; the eight tokens' bytes are
// put together in LDS and leave as 16-byte pieces, where a row at a time writes V's one by one. (By eights and not by whole tiles:
// four times the workgroups, whose waits overlap; 8192 rows of 16 heads, 8 + 8 KV heads of 256: 85 us, by tiles 121.) 3998 rows of 32
// heads, 8 + 8 KV heads of 128: 31 us for 136 MB, 4.4 TB/s, where a large copy reaches 5.1; 7 us of it are the rotation's 64-bit
// operations. Of a part of the dims (FULL false) partners are loaded besides and there are sines for both: 64 of 128 dims 31 us as well,
// 128 of 256 dims, 8192 rows of 16 heads, 98 us for 81.
template <int D, bool FULL>
__global__ __launch_bounds__(D) void k_paged_append_eight(const AppendArgs a) {
    constexpr int L = D / 8, QB = FULL ? 2 : 1;  // threads of a row; q heads under way at a time, as the registers allow
    __shared__ __align__(16) uint8_t image[9 * D];
    const int tid = threadIdx.x, lane = tid & 63, m8 = tid / L, i = 4 * (tid % L), hk = blockIdx.x % a.p.Hkv;
    PagedSpan w;
    if (!paged_find(a.p, blockIdx.x / a.p.Hkv, w)) return;
    const int64_t pos = w.eight * 8 + m8, j = pos - w.past;
    const bool on = j >= 0 && j < w.rows;
    const int64_t r = w.r0 + (on ? j : 0);
    const int half = a.n_dims / 2;

    // of dims i .. i + 3 and i + D / 2 ..: values, and partners (FULL: each other)
    typedef float f4_t __attribute__((ext_vector_type(4)));
    struct Four {
        f4_t x[2], p[FULL ? 1 : 2];
    };
    const auto fetch = [&](const float * x, bool turn) {
        Four f{};
        if (!on) return f;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int d = i + e * (D / 2);
            f.x[e] = *reinterpret_cast<const f4_t *>(x + d);
            if constexpr (!FULL)
                if (turn && d < a.n_dims) f.p[e] = *reinterpret_cast<const f4_t *>(x + (d < half ? d + half : d - half));
        }
        return f;
    };
    const auto q_at = [&](int h) { return a.q + r * a.q_r + min(h, a.H - 1) * a.q_h; };
    Four k = fetch(a.k + r * a.k_r + hk * a.k_h, true), v = fetch(a.v + r * a.v_r + hk * a.v_h, false), q[QB];
    if (a.q)
#pragma unroll
        for (int n = 0; n < QB; n++) q[n] = fetch(q_at(hk + n * a.p.Hkv), true);

    constexpr int NC = FULL ? 1 : 2;
    double cs[NC][4], sn[NC][4];
    if (a.freqs) {
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int d = i + e + c * (D / 2);
                cs[c][e] = 1.0;
                sn[c][e] = 0.0;
                if (FULL || d < a.n_dims) {
                    sincos((double) pos * (double) a.freqs[!FULL && d >= half ? d - half : d], &sn[c][e], &cs[c][e]);
                    cs[c][e] *= (double) a.attn_factor;
                    sn[c][e] *= !FULL && d < half ? -(double) a.attn_factor : (double) a.attn_factor;
                }
            }
    }
    const auto turn = [&](Four & f) {
        if (!a.freqs) return;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float x0 = f.x[0][e], x1 = f.x[1][e];
            if (FULL || i < a.n_dims) f.x[0][e] = FULL ? turned(x0, cs[0][e], x1, -sn[0][e]) : turned(x0, cs[0][e], f.p[0][e], sn[0][e]);
            if (FULL || i + D / 2 < a.n_dims) f.x[1][e] = FULL ? turned(x1, cs[0][e], x0, sn[0][e]) : turned(x1, cs[NC - 1][e], f.p[FULL ? 0 : 1][e], sn[NC - 1][e]);
        }
    };
    const int64_t tile = paged_tile(a.p, w.s, w.eight * 8, hk, D);  // (-1 for all eight or none)
    turn(k);
#pragma unroll
    for (int c = 0; c < 2; c++) {
        int code[2][4];
        float d[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f4_t y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = held((c ? v : k).x[h][e]);
            float m = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
            m = fmaxf(m, lane_pair<1>(m));  // over the block's 8 lanes
            m = fmaxf(m, lane_pair<2>(m));
            m = fmaxf(m, lane_pair<4>(m));
            bool at = false, neg = false;  // the first of the largest
#pragma unroll
            for (int e = 3; e >= 0; e--)
                if (fabsf(y[e]) == m) at = true, neg = y[e] < 0.0f;
            const uint32_t ats = (uint32_t) (__ballot(at) >> (lane & 56)) & 255, negs = (uint32_t) (__ballot(neg) >> (lane & 56));
            d[h] = block_scale(m, negs >> __builtin_ctz(ats) & 1);
            const float id = block_inverse(d[h]);
#pragma unroll
            for (int e = 0; e < 4; e++) code[h][e] = code_of(y[e], id);
        }
        if (c == 0) {
            uint32_t bytes = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) bytes |= (uint32_t) (code[0][e] | code[1][e] << 4) << (8 * e);
            *reinterpret_cast<uint32_t *>(image + Eight<D>::k_byte(m8, i)) = bytes;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) image[Eight<D>::v_byte(m8, i + e)] = (uint8_t) (code[0][e] | code[1][e] << 4);
        }
        if ((lane & 7) == 0)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int b = i / 32 + h * (D / 64);
                *reinterpret_cast<uint16_t *>(image + Eight<D>::scale(m8, b, c)) = f2h_exact(d[h]);
            }
    }
    if (a.q) {
        typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
        for (int h0 = hk; h0 < a.H; h0 += QB * a.p.Hkv) {
            if (h0 != hk)
#pragma unroll
                for (int n = 0; n < QB; n++) q[n] = fetch(q_at(h0 + n * a.p.Hkv), true);
#pragma unroll
            for (int n = 0; n < QB; n++) {
                const int h = h0 + n * a.p.Hkv;
                if (h >= a.H || !on) break;
                turn(q[n]);
                _Float16 * o = a.q_out + (r * a.H + h) * D + i;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const f4_t y = q[n].x[e];
                    const h4_t u = {(_Float16) y[0], (_Float16) y[1], (_Float16) y[2], (_Float16) y[3]};
                    __builtin_memcpy(o + e * (D / 2), &u, 8);
                }
            }
        }
    }
    __syncthreads();
    if (tile < 0 || tid >= Eight<D>::kPieces) return;
    // in part where some of the eight are not this batch's
    const int64_t s0 = w.past - w.eight * 8, s1 = s0 + w.rows;
    const uint32_t have = (s1 >= 8 ? 255 : (1u << s1) - 1) & (s0 > 0 ? 255u << s0 : 255);
    uint8_t * o = a.p.data + tile + Eight<D>::piece(tid, (int) w.eight & 3);
    const uint8_t * from = image + 16 * tid;
    if (have == 255 || (tid < D / 4 && have >> tid / (D / 32) & 1)) *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<const uint4 *>(from);
    else if (tid < D / 4) return;
    else if (tid < D / 2) {
        for (int b = 0; b < 16; b++)
            if (have >> (b & 7) & 1) o[b] = from[b];
    } else {
        for (int e = 0; e < 8; e++)
            if (have >> paged_order(e) & 1) *reinterpret_cast<uint16_t *>(o + 2 * e) = *reinterpret_cast<const uint16_t *>(from + 2 * e);
    }
}

// ------------------------------------------------------------------------------------ read

struct ReadArgs {
    Paged p;
    float * k, * v;
};

// A workgroup takes eight positions for one KV head, by way of LDS; a thread gives four pairs of one row. Bound by its writes:
// 4096 rows of 8 KV heads of 128 in 8.9 us, 38 MB, 4.3 TB/s.
template <int D>
__global__ __launch_bounds__(D) void k_paged_read(const ReadArgs a) {
    constexpr int L = D / 8;
    __shared__ __align__(16) uint8_t image[9 * D];
    const int tid = threadIdx.x, m8 = tid / L, i = 4 * (tid % L), hk = blockIdx.x % a.p.Hkv;
    PagedSpan w;
    if (!paged_find(a.p, blockIdx.x / a.p.Hkv, w)) return;
    const int64_t tile = paged_tile(a.p, w.s, w.eight * 8, hk, D);
    if (tile >= 0 && tid < Eight<D>::kPieces)
        *reinterpret_cast<uint4 *>(image + 16 * tid) = *reinterpret_cast<const uint4 *>(a.p.data + tile + Eight<D>::piece(tid, (int) w.eight & 3));
    __syncthreads();
    const int64_t j = w.eight * 8 + m8 - w.past;
    if (j < 0 || j >= w.rows) return;
    typedef float f4_t __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int c = 0; c < 2; c++) {
        f4_t y[2] = {};
        if (tile >= 0) {
            uint32_t b = 0;
            if (c == 0) b = *reinterpret_cast<const uint32_t *>(image + Eight<D>::k_byte(m8, i));
            else
#pragma unroll
                for (int e = 0; e < 4; e++) b |= (uint32_t) image[Eight<D>::v_byte(m8, i + e)] << (8 * e);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int blk = i / 32 + h * (D / 64);
                const float d = h2f(*reinterpret_cast<const uint16_t *>(image + Eight<D>::scale(m8, blk, c)));
#pragma unroll
                for (int e = 0; e < 4; e++) y[h][e] = d * (float) ((int) (b >> (8 * e + 4 * h) & 15) - 8);
            }
        }
        float * o = (c ? a.v : a.k) + ((w.r0 + j) * a.p.Hkv + hk) * D + i;
        *reinterpret_cast<f4_t *>(o) = y[0];
        *reinterpret_cast<f4_t *>(o + D / 2) = y[1];
    }
}

// ---------------------------------------------------------------------------------- checks

// (messages are put together only where a check fails: a launch costs the host some 3 us, a call's strings were one more)
void require(bool ok, const char * message) {
    if (!ok) fail(message);
}
void need(const void * p, const char * what, size_t align = 1) {
    if (!p) fail(std::string("paged: ") + what + " is NULL");
    if (!aligned(p, align)) fail(std::string("paged: ") + what + " must be " + std::to_string(align) + "-byte aligned");
}

bool shape_ok(int n_pages, int page, int Hkv, int D) {
    return n_pages > 0 && Hkv > 0 && Hkv <= 65535 && (page == 32 || page == 64 || page == 128 || page == 256) &&
           (D == 64 || D == 128 || D == 256);
}

Paged view(const gcq_paged_cache * c, const gcq_paged_batch * b, int64_t n_rows, bool pointers = true) {
    need(c, "cache");
    need(b, "batch");
    require(shape_ok(c->n_pages, c->page_size, c->n_head_kv, c->head_dim),
            "paged: pages of 32, 64, 128 or 256 tokens, heads of 64, 128 or 256 values, at least one page and KV head");
    require(b->n_seq > 0 && b->max_pages > 0 && b->ld_pages >= b->max_pages,
            "paged: a batch has at least one sequence and one page each, ld_pages >= max_pages");
    require(n_rows >= 0 && n_rows < (1 << 30), "paged: n_rows out of range");
    if (pointers) {
        need(c->data, "cache data", 16);
        need(b->pages, "pages", 4);
        need(b->starts, "starts", 4);
        need(b->past, "past", 4);
    }
    Paged p{};
    p.data = (uint8_t *) c->data;
    p.pages = b->pages, p.ld = b->ld_pages, p.starts = b->starts, p.past = b->past;
    p.n_pages = c->n_pages, p.shift = __builtin_ctz((unsigned) c->page_size), p.Hkv = c->n_head_kv;
    p.n_seq = b->n_seq, p.max_pages = b->max_pages, p.n_rows = (int) n_rows;
    return p;
}

// Whether rows are appended eight positions at a time: a sequence fills half an eight at the least, and there are 2^20 values,
// enough to pay for a workgroup's longer way. (64 sequences, 32 heads and 8 KV heads of 128, rows one by one and by
// eights: 2 rows each 6.9 and 7.9 us, 4 rows 8.7 and 8.0, 16 rows 21.1 and 10.6; one sequence: 32 rows 4.4 and 6.3, 128 rows
// 6.7 and 6.4.)
bool by_eights(const AppendArgs & a, int D) {
    return a.p.n_rows >= 4 * std::min(a.p.n_seq, a.p.n_rows) && (int64_t) a.p.n_rows * (a.H + 2 * a.p.Hkv) * D >= 1 << 20;
}
unsigned eight_blocks(const Paged & p, int threads) {  // a sequence's rows may begin and end inside an eight
    return paged_grid((p.n_rows / 8 + 2 * (int64_t) std::min(p.n_seq, p.n_rows)) * p.Hkv, threads);
}
bool vectors(const float * x, int64_t r, int64_t h) { return aligned(x, 16) && r % 4 == 0 && h % 4 == 0; }

template <int D>
void run_append(const AppendArgs & a, hipStream_t s) {
    const bool full = !a.freqs || a.n_dims == D;
    if (by_eights(a, D) && a.n_dims % 8 == 0 && vectors(a.k, a.k_r, a.k_h) && vectors(a.v, a.v_r, a.v_h) &&
        (!a.q || (vectors(a.q, a.q_r, a.q_h) && aligned(a.q_out, 8)))) {
        if (full) k_paged_append_eight<D, true><<<eight_blocks(a.p, D), D, 0, s>>>(a);
        else k_paged_append_eight<D, false><<<eight_blocks(a.p, D), D, 0, s>>>(a);
        return;
    }
    const unsigned grid = paged_grid(((int64_t) a.p.n_rows * a.parts + 3) / 4, 256);
    if (full) k_paged_append<D, true><<<grid, 256, 0, s>>>(a);
    else k_paged_append<D, false><<<grid, 256, 0, s>>>(a);
}
template <int D>
void run_read(const ReadArgs & a, hipStream_t s) {
    k_paged_read<D><<<eight_blocks(a.p, D), D, 0, s>>>(a);
}

}  // namespace

}  // namespace gcq

using namespace gcq;

extern "C" {

size_t gcq_paged_cache_size(int n_pages, int page_size, int n_head_kv, int head_dim) {
    if (!shape_ok(n_pages, page_size, n_head_kv, head_dim)) {
        set_error("paged_cache_size: pages of 32, 64, 128 or 256 tokens, heads of 64, 128 or 256 values");
        return 0;
    }
    return (size_t) n_pages * (size_t) n_head_kv * (size_t) (page_size / kPagedTile) * (size_t) (36 * head_dim);
}

int gcq_paged_append(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows, const float * k,
                     int64_t k_r, int64_t k_h, const float * v, int64_t v_r, int64_t v_h, const float * q, int64_t q_r,
                     int64_t q_h, int n_head, void * q_out, const float * freqs, int n_dims, float attn_factor,
                     void * stream) {
    return guarded([&] {
        AppendArgs a{};
        a.p = view(cache, batch, n_rows);
        if (n_rows == 0) return;
        const int D = cache->head_dim;
        need(k, "k", 4);
        need(v, "v", 4);
        require(k_r >= 0 && k_h >= 0 && v_r >= 0 && v_h >= 0 && q_r >= 0 && q_h >= 0, "paged_append: negative strides");
        if (q) {
            need(q, "q", 4);
            need(q_out, "q_out", 2);
            require(n_head > 0 && n_head <= 65535, "paged_append: n_head must be positive");
        }
        if (freqs) {
            need(freqs, "freqs", 4);
            require(n_dims > 0 && n_dims % 2 == 0 && n_dims <= D, "paged_append: n_dims must be even and <= head_dim");
            require(std::isfinite(attn_factor), "paged_append: attn_factor must be finite");
        }
        a.k = k, a.k_r = k_r, a.k_h = k_h, a.v = v, a.v_r = v_r, a.v_h = v_h;
        a.q = q, a.q_r = q_r, a.q_h = q_h, a.H = q ? n_head : 0, a.q_out = (_Float16 *) q_out;
        a.freqs = freqs, a.n_dims = freqs ? n_dims : D, a.attn_factor = attn_factor;
        const int64_t heads = a.H + 2 * a.p.Hkv;
        // wavefronts: about 4096, one per row at the least
        a.per = (int) std::max<int64_t>(1, std::min(heads, heads * n_rows / 4096));
        if (D == 64) a.per = (a.per + 1) / 2 * 2;
        a.parts = (int) ((heads + a.per - 1) / a.per);
        hipStream_t s = as_stream(stream);
        if (D == 64) run_append<64>(a, s);
        else if (D == 128) run_append<128>(a, s);
        else run_append<256>(a, s);
        check_launch("paged append");
    });
}

int gcq_paged_read(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows, float * k, float * v,
                   void * stream) {
    return guarded([&] {
        ReadArgs a{view(cache, batch, n_rows), k, v};
        if (n_rows == 0) return;
        need(k, "k", 16);
        need(v, "v", 16);
        hipStream_t s = as_stream(stream);
        if (cache->head_dim == 64) run_read<64>(a, s);
        else if (cache->head_dim == 128) run_read<128>(a, s);
        else run_read<256>(a, s);
        check_launch("paged read");
    });
}

size_t gcq_paged_attn_workspace(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows, int n_head,
                                int64_t max_rows) {
    size_t n = 0;
    guarded([&] {
        const Paged p = view(cache, batch, n_rows, false);
        require(n_head > 0 && n_head % p.Hkv == 0, "paged_attn: n_head must be a multiple of n_head_kv");
        require(max_rows > 0, "paged_attn: max_rows must be positive");
        n = std::max<size_t>(256, paged_attn_workspace(p, cache->head_dim, n_head, max_rows));
    });
    return n;
}

int gcq_paged_attn(const gcq_paged_cache * cache, const gcq_paged_batch * batch, int64_t n_rows, const void * q,
                   int64_t q_r, int64_t q_h, int n_head, int64_t max_rows, int window, float scale, float * out, void * ws,
                   size_t ws_size, void * stream) {
    return guarded([&] {
        const Paged p = view(cache, batch, n_rows);
        if (n_rows == 0) return;
        need(q, "q", 16);
        need(out, "out", 16);
        need(ws, "workspace", 256);
        require(n_head > 0 && n_head <= 65535 && n_head % p.Hkv == 0, "paged_attn: n_head must be a multiple of n_head_kv");
        require(q_r >= 0 && q_h >= 0 && q_r % 8 == 0 && q_h % 8 == 0, "paged_attn: q strides must be multiples of 8");
        require(max_rows > 0, "paged_attn: max_rows must be positive");
        require(window >= 0, "paged_attn: window must not be negative");
        require(std::isfinite(scale), "paged_attn: scale must be finite");
        const size_t need_ws = std::max<size_t>(256, paged_attn_workspace(p, cache->head_dim, n_head, max_rows));
        if (ws_size < need_ws) fail("workspace of " + std::to_string(ws_size) + " bytes, need " + std::to_string(need_ws));
        launch_paged_attn(p, cache->head_dim, q, q_r, q_h, n_head, max_rows, window, scale, out, ws, as_stream(stream));
    });
}

}  // extern "C"

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

// A wavefront takes `per` heads of one row. Lane i holds dims i and i + D / 2 (D = 64: a head per half wavefront; 256: two
// such pairs), so a NEOX pair, a code byte and, per register and half wavefront, a whole block are at hand without an
// exchange but the block's maximum. The row's sines are computed once per wavefront, in 64 bits: a 32-bit angle is off by
// 2^-24 of the position, half a percent of a turn at 10^5, and codes would follow the error.
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
                    const double u = y[n][0], w = y[n][1];
                    y[n][0] = (float) (u * cs[n] - w * sn[n]);
                    y[n][1] = (float) (u * sn[n] + w * cs[n]);
                } else {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int d = i + e * (D / 2), c = 2 * n + e;
                        if (d < half) y[n][e] = (float) ((double) y[n][e] * cs[c] - (double) x[d + half] * sn[c]);
                        else if (d < a.n_dims) y[n][e] = (float) ((double) x[d - half] * sn[c] + (double) y[n][e] * cs[c]);
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
#pragma clang fp contract(off)
            int code[2];
            float d[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float w = y[n][e];
                w = w == w ? fminf(fmaxf(w, -kPagedMax), kPagedMax) : 0.0f;
                const float m = wave_max<32>(fabsf(w));
                const uint64_t at = __ballot(fabsf(w) == m), neg = __ballot(w < 0.0f);
                const uint32_t at32 = (uint32_t) (lane < 32 ? at : at >> 32), neg32 = (uint32_t) (lane < 32 ? neg : neg >> 32);
                const bool minus = neg32 >> __builtin_ctz(at32) & 1;  // the first of the largest
                d[e] = (minus ? m : -m) * 0.125f;
                const float id = d[e] != 0.0f ? __fdiv_rn(1.0f, d[e]) : 0.0f;
                code[e] = max(min((int) (w * id + 8.5f), 15), 0);
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

// ------------------------------------------------------------------------------------ read

struct ReadArgs {
    Paged p;
    float * k, * v;
};

// A wavefront takes one row of one KV head, keys and values.
template <int D>
__global__ __launch_bounds__(256) void k_paged_read(const ReadArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    const int r = (int) (unit / a.p.Hkv), h = (int) (unit % a.p.Hkv);
    if (r >= a.p.n_rows) return;
    const int s = paged_seq(a.p, r);
    if (s < 0) return;
    const int64_t pos = (int64_t) a.p.past[s] + (r - a.p.starts[s]);
    const int slot = (int) pos & 31;
    const int64_t tile = paged_tile(a.p, s, pos, h, D);
#pragma unroll
    for (int c = 0; c < 2; c++) {
        float * o = (c ? a.v : a.k) + unit * D;
        for (int i = lane; i < D / 2; i += 64) {
            float lo = 0.0f, hi = 0.0f;
            if (tile >= 0) {
                const uint8_t * t = a.p.data + tile;
                const int b = t[c ? paged_v_byte<D>(slot, i) : paged_k_byte<D>(slot, i)];
                const auto scale = [&](int blk) { return h2f(*(const uint16_t *) (t + (c ? paged_v_scale<D>(slot, blk) : paged_k_scale<D>(slot, blk)))); };
                lo = scale(i / 32) * (float) ((b & 15) - 8);
                hi = scale(i / 32 + D / 64) * (float) ((b >> 4) - 8);
            }
            o[i] = lo;
            o[i + D / 2] = hi;
        }
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

unsigned blocks(int64_t waves) {
    require(waves <= (int64_t) 4 * INT32_MAX, "paged: too many rows and heads");
    return (unsigned) ((waves + 3) / 4);
}

template <int D>
void run_append(const AppendArgs & a, hipStream_t s) {
    const unsigned grid = blocks((int64_t) a.p.n_rows * a.parts);
    if (!a.freqs || a.n_dims == D) k_paged_append<D, true><<<grid, 256, 0, s>>>(a);
    else k_paged_append<D, false><<<grid, 256, 0, s>>>(a);
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
        need(k, "k", 4);
        need(v, "v", 4);
        hipStream_t s = as_stream(stream);
        const unsigned grid = blocks(n_rows * a.p.Hkv);
        if (cache->head_dim == 64) k_paged_read<64><<<grid, 256, 0, s>>>(a);
        else if (cache->head_dim == 128) k_paged_read<128><<<grid, 256, 0, s>>>(a);
        else k_paged_read<256><<<grid, 256, 0, s>>>(a);
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

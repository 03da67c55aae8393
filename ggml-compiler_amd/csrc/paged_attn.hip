// paged_attn.hip - attention over the paged 4-bit cache (include/gcq_paged.h; layout in paged.h).
#include "paged.h"

namespace gcq {

namespace {

struct AttnArgs {
    Paged p;
    const _Float16 * q;
    int64_t q_r, q_h;
    int H, window, max_rows;
    float scale2;  // scale * log2(e)
    float * out;
};

// One wavefront per (row, query head): 64 keys at a time, a key per lane for the scores, dims by lane for P V.
template <int D>
__global__ __launch_bounds__(64) void k_paged_attn_row(const AttnArgs a) {
    __shared__ float sq[D], sp[64];
    __shared__ int64_t st[64];
    const int lane = threadIdx.x, r = blockIdx.x, h = blockIdx.y, hk = h / (a.H / a.p.Hkv);
    const int s = paged_seq(a.p, r);
    if (s < 0 || r - a.p.starts[s] >= a.max_rows) return;
    const int64_t pos = (int64_t) a.p.past[s] + (r - a.p.starts[s]);
    const int64_t end = min(pos + 1, (int64_t) a.p.max_pages << a.p.shift);
    const int64_t first = a.window && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    for (int i = lane; i < D; i += 64) sq[i] = (float) a.q[r * a.q_r + h * a.q_h + i];
    float m = -INFINITY, l = 0.0f, o[D / 64] = {};
    for (int64_t j0 = first & ~(int64_t) 63; j0 < end; j0 += 64) {
        __syncthreads();
        const int64_t j = j0 + lane;
        const int64_t tile = j >= first && j < end ? paged_tile(a.p, s, j, hk, D) : -1;
        float x = -INFINITY;
        if (tile >= 0) {
            const uint8_t * t = a.p.data + tile;
            x = 0.0f;
            for (int b = 0; b < D / 32; b++) {
                float dot = 0.0f;
                for (int e = 0; e < 32; e++) {
                    const int d = 32 * b + e, c = t[paged_k_byte<D>((int) j & 31, d % (D / 2))];
                    dot = fmaf(sq[d], (float) ((d < D / 2 ? c & 15 : c >> 4) - 8), dot);
                }
                x = fmaf(h2f(*(const uint16_t *) (t + paged_k_scale<D>((int) j & 31, b))), dot, x);
            }
            x *= a.scale2;
        }
        const float mn = fmaxf(m, wave_max(x));
        const float base = mn == -INFINITY ? 0.0f : mn, al = __builtin_amdgcn_exp2f(m - base);
        const float p = __builtin_amdgcn_exp2f(x - base);
        m = mn;
        l = fmaf(l, al, wave_sum(p));
        sp[lane] = p;
        st[lane] = tile;
        __syncthreads();
        for (int n = 0; n < D / 64; n++) o[n] *= al;
        for (int k = 0; k < 64; k++) {
            if (st[k] < 0) continue;
            const uint8_t * t = a.p.data + st[k];
            for (int n = 0; n < D / 64; n++) {
                const int d = lane + 64 * n, c = t[paged_v_byte<D>((int) (j0 + k) & 31, d % (D / 2))];
                const float v = h2f(*(const uint16_t *) (t + paged_v_scale<D>((int) (j0 + k) & 31, d / 32))) *
                                (float) ((d < D / 2 ? c & 15 : c >> 4) - 8);
                o[n] = fmaf(sp[k], v, o[n]);
            }
        }
    }
    for (int n = 0; n < D / 64; n++) a.out[((int64_t) r * a.H + h) * D + lane + 64 * n] = l == 0.0f ? 0.0f : o[n] / l;
}

}  // namespace

size_t paged_attn_workspace(const Paged &, int, int, int64_t) { return 256; }

void launch_paged_attn(const Paged & p, int D, const void * q, int64_t q_r, int64_t q_h, int H, int64_t max_rows, int window,
                       float scale, float * out, void *, hipStream_t s) {
    AttnArgs a{};
    a.p = p, a.q = (const _Float16 *) q, a.q_r = q_r, a.q_h = q_h, a.H = H, a.window = window;
    a.max_rows = (int) (max_rows < p.n_rows ? max_rows : p.n_rows);
    a.scale2 = (float) ((double) scale * 1.4426950408889634074);
    a.out = out;
    const dim3 grid((unsigned) p.n_rows, (unsigned) H);
    if (D == 64) k_paged_attn_row<64><<<grid, 64, 0, s>>>(a);
    else if (D == 128) k_paged_attn_row<128><<<grid, 64, 0, s>>>(a);
    else k_paged_attn_row<256><<<grid, 64, 0, s>>>(a);
    check_launch("paged attn");
}

}  // namespace gcq

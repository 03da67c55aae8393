// paged_attn.hip - attention over the paged 4-bit cache (include/gcq_paged.h; layout in paged.h).
//
// k_paged_few: a wavefront takes 16 rows, a row being a (query, head) pair of one KV head (row j G + g), and tiles of 32
// keys, straight from memory into the matrix cores' operands:
//   - scores S^T[key][row] = K Q^T, one v_mfma_f32_16x16x32_f16 per Q4_0 block of 32 dims and 16 keys, on the codes c - 8
//     themselves (exact in f16); a block's sum is scaled by its d in f32.
//   - lane (row, g) is left with the scores of keys 8 g .. 8 g + 7, in the order that P V's operand wants them;
//   - O^T[dim][row] += V^T P^T, V's values d (c - 8) as two f16 parts (15 bits: exact), P as two of 11 bits, cut off; the
//     sum of weights goes through the same two parts (a row of ones), so that numerator and denominator see the same.
// The softmax runs in powers of two against an integer reference R that follows the maximum in steps: it moves when a score
// passes it by 4, which is rare, and moving it scales by an exact power of two. Chains inside the MFMAs (whose sums are
// cut off, not rounded) start from zero for each tile; tiles are added in f32.
//
// Work: a sequence's tiles are cut into splits of `chunk` tiles, the same for all sequences, chosen so that all splits of all
// sequences make about kTarget workgroups. Every workgroup computes that plan from the batch's arrays by itself (no planning
// launch, and a captured graph follows the arrays), finds its split by a prefix sum over the sequences, deals its
// tiles to its wavefronts in turn and joins their sums in LDS. Sequences of several splits are joined by k_paged_merge.
#include "paged.h"

#include <algorithm>

namespace gcq {

namespace {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr int kTarget = 1024;    // workgroups that the splits aim at
constexpr int kMinChunk = 16;    // tiles: a shorter split costs more in the merge than it saves
constexpr float kSlack = 4.0f;   // how far a score's exponent may pass R
constexpr float kBig = 0x1p20f;  // exponents from here on are no longer exact to 2^-4
constexpr float kP = 2048.0f;    // P's scale: 2^11 2^kSlack is f16's 2^15

struct AttnArgs {
    Paged p;
    const _Float16 * q;
    int64_t q_r, q_h;
    int H, G, window, max_rows, items;
    float c2;     // |scale| log2(e)
    bool negate;  // the scale is negative
    float * out, * part_o;
    float2 * part_ml;
};

// A sequence's rows, the keys [lo, hi) that any of them sees, their tiles and row tiles.
struct SeqWork {
    int r0, rows, tile0, tiles, rts;
    int64_t past;
};
template <int ROWS>
__device__ __forceinline__ SeqWork seq_work(const AttnArgs & a, int s) {
    SeqWork w{};
    if (s >= a.p.n_seq) return w;
    w.r0 = a.p.starts[s];
    const int r1 = min(a.p.starts[s + 1], a.p.n_rows);
    if (w.r0 < 0 || r1 <= w.r0) return w;
    w.rows = min(r1 - w.r0, a.max_rows);
    w.past = a.p.past[s];
    const int64_t hi = min(w.past + w.rows, (int64_t) a.p.max_pages << a.p.shift);
    const int64_t lo = a.window && w.past - a.window + 1 > 0 ? w.past - a.window + 1 : 0;
    w.tile0 = (int) (lo >> 5);
    w.tiles = hi > lo ? (int) ((hi + 31) >> 5) - w.tile0 : 0;
    w.rts = (int) (((int64_t) w.rows * a.G + ROWS - 1) / ROWS);
    return w;
}
__device__ __forceinline__ int splits(int tiles, int chunk) { return max(1, (tiles + chunk - 1) / chunk); }

// Tiles per split (all lanes together).
template <int ROWS>
__device__ __forceinline__ int plan_chunk(const AttnArgs & a) {
    double u = 0.0;
    for (int s0 = 0; s0 < a.p.n_seq; s0 += 64) {
        const SeqWork w = seq_work<ROWS>(a, s0 + (threadIdx.x & 63));
        u += (double) w.rts * w.tiles;
    }
    u = wave_sum_d(u) * a.p.Hkv;
    return __builtin_amdgcn_readfirstlane((int) max((double) kMinChunk, min(u / kTarget + 1.0, 1e9)));
}

// The sequence whose items hold `item` (-1: none), and the first of its items. Items of a sequence: [KV head][row tile][split].
template <int ROWS>
__device__ __forceinline__ int find_item(const AttnArgs & a, int chunk, int item, int & base) {
    const int lane = threadIdx.x & 63;
    base = 0;
    for (int s0 = 0; s0 < a.p.n_seq; s0 += 64) {
        const SeqWork w = seq_work<ROWS>(a, s0 + lane);
        const int n = w.rts * a.p.Hkv * splits(w.tiles, chunk);
        int sum = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(sum, o, 64);
            if (lane >= o) sum += t;
        }
        const uint64_t after = __ballot(base + sum > item);
        if (after) {
            const int l = __builtin_ctzll(after);
            base += __builtin_amdgcn_readlane(sum - n, l);
            return s0 + l;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}

__device__ __forceinline__ float xor16_max(float v) {
    v = row_pair<16>(v, fmaxf_op);
    return row_pair<32>(v, fmaxf_op);
}

// 8 codes of low (H = 0) or high nibbles as values c - 8, in pairs of f16. (As they lie, masked out as f16 subnormals, they
// cost half the operations, but an MFMA aligns a subnormal's product by its exponent field: 6 to 10 bits of the sum go.)
template <int H>
__device__ __forceinline__ void code_values(uint32_t w0, uint32_t w1, h2_t (&c)[4]) {
    constexpr uint32_t m = H ? 0x00f000f0u : 0x000f000fu;
    const uint32_t w[4] = {w0, w0 >> 8, w1, w1 >> 8};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const h2_t x = __builtin_bit_cast(h2_t, (w[i] & m) | 0x64006400u);  // 1024 + c, 1024 + 16 c
        if constexpr (H) c[i] = x * h2_t{(_Float16) 0.0625f, (_Float16) 0.0625f} - h2_t{(_Float16) 72.0f, (_Float16) 72.0f};
        else c[i] = x - h2_t{(_Float16) 1032.0f, (_Float16) 1032.0f};
    }
}
template <int H>
__device__ __forceinline__ h8_t code_frag(u2_t w) {
    h2_t c[4];
    code_values<H>(w.x, w.y, c);
    return h8_t{c[0].x, c[0].y, c[1].x, c[1].y, c[2].x, c[2].y, c[3].x, c[3].y};
}

template <int D> struct TileRegs {
    u2_t kc[2][D / 64];  // codes of keys order(4 T + ..) of lane group l & 15
    h8_t kd[D / 32];     // scales of the 8 keys of lane group l >> 4
    u4_t vc[D / 64];
    h8_t vd[D / 32];
};

template <int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 256 ? 1 : 2) void k_paged_few(const AttnArgs a) {
    constexpr int ROWS = 16, NB = D / 32, NT = D / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
    const int chunk = plan_chunk<ROWS>(a);
    int base;
    const int s = find_item<ROWS>(a, chunk, blockIdx.x, base);
    if (s < 0) return;
    const SeqWork sw = seq_work<ROWS>(a, s);
    const int ns = splits(sw.tiles, chunk), id = blockIdx.x - base;
    const int split = id % ns, rt = id / ns % sw.rts, hk = id / ns / sw.rts;

    const int x = rt * ROWS + lr, rows = sw.rows * a.G;   // this lane's row
    const int j = min(x, rows - 1) / a.G, h = hk * a.G + min(x, rows - 1) % a.G;
    const int64_t pos = sw.past + j;
    const int64_t pos0 = sw.past + rt * ROWS / a.G, pos1 = sw.past + min(rt * ROWS + ROWS - 1, rows - 1) / a.G;
    // this row tile's keys within the split
    const int64_t cap = (int64_t) a.p.max_pages << a.p.shift;
    const int first = max(sw.tile0 + split * chunk, a.window && pos0 - a.window + 1 > 0 ? (int) ((pos0 - a.window + 1) >> 5) : 0);
    const int last = min(sw.tile0 + min(sw.tiles, (split + 1) * chunk), (int) ((min(pos1 + 1, cap) + 31) >> 5));

    // Q: this lane's row, dims 32 b + 8 g + order(0 .. 7)
    h8_t qf[NB];
    {
        const _Float16 * qp = a.q + (sw.r0 + j) * a.q_r + h * a.q_h + 8 * g;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            h8_t v = *reinterpret_cast<const h8_t *>(qp + 32 * b);
            if (x >= rows) v = h8_t{};
            if (a.negate) v = -v;
            qf[b] = h8_t{v[0], v[2], v[1], v[3], v[4], v[6], v[5], v[7]};
        }
    }

    f4_t O[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) O[t] = f4_t{};
    float R = -INFINITY, l = 0.0f;
    const float c2 = a.c2;
    bool big = false;

    // the tiles of this wavefront: first + wave, + NW, ..; their page entries lie in the lanes, 64 at a time
    const int n = first + wave < last ? (last - first - wave + NW - 1) / NW : 0;
    const int32_t * pages = a.p.pages + s * a.p.ld;
    int ent = 0;
    const auto entries = [&](int k) {
        const int t = first + wave + NW * (k + lane);
        ent = k + lane < n ? pages[t >> (a.p.shift - 5)] : -1;
    };
    const auto tile_base = [&](int k) -> const uint8_t * {
        const int e = __builtin_amdgcn_readlane(ent, k & 63);
        if ((unsigned) e >= (unsigned) a.p.n_pages) return nullptr;
        const int t = first + wave + NW * k;
        return a.p.data + ((((int64_t) e * a.p.Hkv + hk) << (a.p.shift - 5)) + (t & ((1 << (a.p.shift - 5)) - 1))) * (36 * D);
    };
    TileRegs<D> r;
    // lane lr = 4 g' + i loads the keys 8 g' + order(4 T + i), T = 0, 1
    const int kkey = 8 * (lr >> 2) + paged_order(lr & 3);
    const auto load_k = [&](const uint8_t * t) {
#pragma unroll
        for (int T = 0; T < 2; T++) {
            const uint8_t * p = t + (kkey + 4 * T) * (D / 2) + g * (D / 8);
#pragma unroll
            for (int b = 0; b < D / 64; b++) r.kc[T][b] = reinterpret_cast<const u2_t *>(p)[b];
        }
#pragma unroll
        for (int b = 0; b < NB; b++) r.kd[b] = *reinterpret_cast<const h8_t *>(t + 32 * D + 64 * b + 16 * g);
    };
    const auto load_v = [&](const uint8_t * t) {
#pragma unroll
        for (int b = 0; b < D / 64; b++) r.vc[b] = *reinterpret_cast<const u4_t *>(t + 16 * D + 1024 * b + 16 * lane);
#pragma unroll
        for (int b = 0; b < NB; b++) r.vd[b] = *reinterpret_cast<const h8_t *>(t + 34 * D + 64 * b + 16 * g);
    };
    if (n) entries(0);
    // k: the tile at hand, kn: the next that is there
    const auto next = [&](int k, const uint8_t *& t) {
        for (; k < n; k++) {
            if ((k & 63) == 0 && k) entries(k);
            if (const uint8_t * c = tile_base(k)) {
                t = c;
                break;
            }
        }
        return k;
    };
    const uint8_t * t = nullptr;
    int k = next(0, t);
    if (k < n) {
        load_k(t);
        load_v(t);
    }
    while (k < n) {
        const int64_t key0 = 32 * (int64_t) (first + wave + NW * k);
        const uint8_t * tn = t;
        const int kn = next(k + 1, tn);

        float S[2][4] = {};
#pragma unroll
        for (int T = 0; T < 2; T++)
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const u2_t w = r.kc[T][b % (D / 64)];
                f4_t A = {};
                A = __builtin_amdgcn_mfma_f32_16x16x32_f16(b < D / 64 ? code_frag<0>(w) : code_frag<1>(w), qf[b], A, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) S[T][i] = fmaf((float) r.kd[b][4 * T + i], A[i], S[T][i]);
            }
        load_k(tn);

        // keys this lane's row does not see
        const bool edge = key0 + 31 > pos0 || (a.window && key0 <= pos1 - a.window) || key0 + 32 > cap;
        uint32_t hide = 0;
        if (edge) {
            const int64_t end = min(pos + 1, cap) - key0 - 8 * g, low = a.window ? pos - a.window + 1 - key0 - 8 * g : 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = (e & 4) | (e & 1) << 1 | (e >> 1 & 1);  // order(e)
                const bool gone = key >= end || key < low;
                S[e >> 2][e & 3] = gone ? -INFINITY : S[e >> 2][e & 3];
                hide |= (uint32_t) gone << e;
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])), fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])));
        mx *= c2;
        if (__any(mx > R + kSlack || R == -INFINITY)) {
            const float top = xor16_max(mx), Rn = top > R + kSlack ? ceilf(top) : R;  // (a row's R goes by its own scores)
            const float al = R == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(R - Rn);
            R = Rn;
            l *= al;
#pragma unroll
            for (int i = 0; i < NT; i++) O[i] *= al;
            big = __any(fabsf(R) >= kBig && R != -INFINITY);
        }
        const float rb = R == -INFINITY ? 0.0f : R;
        float c = c2;
        if (big) {  // a row's R is its largest exponent rounded: round all alike
            const bool mine = fabsf(rb) >= kBig;
#pragma unroll
            for (int e = 0; e < 8; e++) S[e >> 2][e & 3] *= mine ? c2 : 1.0f;
            c = mine ? 1.0f : c2;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) S[e >> 2][e & 3] = __builtin_amdgcn_exp2f(fmaf(S[e >> 2][e & 3], c, -rb)) * kP;
        if (edge)
#pragma unroll
            for (int e = 0; e < 8; e++) S[e >> 2][e & 3] = hide >> e & 1 ? 0.0f : S[e >> 2][e & 3];
        h8_t ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float p0 = S[e >> 2][e & 3], p1 = S[e >> 2][(e & 3) + 1];
            const h2_t w = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
            const h2_t u = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float) w.x, -1.0f, p0), fmaf((float) w.y, -1.0f, p1)));
            ph[e] = w.x, ph[e + 1] = w.y, pl[e] = u.x, pl[e + 1] = u.y;
        }
        {
            h8_t one;
#pragma unroll
            for (int e = 0; e < 8; e++) one[e] = (_Float16) 1.0f;
            f4_t z = {};
            z = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, pl, z, 0, 0, 0);
            z = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, ph, z, 0, 0, 0);
            l += z[0];
        }
        // Keys that no row sees may hold anything, a NaN for a scale too: theirs are taken as 0.
        if (edge) {
            const int64_t end = min(pos1 + 1, cap) - key0 - 8 * g, low = a.window ? pos0 - a.window + 1 - key0 - 8 * g : 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = (e & 4) | (e & 1) << 1 | (e >> 1 & 1);
#pragma unroll
                for (int b = 0; b < NB; b++)
                    if (key >= end || key < low) r.vd[b][e] = (_Float16) 0.0f;
            }
        }
#pragma unroll
        for (int b = 0; b < D / 64; b++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int H = 0; H < 2; H++) {
                    const int td = 2 * b + u + H * (D / 32);  // dims 16 td ..
                    h2_t cv[4];
                    if (H) code_values<1>(r.vc[b][2 * u], r.vc[b][2 * u + 1], cv);
                    else code_values<0>(r.vc[b][2 * u], r.vc[b][2 * u + 1], cv);
                    h8_t vh, vl;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const h2_t d = {r.vd[td / 2][2 * i], r.vd[td / 2][2 * i + 1]};
                        const h2_t hi = cv[i] * d, lo = __builtin_elementwise_fma(cv[i], d, -hi);
                        vh[2 * i] = hi.x, vh[2 * i + 1] = hi.y, vl[2 * i] = lo.x, vl[2 * i + 1] = lo.y;
                    }
                    f4_t z = {};
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph, z, 0, 0, 0);
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl, z, 0, 0, 0);
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph, z, 0, 0, 0);
                    O[td] += z;
                }
        load_v(tn);
        t = tn;
        k = kn;
    }

    // the wavefronts' sums: the upper half hands its to the lower, until one is left
    __shared__ f4_t ex[NW / 2][NT][64];
    __shared__ float2 exml[NW / 2][64];
#pragma unroll
    for (int half = NW / 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int i = 0; i < NT; i++) ex[wave - half][i][lane] = O[i];
            exml[wave - half][lane] = make_float2(R, l);
        }
        __syncthreads();
        if (wave < half) {
            const float2 ml = exml[wave][lane];
            const float Rn = fmaxf(R, ml.x);
            const float a0 = R == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(R - Rn);
            const float a1 = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - Rn);
            R = Rn;
            l = l * a0 + ml.y * a1;
#pragma unroll
            for (int i = 0; i < NT; i++) O[i] = O[i] * a0 + ex[wave][i][lane] * a1;
        }
        __syncthreads();
    }
    if (wave || x >= rows) return;
    if (ns == 1) {
        float * o = a.out + ((int64_t) (sw.r0 + j) * a.H + h) * D + 4 * g;
        const float inv = 1.0f / l;
#pragma unroll
        for (int i = 0; i < NT; i++) *reinterpret_cast<f4_t *>(o + 16 * i) = l == 0.0f ? f4_t{} : O[i] * inv;
        return;
    }
    float * o = a.part_o + ((int64_t) blockIdx.x * ROWS + lr) * D + 4 * g;
#pragma unroll
    for (int i = 0; i < NT; i++) *reinterpret_cast<f4_t *>(o + 16 * i) = O[i];
    if (g == 0) a.part_ml[(int64_t) blockIdx.x * ROWS + lr] = make_float2(R, l);
}

// One (row, head): its splits' sums, weighted by 2^(R - the largest R).
template <int D, int ROWS>
__global__ __launch_bounds__(256) void k_paged_merge(const AttnArgs a) {
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int s = paged_seq(a.p, row);
    if (s < 0) return;
    const int chunk = plan_chunk<ROWS>(a);
    const SeqWork sw = seq_work<ROWS>(a, s);
    const int ns = splits(sw.tiles, chunk), j = row - sw.r0;
    if (ns == 1 || j >= sw.rows) return;
    // the first item of sequence s
    int base = 0;
    for (int s0 = 0; s0 < s; s0 += 64) {
        const SeqWork w = seq_work<ROWS>(a, s0 + lane < s ? s0 + lane : a.p.n_seq);
        base += wave_isum(w.rts * a.p.Hkv * splits(w.tiles, chunk));
    }
    const int x = j * a.G + h % a.G;
    const int64_t item = base + ((int64_t) (h / a.G) * sw.rts + x / ROWS) * ns;
    if (item < 0 || item + ns > a.items) return;  // (starts that do not ascend)
    const float2 * ml = a.part_ml + item * ROWS + x % ROWS;
    const float * o = a.part_o + (item * ROWS + x % ROWS) * D;
    float R = -INFINITY;
    for (int i = lane; i < ns; i += 64) R = fmaxf(R, ml[(int64_t) i * ROWS].x);
    R = wave_max(R);
    constexpr int NP = 256 / (D / 4);  // splits at a time, a thread taking four dims
    const int d4 = tid % (D / 4), part = tid / (D / 4);
    f4_t acc = {};
    float l = 0.0f;
#pragma unroll 4
    for (int i = part; i < ns; i += NP) {
        const float2 m = ml[(int64_t) i * ROWS];
        const float w = m.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m.x - R);
        l = fmaf(m.y, w, l);
        acc += *reinterpret_cast<const f4_t *>(o + (int64_t) i * ROWS * D + 4 * d4) * w;
    }
    __shared__ f4_t so[NP][D / 4];
    __shared__ float sl[NP];
    so[part][d4] = acc;
    if (d4 == 0) sl[part] = l;
    __syncthreads();
    if (part) return;
    for (int i = 1; i < NP; i++) {
        acc += so[i][d4];
        l += sl[i];
    }
    const float inv = 1.0f / l;
    *reinterpret_cast<f4_t *>(a.out + ((int64_t) row * a.H + h) * D + 4 * d4) = l == 0.0f ? f4_t{} : acc * inv;
}

// Workgroups that may have work: the splits (kTarget of them, one more for each row tile and KV head), or every row
// tile's longest possible number of splits.
struct Grid {
    int64_t items;
    int most;  // splits of a sequence
};
Grid grid_for(const Paged & p, int G, int64_t max_rows, int ROWS) {
    const int64_t rts = p.Hkv * std::min<int64_t>((int64_t) p.n_rows * G / ROWS + std::min<int64_t>(p.n_seq, p.n_rows),
                                                  p.n_seq * ((std::min<int64_t>(max_rows, p.n_rows) * G + ROWS - 1) / ROWS));
    const int64_t most = (((int64_t) p.max_pages << p.shift) / kPagedTile + kMinChunk - 1) / kMinChunk;
    return {std::min(rts + kTarget, rts * most), (int) std::min<int64_t>(most, INT32_MAX)};
}

template <int D>
void run(const AttnArgs & a, int64_t items, bool merge, hipStream_t s) {
    constexpr int NW = D == 256 ? 4 : 8;
    k_paged_few<D, NW><<<(unsigned) items, 64 * NW, 0, s>>>(a);
    check_launch("paged attn");
    if (merge) k_paged_merge<D, 16><<<dim3((unsigned) a.p.n_rows, (unsigned) a.H), 256, 0, s>>>(a);
    check_launch("paged attn merge");
}

}  // namespace

size_t paged_attn_workspace(const Paged & p, int D, int H, int64_t max_rows) {
    if (p.n_rows == 0) return 0;
    const Grid g = grid_for(p, H / p.Hkv, max_rows, 16);
    if (g.most == 1) return 0;
    return (size_t) g.items * 16 * (D * sizeof(float) + sizeof(float2));
}

void launch_paged_attn(const Paged & p, int D, const void * q, int64_t q_r, int64_t q_h, int H, int64_t max_rows, int window,
                       float scale, float * out, void * ws, hipStream_t s) {
    AttnArgs a{};
    a.p = p, a.q = (const _Float16 *) q, a.q_r = q_r, a.q_h = q_h, a.H = H, a.G = H / p.Hkv, a.window = window;
    a.max_rows = (int) std::min<int64_t>(max_rows, p.n_rows);
    // (from 0 up to 2^-100: scores of 0 either way, but -inf for a hidden key)
    a.c2 = (float) (std::max(fabs((double) scale), 0x1p-100) * 1.4426950408889634074);
    a.negate = scale < 0.0f;
    a.out = out;
    const Grid g = grid_for(p, a.G, max_rows, 16);
    require(g.items < INT32_MAX, "paged_attn: too many rows and heads");
    a.items = (int) g.items;
    a.part_o = (float *) ws;
    a.part_ml = (float2 *) ((char *) ws + (size_t) g.items * 16 * D * sizeof(float));
    if (D == 64) run<64>(a, g.items, g.most > 1, s);
    else if (D == 128) run<128>(a, g.items, g.most > 1, s);
    else run<256>(a, g.items, g.most > 1, s);
}

}  // namespace gcq

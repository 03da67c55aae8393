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
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr int kMinChunk = 16;    // tiles: a shorter split costs more in the merge than it saves
constexpr float kSlack = 4.0f;   // how far a score's exponent may pass R
constexpr float kBig = 0x1p20f;  // exponents from here on are no longer exact to 2^-4
constexpr float kP = 2048.0f;    // P's scale: 2^11 2^kSlack is f16's 2^15

struct AttnArgs {
    Paged p;
    const _Float16 * q;
    int64_t q_r, q_h;
    int H, G, window, max_rows, items, target;  // target: workgroups that the splits aim at
    float c2;     // |scale| log2(e)
    bool negate;  // the scale is negative
    float * out, * part_o;
    float2 * part_ml;
};

// A sequence's rows, and the tiles of the keys that any of them sees.
struct SeqWork {
    int r0, rows, tile0, tiles, rts, past;
};
template <int ROWS>
__device__ __forceinline__ SeqWork seq_work(const AttnArgs & a, int s) {
    SeqWork w{};
    if (s >= a.p.n_seq) return w;
    w.r0 = a.p.starts[s];
    const int r1 = min(a.p.starts[s + 1], a.p.n_rows);
    w.past = a.p.past[s];
    if (w.r0 < 0 || r1 <= w.r0) return w;
    w.rows = min(r1 - w.r0, a.max_rows);
    const int64_t hi = min((int64_t) w.past + w.rows, (int64_t) a.p.max_pages << a.p.shift);
    const int64_t lo = a.window && (int64_t) w.past - a.window + 1 > 0 ? (int64_t) w.past - a.window + 1 : 0;
    w.tile0 = (int) (lo >> 5);
    w.tiles = hi > lo ? (int) ((hi + 31) >> 5) - w.tile0 : 0;
    w.rts = (int) (((int64_t) w.rows * a.G + ROWS - 1) / ROWS);
    return w;
}
__device__ __forceinline__ int splits(int tiles, int chunk) { return max(1, (tiles + chunk - 1) / chunk); }

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

// The plan, the same in every wavefront: tiles per split, and a sequence's first item. Items of a sequence: [KV
// head][row tile][split]. The batch's arrays are read once where the sequences fit the lanes.
template <int ROWS>
struct Plan {
    const AttnArgs & a;
    SeqWork w;  // of sequence s0 + lane
    int chunk, s, base, lane_at;

    __device__ __forceinline__ Plan(const AttnArgs & args) : a(args) {
        const int lane = threadIdx.x & 63;
        w = seq_work<ROWS>(a, lane);
        double u = (double) w.rts * w.tiles, n = w.rts;
        for (int s0 = 64; s0 < a.p.n_seq; s0 += 64) {
            const SeqWork x = seq_work<ROWS>(a, s0 + lane);
            u += (double) x.rts * x.tiles;
            n += x.rts;
        }
        u = wave_sum_d(u) * a.p.Hkv;
        n = wave_sum_d(n) * a.p.Hkv;
        const double cut = fmax(a.target - n, 0.5 * a.target);
        chunk = __builtin_amdgcn_readfirstlane((int) fmax((double) kMinChunk, fmin(u / cut + 1.0, 1e9)));
    }
    __device__ __forceinline__ int items(const SeqWork & x) const { return x.rts * a.p.Hkv * splits(x.tiles, chunk); }

    // The sequence found, uniform.
    __device__ __forceinline__ SeqWork picked() {
        const int l = __builtin_amdgcn_readfirstlane(lane_at);
        const auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
        base = __builtin_amdgcn_readfirstlane(base);
        s = __builtin_amdgcn_readfirstlane(s);
        return {pick(w.r0), pick(w.rows), pick(w.tile0), pick(w.tiles), pick(w.rts), pick(w.past)};
    }
    // To the sequence that `found` (a ballot over the sequences s0 .. s0 + 63, their inclusive item sums given) picks
    // first.
    template <class F>
    __device__ __forceinline__ bool find(F && found) {
        const int lane = threadIdx.x & 63;
        base = 0;
        for (int s0 = 0; s0 < a.p.n_seq; s0 += 64) {
            if (s0) w = seq_work<ROWS>(a, s0 + lane);
            const int n = items(w), sum = wave_scan(n);
            const uint64_t at = found(s0 + lane, base + sum);
            if (at) {
                lane_at = __builtin_ctzll(at);
                base += __builtin_amdgcn_readlane(sum - n, lane_at);
                s = s0 + lane_at;
                return true;
            }
            base += __builtin_amdgcn_readlane(sum, 63);
        }
        return false;
    }
};

__device__ __forceinline__ float xor16_max(float v) {
    v = row_pair<16>(v, fmaxf_op);
    return row_pair<32>(v, fmaxf_op);
}

// 8 codes of low (H = 0) or high nibbles as values c - 8, in pairs of f16. (As they lie, masked out as f16 subnormals, they
// cost half the operations, but an MFMA aligns a subnormal's product by its exponent field: 6 to 10 bits of the sum go.)
template <int H>
__device__ __forceinline__ void code_values(uint32_t w0, uint32_t w1, h2_t (&c)[4]) {
    uint32_t m = H ? 0x00f000f0u : 0x000f000fu;
    asm("" : "+v"(m));  // in a register: v_and_or_b32 takes no literal
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

// A tile from memory into LDS, without registers in between: 1 KiB per instruction, 16 bytes per lane, the last one partly.
// (As inline code, m0 set and used in one piece, since the compiler has a builtin's loads waited for, all of them, before any LDS read.)
template <int D> constexpr int kTileLoads = (36 * D + 1023) / 1024;
template <int OFF>
__device__ __forceinline__ void lds_load(const uint8_t * base, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%3" ::"v"(voff), "s"(base), "s"(lds), "n"(OFF) : "memory");
}
template <int D>
__device__ __forceinline__ void tile_load(const uint8_t * data, int64_t off, uint32_t lds, int lane) {
    const uint64_t p = (uint64_t) (uintptr_t) (data + off);
    const uint8_t * t = (const uint8_t *) (uintptr_t) ((uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (p >> 32)) << 32 |
                                                       (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) p));
    lds = __builtin_amdgcn_readfirstlane(lds);
    constexpr int full = 36 * D / 1024, rest = (36 * D % 1024) / 16;
#pragma unroll
    for (int i = 0; i < full; i += 3) {
        const uint32_t v = 16 * lane + 1024 * i;
        lds_load<0>(t, v, lds + 1024 * i);
        if (i + 1 < full) lds_load<1024>(t, v, lds + 1024 * i);
        if (i + 2 < full) lds_load<2048>(t, v, lds + 1024 * i);
    }
    if (rest && lane < rest) lds_load<0>(t, 16 * lane + 1024 * full, lds + 1024 * full);
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <int D> constexpr int kRing = D == 64 ? 4 : 2;       // tiles in LDS per wavefront
template <int D> constexpr int kPerSimd = D == 256 ? 2 : 4;   // wavefronts per SIMD

template <int D, int NW>
__global__ __launch_bounds__(64 * NW, kPerSimd<D>) void k_paged_few(const AttnArgs a) {
    constexpr int ROWS = 16, NB = D / 32, NT = D / 16, RING = kRing<D>, NL = kTileLoads<D>, P = D + 4;
    constexpr int kShared = NW * RING * 36 * D > NW * ROWS * P * 4 ? NW * RING * 36 * D : NW * ROWS * P * 4;
    __shared__ __align__(16) uint8_t shared[kShared];
    __shared__ float2 exml[NW][ROWS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
    Plan<ROWS> plan(a);
    if (!plan.find([&](int, int sum) { return __ballot(sum > (int) blockIdx.x); })) return;
    const SeqWork sw = plan.picked();
    const int ns = splits(sw.tiles, plan.chunk), id = blockIdx.x - plan.base;
    const int split = id % ns, rt = id / ns % sw.rts, hk = id / ns / sw.rts;

    const int rows = sw.rows * a.G, x0 = rt * ROWS, nr = min(ROWS, rows - x0);  // this tile's rows
    const int x = x0 + min(lr, nr - 1), j = x / a.G, h = hk * a.G + x % a.G;       // this lane's (the last for those past it)
    const int64_t pos = (int64_t) sw.past + j, pos0 = (int64_t) sw.past + x0 / a.G, pos1 = (int64_t) sw.past + (x0 + nr - 1) / a.G;
    // this row tile's keys within the split; tiles below e0 or from e1 on are not seen whole by every row
    const int64_t cap = (int64_t) a.p.max_pages << a.p.shift;
    const int first = max(sw.tile0 + split * plan.chunk, a.window && pos0 - a.window + 1 > 0 ? (int) ((pos0 - a.window + 1) >> 5) : 0);
    const int last = min(sw.tile0 + min(sw.tiles, (split + 1) * plan.chunk), (int) ((min(pos1 + 1, cap) + 31) >> 5));
    const int e0 = a.window ? (int) ((pos1 - a.window) >> 5) + 1 : 0, e1 = (int) ((pos0 + 1) >> 5);

    // the tiles of this wavefront: first + wave, + NW, ..; their page entries lie in the lanes, 64 at a time
    const int n = first + wave < last ? (last - first - wave + NW - 1) / NW : 0;
    const int32_t * pages = a.p.pages + plan.s * a.p.ld;
    const int sub = a.p.shift - 5;
    int ent = -1;
    const auto entries = [&](int k) { ent = k + lane < n ? pages[(first + wave + NW * (k + lane)) >> sub] : -1; };
    if (n) entries(0);

    // Q: this lane's row, dims 32 b + 8 g + order(0 .. 7)
    h8_t qf[NB];
    {
        const _Float16 * qp = a.q + (int64_t) (sw.r0 + j) * a.q_r + (int64_t) h * a.q_h + 8 * g;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            h8_t v = *reinterpret_cast<const h8_t *>(qp + 32 * b);
            if (lr >= nr) v = h8_t{};
            if (a.negate) v = -v;
            qf[b] = h8_t{v[0], v[2], v[1], v[3], v[4], v[6], v[5], v[7]};
        }
    }

    uint8_t * const ring = shared + wave * (RING * 36 * D);
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane((uint32_t) (uintptr_t) (__attribute__((address_space(3))) uint8_t *) ring);
    int at = 0, issued = 0, tile_of = 0;  // next of this wavefront's tiles, tiles under way or done, the ring's tiles (by lane)
    const auto issue = [&] {
        for (; at < n; at++) {
            if ((at & 63) == 0 && at) entries(at);
            const int e = __builtin_amdgcn_readlane(ent, at & 63), t = first + wave + NW * at;
            if ((unsigned) e >= (unsigned) a.p.n_pages) continue;  // a page that is not there
            const int slot = issued % RING;
            tile_of = lane == slot ? t : tile_of;
            tile_load<D>(a.p.data, ((((int64_t) e * a.p.Hkv + hk) << sub) + (t & ((1 << sub) - 1))) * (36 * D), ring_at + slot * (36 * D), lane);
            issued++;
            at++;
            return;
        }
    };
#pragma unroll
    for (int i = 0; i < RING; i++) issue();

    f4_t O[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) O[t] = f4_t{};
    float R = -INFINITY, l = 0.0f;
    const float c2 = a.c2;
    bool big = false;
    // lane lr = 4 g' + i takes the keys 8 g' + order(4 T + i), T = 0, 1, as its MFMA row
    const uint32_t ko = (8 * (lr >> 2) + paged_order(lr & 3)) * (D / 2) + g * (D / 8), vo = 16 * D + 16 * lane, so = 32 * D + 16 * g;

    for (int done = 0; done < issued; done++) {
        if (issued - done == RING) wait_loads<(RING - 1) * NL>();
        else wait_loads<0>();
        const int slot = done % RING, tile = __builtin_amdgcn_readlane(tile_of, slot);
        uint8_t * const t = ring + slot * (36 * D);

        float S[2][4] = {};
#pragma unroll
        for (int T = 0; T < 2; T++) {
            u2_t kc[D / 64];
            if constexpr (D == 64) kc[0] = *reinterpret_cast<const u2_t *>(t + ko + T * (2 * D));
            else
#pragma unroll
                for (int b = 0; b < D / 64; b += 2) {
                    const u4_t w = *reinterpret_cast<const u4_t *>(t + ko + (T * (2 * D) + 8 * b));
                    kc[b] = u2_t{w.x, w.y};
                    kc[b + 1] = u2_t{w.z, w.w};
                }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                f4_t A = {};
                A = __builtin_amdgcn_mfma_f32_16x16x32_f16(b < D / 64 ? code_frag<0>(kc[b % (D / 64)]) : code_frag<1>(kc[b % (D / 64)]), qf[b], A, 0, 0, 0);
                const h4_t d = *reinterpret_cast<const h4_t *>(t + so + (64 * b + 8 * T));
#pragma unroll
                for (int i = 0; i < 4; i++) S[T][i] = fmaf((float) d[i], A[i], S[T][i]);
            }
        }

        // keys this lane's row does not see
        const bool edge = tile < e0 || tile >= e1;
        if (edge) {
            const int64_t k0 = 32 * (int64_t) tile + 8 * g;
            const int end = (int) (min(pos + 1, cap) - k0), low = a.window ? (int) max(pos - a.window + 1 - k0, (int64_t) 0) : 0;
            const int end1 = (int) (min(pos1 + 1, cap) - k0), low0 = a.window ? (int) max(pos0 - a.window + 1 - k0, (int64_t) 0) : 0;
            // A key that no row sees may hold anything, a NaN for a scale too: its values' scales are set to 0.
            h8_t * const vd = reinterpret_cast<h8_t *>(t + so + (2 * D + 64 * lr));
            h8_t z = lr < NB ? *vd : h8_t{};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = (e & 4) | (e & 1) << 1 | (e >> 1 & 1);  // order(e)
                S[e >> 2][e & 3] = key >= end || key < low ? -INFINITY : S[e >> 2][e & 3];
                z[e] = key >= end1 || key < low0 ? (_Float16) 0.0f : z[e];
            }
            if (lr < NB) *vd = z;
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
#pragma unroll
        for (int b = 0; b < D / 64; b++) {
            const u4_t vc = *reinterpret_cast<const u4_t *>(t + vo + 1024 * b);
#pragma unroll
            for (int H = 0; H < 2; H++) {
                const h8_t vd = *reinterpret_cast<const h8_t *>(t + so + (2 * D + 64 * (b + H * (D / 64))));
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int td = 2 * b + u + H * (D / 32);  // dims 16 td ..
                    h2_t cv[4];
                    if (H) code_values<1>(vc[2 * u], vc[2 * u + 1], cv);
                    else code_values<0>(vc[2 * u], vc[2 * u + 1], cv);
                    h8_t vh, vl;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const h2_t d = {vd[2 * i], vd[2 * i + 1]};
                        const h2_t hi = cv[i] * d, lo = __builtin_elementwise_fma(cv[i], d, -hi);
                        vh[2 * i] = hi.x, vh[2 * i + 1] = hi.y, vl[2 * i] = lo.x, vl[2 * i + 1] = lo.y;
                    }
                    f4_t z = {};
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph, z, 0, 0, 0);
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl, z, 0, 0, 0);
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph, z, 0, 0, 0);
                    O[td] += z;
                }
            }
        }
        wait_lds();  // the slot is read before the next tile is sent into it
        issue();
    }
    __syncthreads();

    // the wavefronts' sums, brought to one R and added
    float (*ex)[ROWS][P] = reinterpret_cast<float (*)[ROWS][P]>(shared);
    if (g == 0) exml[wave][lr] = make_float2(R, l);
    __syncthreads();
    float Rm = exml[0][lr].x;
#pragma unroll
    for (int w = 1; w < NW; w++) Rm = fmaxf(Rm, exml[w][lr].x);
    const float f = R == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(R - Rm);
    if (lr < nr)
#pragma unroll
        for (int i = 0; i < NT; i++) *reinterpret_cast<f4_t *>(&ex[wave][lr][16 * i + 4 * g]) = O[i] * f;
    __syncthreads();
    for (int e = threadIdx.x; e < nr * (D / 4); e += 64 * NW) {
        const int y = e / (D / 4), d = 4 * (e % (D / 4));
        float2 ml[NW];
        float m = -INFINITY, sum = 0.0f;
        f4_t o = {};
#pragma unroll
        for (int w = 0; w < NW; w++) ml[w] = exml[w][y], m = fmaxf(m, ml[w].x);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            sum += ml[w].x == -INFINITY ? ml[w].y * 0.0f : ml[w].y * __builtin_amdgcn_exp2f(ml[w].x - m);
            o += *reinterpret_cast<const f4_t *>(&ex[w][y][d]);
        }
        if (ns == 1) {
            const int xx = x0 + y;
            const float inv = 1.0f / sum;
            *reinterpret_cast<f4_t *>(a.out + ((int64_t) (sw.r0 + xx / a.G) * a.H + hk * a.G + xx % a.G) * D + d) =
                sum == 0.0f ? f4_t{} : o * inv;
        } else {
            *reinterpret_cast<f4_t *>(a.part_o + ((int64_t) blockIdx.x * ROWS + y) * D + d) = o;
            if (d == 0) a.part_ml[(int64_t) blockIdx.x * ROWS + y] = make_float2(m, sum);
        }
    }
}

// One (row, head): its splits' sums, weighted by 2^(R - the largest R).
template <int D, int ROWS>
__global__ __launch_bounds__(256) void k_paged_merge(const AttnArgs a) {
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    Plan<ROWS> plan(a);
    if (!plan.find([&](int s, int) { return __ballot(s < a.p.n_seq && plan.w.r0 <= row && row < plan.w.r0 + plan.w.rows); })) return;
    const SeqWork sw = plan.picked();
    const int ns = splits(sw.tiles, plan.chunk), j = row - sw.r0;
    if (ns == 1) return;
    const int x = j * a.G + h % a.G;
    const int64_t item = plan.base + ((int64_t) (h / a.G) * sw.rts + x / ROWS) * ns;
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
        l += m.y * w;
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

constexpr int kWaves = 4;
// Workgroups resident at once: what the splits aim at.
int target(int D) { return 256 * (D == 256 ? kPerSimd<256> : kPerSimd<64>) * 4 / kWaves; }

// Workgroups that may have work: the splits (`target` of them, one more for each row tile and KV head), or every row
// tile's longest possible number of splits.
struct Grid {
    int64_t items;
    int64_t most;  // splits of a sequence
};
Grid grid_for(const Paged & p, int D, int G, int64_t max_rows, int ROWS) {
    const int64_t rts = p.Hkv * std::min<int64_t>((int64_t) p.n_rows * G / ROWS + std::min<int64_t>(p.n_seq, p.n_rows),
                                                  p.n_seq * ((std::min<int64_t>(max_rows, p.n_rows) * G + ROWS - 1) / ROWS));
    const int64_t most = (((int64_t) p.max_pages << p.shift) / kPagedTile + kMinChunk - 1) / kMinChunk;
    return {std::min(rts + target(D), rts * most), most};
}

template <int D>
void run(const AttnArgs & a, bool merge, hipStream_t s) {
    k_paged_few<D, kWaves><<<(unsigned) a.items, 64 * kWaves, 0, s>>>(a);
    check_launch("paged attn");
    if (merge) k_paged_merge<D, 16><<<dim3((unsigned) a.p.n_rows, (unsigned) a.H), 256, 0, s>>>(a);
    check_launch("paged attn merge");
}

}  // namespace

size_t paged_attn_workspace(const Paged & p, int D, int H, int64_t max_rows) {
    if (p.n_rows == 0) return 0;
    const Grid g = grid_for(p, D, H / p.Hkv, max_rows, 16);
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
    const Grid g = grid_for(p, D, a.G, max_rows, 16);
    require(g.items < INT32_MAX, "paged_attn: too many rows and heads");
    a.items = (int) g.items, a.target = target(D);
    a.part_o = (float *) ws;
    a.part_ml = (float2 *) ((char *) ws + (size_t) g.items * 16 * D * sizeof(float));
    if (D == 64) run<64>(a, g.most > 1, s);
    else if (D == 128) run<128>(a, g.most > 1, s);
    else run<256>(a, g.most > 1, s);
}

}  // namespace gcq

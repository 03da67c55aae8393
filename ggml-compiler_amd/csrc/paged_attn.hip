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
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kMinChunk = 16;    // tiles: a shorter split costs more in the merge than it saves
constexpr float kSlack = 4.0f;   // how far a score's exponent may pass R
constexpr float kBig = 0x1p20f;  // exponents from here on are no longer exact to 2^-4
constexpr float kP = 4.0f;       // the exponent of P's scale: with kSlack at most 2^8; parts down to 2^-28 of 2^R

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
// head][row tile, the last, which sees most, first][split]. The batch's arrays are read once where the sequences fit the lanes.
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

// v as an f32, whatever it is an operand of.
__device__ __forceinline__ float rounded(float v) {
    asm("" : "+v"(v));
    return v;
}
__device__ __forceinline__ float xor16_max(float v) {
    v = row_pair<16>(v, fmaxf_op);
    return row_pair<32>(v, fmaxf_op);
}

// The largest of 8, NaNs passed over, as medians with infinity: fmaxf quiets its operands first, twice the operations.
__device__ __forceinline__ float max8(const float (&x)[8]) {
    const auto m = [](float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); };
    return m(m(m(x[0], x[1]), m(x[2], x[3])), m(m(x[4], x[5]), m(x[6], x[7])));
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

template <int D> constexpr int kRing = D == 64 ? 4 : 2;  // tiles in LDS per wavefront
// Wavefronts per SIMD that the registers hold.
template <int D, int RT> constexpr int kPerSimd = D * RT <= 128 ? 4 : D * RT <= 256 ? 2 : 1;

template <int D, int RT, int NW>
__global__ __launch_bounds__(64 * NW, (kPerSimd<D, RT>)) void k_paged_few(const AttnArgs a) {
    constexpr int ROWS = 16 * RT, NB = D / 32, NT = D / 16, RING = kRing<D>, NL = kTileLoads<D>, P = D + 4;
    // LDS: the wavefronts' rings (then their sums of 16 rows), and the row tile's Q as MFMA operands (from two times 16
    // rows on; registers hold 16)
    constexpr int kRings = NW * RING * 36 * D, kSums = NW * 16 * (P * 4 + 8), kQ = RT > 1 ? ROWS * D * 2 : 0;
    __shared__ __align__(16) uint8_t shared[(kRings > kSums ? kRings : kSums) + kQ];
    h8_t * const sq = reinterpret_cast<h8_t *>(shared + (kRings > kSums ? kRings : kSums));  // [16 rows][block][lane]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
    Plan<ROWS> plan(a);
    if (!plan.find([&](int, int sum) { return __ballot(sum > (int) blockIdx.x); })) return;
    const SeqWork sw = plan.picked();
    const int ns = splits(sw.tiles, plan.chunk), id = blockIdx.x - plan.base;
    const int split = id % ns, rt = sw.rts - 1 - id / ns % sw.rts, hk = id / ns / sw.rts;

    const int rows = sw.rows * a.G, x0 = rt * ROWS, nr = min(ROWS, rows - x0);  // this tile's rows
    const int64_t pos0 = (int64_t) sw.past + x0 / a.G, pos1 = (int64_t) sw.past + (x0 + nr - 1) / a.G;
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

    // Q: of a lane's row, dims 32 b + 8 g + order(0 .. 7)
    const auto load_q = [&](int i, int b) {
        const int y = 16 * i + lr, x = x0 + min(y, nr - 1);
        h8_t v = *reinterpret_cast<const h8_t *>(a.q + (int64_t) (sw.r0 + x / a.G) * a.q_r + (int64_t) (hk * a.G + x % a.G) * a.q_h + 32 * b + 8 * g);
        if (y >= nr) v = h8_t{};
        if (a.negate) v = -v;
        return h8_t{v[0], v[2], v[1], v[3], v[4], v[6], v[5], v[7]};
    };
    h8_t qf[RT > 1 ? 1 : NB];
    if constexpr (RT == 1) {
#pragma unroll
        for (int b = 0; b < NB; b++) qf[b] = load_q(0, b);
    } else {
        for (int b = wave; b < NB * RT; b += NW) sq[b * 64 + lane] = load_q(b / NB, b % NB);
        __syncthreads();
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

    // the work on RA times 16 rows
    const auto body = [&](auto ra) {
        constexpr int RA = decltype(ra)::value;
        f4_t O[RA][NT];
        float R[RA], l[RA], top[RA], shift[RA];  // the reference exponent; R + kSlack; kP - R
#pragma unroll
        for (int i = 0; i < RA; i++) {
            R[i] = top[i] = -INFINITY;
            l[i] = 0.0f;
            shift[i] = kP;
#pragma unroll
            for (int t = 0; t < NT; t++) O[i][t] = f4_t{};
        }
        const float c2 = a.c2;
        bool big = false;
        const auto barrier = [] {  // (the order as written: the scheduler's holds more than the registers do)
            if constexpr (RA > 1) __builtin_amdgcn_sched_barrier(0);
        };
        // lane lr = 4 g' + i takes the keys 8 g' + order(4 T + i), T = 0, 1, as its MFMA row
        const uint32_t ko = (8 * (lr >> 2) + paged_order(lr & 3)) * (D / 2) + g * (D / 8), vo = 16 * D + 16 * lane, so = 32 * D + 16 * g;

        for (int done = 0; done < issued; done++) {
            if (issued - done == RING) wait_loads<(RING - 1) * NL>();
            else wait_loads<0>();
            const int slot = done % RING, tile = __builtin_amdgcn_readlane(tile_of, slot);
            uint8_t * const t = ring + slot * (36 * D);

            // scores: a block's MFMAs, then the next block's Q on its way while the sums are scaled
            float S[RA][8] = {};
            u2_t kc[2][D / 64];
#pragma unroll
            for (int T = 0; T < 2; T++) {
                if constexpr (D == 64) kc[T][0] = *reinterpret_cast<const u2_t *>(t + ko + T * (2 * D));
                else
#pragma unroll
                    for (int b = 0; b < D / 64; b += 2) {
                        const u4_t w = *reinterpret_cast<const u4_t *>(t + ko + (T * (2 * D) + 8 * b));
                        kc[T][b] = u2_t{w.x, w.y};
                        kc[T][b + 1] = u2_t{w.z, w.w};
                    }
            }
            h8_t qb[RA];
            const auto next_q = [&](int b) {
#pragma unroll
                for (int i = 0; i < RA; i++) qb[i] = RT == 1 ? qf[RT == 1 ? b : 0] : sq[(i * NB + b) * 64 + lane];
            };
            next_q(0);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const h8_t d = *reinterpret_cast<const h8_t *>(t + so + 64 * b);
                h8_t kf[2];
#pragma unroll
                for (int T = 0; T < 2; T++) kf[T] = b < D / 64 ? code_frag<0>(kc[T][b % (D / 64)]) : code_frag<1>(kc[T][b % (D / 64)]);
                barrier();
                f4_t A[RA][2];
#pragma unroll
                for (int i = 0; i < RA; i++)
#pragma unroll
                    for (int T = 0; T < 2; T++) A[i][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[T], qb[i], f4_t{}, 0, 0, 0);
                barrier();
                if (b + 1 < NB) next_q(b + 1);
                barrier();
#pragma unroll
                for (int i = 0; i < RA; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) S[i][e] = fmaf((float) d[e], A[i][e >> 2][e & 3], S[i][e]);
            }

            if (tile < e0 || tile >= e1) {  // keys that some row does not see
                const int64_t k0 = 32 * (int64_t) tile + 8 * g;
                // (the first of a lane's 8 keys that a row at `pos` sees, and how many from there on)
                const auto seen = [&](int64_t first_pos, int64_t pos, int & low, int & span) {
                    low = a.window ? (int) max(first_pos - a.window + 1 - k0, (int64_t) 0) : 0;
                    span = max((int) (min(pos + 1, cap) - k0) - low, 0);
                };
                int low, span;
#pragma unroll
                for (int i = 0; i < RA; i++) {
                    const int64_t pos = (int64_t) sw.past + (x0 + min(16 * i + lr, nr - 1)) / a.G;
                    seen(pos, pos, low, span);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int key = (e & 4) | (e & 1) << 1 | (e >> 1 & 1);  // order(e)
                        S[i][e] = (unsigned) (key - low) < (unsigned) span ? S[i][e] : -INFINITY;
                    }
                }
                // A key that no row sees may hold anything, a NaN for a scale too: its values' scales are set to 0.
                seen(pos0, pos1, low, span);
                h8_t * const vd = reinterpret_cast<h8_t *>(t + so + (2 * D + 64 * lr));
                if (lr < NB) {
                    h8_t z = *vd;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int key = (e & 4) | (e & 1) << 1 | (e >> 1 & 1);
                        z[e] = (unsigned) (key - low) < (unsigned) span ? z[e] : (_Float16) 0.0f;
                    }
                    *vd = z;
                }
            }
            h8_t ph[RA], pl[RA];
#pragma unroll
            for (int i = 0; i < RA; i++) {
                barrier();
                const float mx = max8(S[i]) * c2;
                if (__any(mx > top[i])) {
                    const float m = xor16_max(mx), Rn = m > top[i] ? ceilf(m) : R[i];  // (a row's R goes by its own scores)
                    const float al = R[i] == Rn ? 1.0f : __builtin_amdgcn_exp2f(R[i] - Rn);
                    R[i] = Rn;
                    top[i] = Rn + kSlack;
                    shift[i] = kP - (Rn == -INFINITY ? 0.0f : Rn);
                    l[i] *= al;
#pragma unroll
                    for (int t = 0; t < NT; t++) O[i][t] *= al;
                    big = big || __any(fabsf(Rn) >= kBig && Rn != -INFINITY);
                }
                float c = c2;
                if (big) {  // a row's R is its largest exponent rounded: round all alike
                    const bool mine = fabsf(shift[i]) >= kBig;
#pragma unroll
                    for (int e = 0; e < 8; e++) S[i][e] = mine ? rounded(S[i][e] * c2) - R[i] : S[i][e];
                    c = mine ? 1.0f : c2;
                }
                const float sh = big && fabsf(shift[i]) >= kBig ? kP : shift[i];
#pragma unroll
                for (int e = 0; e < 8; e++) S[i][e] = __builtin_amdgcn_exp2f(fmaf(S[i][e], c, sh));
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float p0 = S[i][e], p1 = S[i][e + 1];
                    const h2_t w = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
                    const h2_t u = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float) w.x, -1.0f, p0), fmaf((float) w.y, -1.0f, p1)));
                    ph[i][e] = w.x, ph[i][e + 1] = w.y, pl[i][e] = u.x, pl[i][e + 1] = u.y;
                }
                h8_t one;
#pragma unroll
                for (int e = 0; e < 8; e++) one[e] = (_Float16) 1.0f;
                f4_t z = {};
                z = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, pl[i], z, 0, 0, 0);
                z = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, ph[i], z, 0, 0, 0);
                l[i] += z[0];
            }
            // P V: 16 dims' MFMAs, then the next 16 dims' operands while they run, then their sums
            u4_t vc;
            h8_t vd[2], vh, vl;
            const auto next_v = [&](int n) {  // n: [b][u][low, high nibbles]
                const int b = n >> 2, u = n >> 1 & 1, H = n & 1;
                if ((n & 3) == 0) {
                    vc = *reinterpret_cast<const u4_t *>(t + vo + 1024 * b);
#pragma unroll
                    for (int h = 0; h < 2; h++) vd[h] = *reinterpret_cast<const h8_t *>(t + so + (2 * D + 64 * (b + h * (D / 64))));
                }
                h2_t cv[4];
                if (H) code_values<1>(vc[2 * u], vc[2 * u + 1], cv);
                else code_values<0>(vc[2 * u], vc[2 * u + 1], cv);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const h2_t d = {vd[H][2 * i], vd[H][2 * i + 1]};
                    const h2_t hi = cv[i] * d, lo = __builtin_elementwise_fma(cv[i], d, -hi);
                    vh[2 * i] = hi.x, vh[2 * i + 1] = hi.y, vl[2 * i] = lo.x, vl[2 * i + 1] = lo.y;
                }
            };
            next_v(0);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int td = 2 * (n >> 2) + (n >> 1 & 1) + (n & 1) * (D / 32);  // dims 16 td ..
                f4_t z[RA];
                barrier();
#pragma unroll
                for (int i = 0; i < RA; i++) z[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[i], f4_t{}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < RA; i++) z[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[i], z[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < RA; i++) z[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[i], z[i], 0, 0, 0);
                barrier();
                if (n + 1 < NT) next_v(n + 1);
                barrier();
#pragma unroll
                for (int i = 0; i < RA; i++) {
                    O[i][td] += z[i];
                    asm volatile("" : "+v"(O[i][td]));  // here: put off to the loop's end, every z keeps its registers
                }
            }
            wait_lds();  // the slot is read before the next tile is sent into it
            issue();
        }

        // the wavefronts' sums, brought to one R and added, 16 rows at a time
        float (*ex)[16][P] = reinterpret_cast<float (*)[16][P]>(shared);
        float2 (*exml)[16] = reinterpret_cast<float2 (*)[16]>(shared + NW * 16 * P * 4);
#pragma unroll
        for (int i = 0; i < RA; i++) {
            const int y0 = 16 * i, ny = min(16, nr - y0);
            __syncthreads();  // the rings, or the last 16 rows' sums, are read
            if (g == 0) exml[wave][lr] = make_float2(R[i], l[i]);
            __syncthreads();
            float Rm = exml[0][lr].x;
#pragma unroll
            for (int w = 1; w < NW; w++) Rm = fmaxf(Rm, exml[w][lr].x);
            const float f = R[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(R[i] - Rm);
            if (lr < ny)
#pragma unroll
                for (int t = 0; t < NT; t++) *reinterpret_cast<f4_t *>(&ex[wave][lr][16 * t + 4 * g]) = O[i][t] * f;
            __syncthreads();
            for (int e = threadIdx.x; e < ny * (D / 4); e += 64 * NW) {
                const int y = e / (D / 4), d = 4 * (e % (D / 4)), xx = x0 + y0 + y;
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
                    const float inv = 1.0f / sum;
                    *reinterpret_cast<f4_t *>(a.out + ((int64_t) (sw.r0 + xx / a.G) * a.H + hk * a.G + xx % a.G) * D + d) =
                        sum == 0.0f ? f4_t{} : o * inv;
                } else {
                    *reinterpret_cast<f4_t *>(a.part_o + ((int64_t) blockIdx.x * ROWS + y0 + y) * D + d) = o;
                    if (d == 0) a.part_ml[(int64_t) blockIdx.x * ROWS + y0 + y] = make_float2(m, sum);
                }
            }
        }
    };
    // (a sequence's single row beside others' prompts)
    if (RT == 1 || nr <= 16) body(std::integral_constant<int, 1>{});
    else body(std::integral_constant<int, RT>{});
}

// ------------------------------------------------------------------------ many rows of a sequence

// k_paged_many: a workgroup of four wavefronts takes 128 rows of a KV head, 32 a wavefront, and KT tiles of keys at a time. Each
// wavefront turns its share of the tiles' codes into operands of v_mfma_f32_32x32x16_f16, K's and V's values d (c - 8) as two f16
// parts each (15 bits: exact), and leaves them in LDS, lane by lane as the MFMAs take them, so that all four read them without a
// conflict; the next tiles' codes come into registers meanwhile. Scores, weights and sums as in k_paged_few, but that a score's
// chain runs over all dims (the small parts first). A lane holds the scores of one row and, of each tile, of the keys
// 8 G + order(j), G = 2 kc + lk: what its P V operand of chunk kc holds, V's operand being made of the same keys.
template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_paged_many(const AttnArgs a) {
    constexpr int NW = 4, KT = D == 256 ? 1 : 2, PP = NW / KT, ROWS = 32 * NW, NC = D / 16, ND = D / 32;
    constexpr int KU = D / 64 < PP / 2 ? 1 : D / 64 / (PP / 2);  // 64-dim groups of K codes of half the keys, per wavefront
    constexpr int VU = D / 32 / PP;                              // 32-dim groups of V codes of all keys, per wavefront
    __shared__ __align__(16) h8_t sk[KT][NC][2][64], sv[KT][ND][2][2][64];  // [tile][chunk][part][lane], [tile][dims][chunk][part][lane]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 31, lk = lane >> 5;
    Plan<ROWS> plan(a);
    if (!plan.find([&](int, int sum) { return __ballot(sum > (int) blockIdx.x); })) return;
    const SeqWork sw = plan.picked();
    const int ns = splits(sw.tiles, plan.chunk), id = blockIdx.x - plan.base;
    const int split = id % ns, rt = sw.rts - 1 - id / ns % sw.rts, hk = id / ns / sw.rts;

    const int rows = sw.rows * a.G, x0 = rt * ROWS, nr = min(ROWS, rows - x0);  // the workgroup's rows
    const int w0 = 32 * wave, wn = max(0, min(32, nr - w0));                     // this wavefront's of them
    const int64_t cap = (int64_t) a.p.max_pages << a.p.shift;
    const auto pos_of = [&](int y) { return (int64_t) sw.past + (x0 + y) / a.G; };
    const auto low_of = [&](int64_t pos) { return a.window ? max(pos - a.window + 1, (int64_t) 0) : (int64_t) 0; };
    const int64_t pos0 = pos_of(0), pos1 = pos_of(nr - 1);
    const int first = max(sw.tile0 + split * plan.chunk, (int) (low_of(pos0) >> 5));
    const int last = min(sw.tile0 + min(sw.tiles, (split + 1) * plan.chunk), (int) ((min(pos1 + 1, cap) + 31) >> 5));
    // the tiles that this wavefront's rows see; below e0 or from e1 on not whole
    const int64_t wp0 = pos_of(min(w0, nr - 1)), wp1 = pos_of(min(w0 + max(wn, 1) - 1, nr - 1));
    const int wf = wn ? (int) (low_of(wp0) >> 5) : 0, wl = wn ? (int) ((min(wp1 + 1, cap) + 31) >> 5) : 0;
    const int e0 = a.window ? (int) ((wp1 - a.window) >> 5) + 1 : 0, e1 = (int) ((wp0 + 1) >> 5);

    // the tiles' page entries, in the lanes, 64 at a time (KT divides 64)
    const int n = max(0, last - first);
    const int32_t * pages = a.p.pages + plan.s * a.p.ld;
    const int sub = a.p.shift - 5;
    int ent = -1;
    const auto entries = [&](int k) { ent = k + lane < n ? pages[(first + k + lane) >> sub] : -1; };
    if (n) entries(0);
    const auto there = [&](int k) { return k < n && (unsigned) __builtin_amdgcn_readlane(ent, k & 63) < (unsigned) a.p.n_pages; };

    // Q of the lane's row: chunk cc = [nibble H][block b of D/64][g >> 1], its half lk the dims D/2 H + 32 b + 8 g + order(0 .. 7)
    const int row = x0 + min(w0 + lr, nr - 1);
    const int64_t pos = (int64_t) sw.past + row / a.G;
    h8_t qf[NC];
    {
        const _Float16 * qp = a.q + (int64_t) (sw.r0 + row / a.G) * a.q_r + (int64_t) (hk * a.G + row % a.G) * a.q_h + 8 * lk;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            h8_t v = *reinterpret_cast<const h8_t *>(qp + 16 * c);
            if (w0 + lr >= nr) v = h8_t{};
            if (a.negate) v = -v;
            qf[c] = h8_t{v[0], v[2], v[1], v[3], v[4], v[6], v[5], v[7]};
        }
    }

    // This wavefront's share of a stage: of tile mt, K codes of the keys 16 T + (lane & 15), group g = lane >> 4 of 8 dims of each
    // block, of the 64-dim groups kb ..; V codes of the lane's 8 keys and its dims of the 32-dim groups vb ..
    const int mt = wave / PP, piece = wave % PP, T = piece & 1, c16 = lane & 15, g = lane >> 4;
    const int kb = (piece >> 1) * KU, vb = piece * VU;
    const int key = 16 * T + c16, slot = paged_order(key & 7);
    const uint32_t ko = key * (D / 2) + g * (D / 8) + 8 * kb, kdo = 32 * D + 2 * ((key & 24) + slot);
    // (MFMA row of the key: its slot (kc, lk, j) in P V's order)
    const int krow = 16 * (key >> 4) + 8 * (slot >> 2) + 4 * (key >> 3 & 1) + (slot & 3) + 32 * (g & 1);
    u2_t kr[KU], vr[VU];
    _Float16 kd[KU][2] = {};
    h8_t vd[VU][2] = {};
    const auto load = [&](int k) {  // the tile k + mt
        if (!there(k + mt)) {
#pragma unroll
            for (int u = 0; u < VU; u++) vd[u][0] = vd[u][1] = h8_t{};
            return;
        }
        const int e = __builtin_amdgcn_readlane(ent, (k + mt) & 63), t = first + k + mt;
        const uint8_t * p = a.p.data + ((((int64_t) e * a.p.Hkv + hk) << sub) + (t & ((1 << sub) - 1))) * (36 * D);
#pragma unroll
        for (int u = 0; u < KU; u++) {
            kr[u] = *reinterpret_cast<const u2_t *>(p + ko + 8 * u);
#pragma unroll
            for (int H = 0; H < 2; H++) kd[u][H] = *reinterpret_cast<const _Float16 *>(p + kdo + 64 * (kb + u + H * (D / 64)));
        }
#pragma unroll
        for (int u = 0; u < VU; u++) {  // 32-dim group vb + u: byte group u & 1 of t = u >> 1
            vr[u] = *reinterpret_cast<const u2_t *>(p + 16 * D + 1024 * ((vb + u) >> 1) + 16 * lane + 8 * ((vb + u) & 1));
#pragma unroll
            for (int H = 0; H < 2; H++) vd[u][H] = *reinterpret_cast<const h8_t *>(p + 34 * D + 64 * (((vb + u) >> 1) + H * (D / 64)) + 16 * g);
        }
        // A key that no row sees may hold anything, a NaN for a scale too: its values' scales are taken as 0.
        const int64_t k0 = 32 * (int64_t) t;
        if (k0 + 31 > pos1 || k0 < low_of(pos0)) {
            const int low = (int) max(low_of(pos0) - k0 - 8 * g, (int64_t) 0), span = max((int) (min(pos1 + 1, cap) - k0 - 8 * g) - low, 0);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool gone = (unsigned) (((j & 4) | (j & 1) << 1 | (j >> 1 & 1)) - low) >= (unsigned) span;
#pragma unroll
                for (int u = 0; u < VU; u++) {
                    vd[u][0][j] = gone ? (_Float16) 0.0f : vd[u][0][j];
                    vd[u][1][j] = gone ? (_Float16) 0.0f : vd[u][1][j];
                }
            }
        }
    };
    const auto parts = [](const h2_t (&c)[4], const h8_t & d, h8_t & hi, h8_t & lo) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const h2_t di = {d[2 * i], d[2 * i + 1]}, h = c[i] * di, r = __builtin_elementwise_fma(c[i], di, -h);
            hi[2 * i] = h.x, hi[2 * i + 1] = h.y, lo[2 * i] = r.x, lo[2 * i + 1] = r.y;
        }
    };
    const auto store = [&] {
#pragma unroll
        for (int u = 0; u < KU; u++)
#pragma unroll
            for (int H = 0; H < 2; H++) {
                h2_t c[4];
                if (H) code_values<1>(kr[u].x, kr[u].y, c);
                else code_values<0>(kr[u].x, kr[u].y, c);
                h8_t d, hi, lo;
#pragma unroll
                for (int j = 0; j < 8; j++) d[j] = kd[u][H];
                parts(c, d, hi, lo);
                h8_t * o = sk[mt][((H * (D / 64) + kb + u) << 1) + (g >> 1)][0] + krow;
                o[0] = hi;
                o[64] = lo;
            }
#pragma unroll
        for (int u = 0; u < VU; u++)
#pragma unroll
            for (int H = 0; H < 2; H++) {
                h2_t c[4];
                if (H) code_values<1>(vr[u].x, vr[u].y, c);
                else code_values<0>(vr[u].x, vr[u].y, c);
                h8_t hi, lo;
                parts(c, vd[u][H], hi, lo);
                h8_t * o = sv[mt][((vb + u) >> 1) + H * (D / 64)][g >> 1][0] + 16 * ((vb + u) & 1) + c16 + 32 * (g & 1);
                o[0] = hi;
                o[64] = lo;
            }
    };

    v16f O[ND];
    float R = -INFINITY, l = 0.0f, shift = kP;  // the reference exponent; this lane's part of the sum of weights; kP - R
#pragma unroll
    for (int t = 0; t < ND; t++) O[t] = v16f{};
    const float c2 = a.c2;

    // the next stage with a tile in it, from tile k on (a multiple of KT)
    const auto next = [&](int k) {
        for (; k < n; k += KT) {
            if ((k & 63) == 0 && k) entries(k);
            bool any = false;
#pragma unroll
            for (int t = 0; t < KT; t++) any = any || there(k + t);
            if (any) break;
        }
        return k;
    };
    int k = next(0);
    if (k < n) load(k);
    while (k < n) {
        uint32_t live = 0;  // tiles that are there and that some of this wavefront's rows see
        const int tile0 = first + k;
#pragma unroll
        for (int t = 0; t < KT; t++) live |= (uint32_t) (there(k + t) && tile0 + t >= wf && tile0 + t < wl) << t;
        __syncthreads();  // the last stage is read
        store();
        __syncthreads();
        k = next(k + KT);
        if (k < n) load(k);
        if (!live) continue;

        v16f S[KT];
#pragma unroll
        for (int t = 0; t < KT; t++) {
            v16f A{};
#pragma unroll
            for (int p = 1; p >= 0; p--)
#pragma unroll
                for (int c = 0; c < NC; c++) A = __builtin_amdgcn_mfma_f32_32x32x16_f16(sk[t][c][p][lane], qf[c], A, 0, 0, 0);
            S[t] = A;
        }
#pragma unroll
        for (int t = 0; t < KT; t++)
            if (tile0 + t < e0 || tile0 + t >= e1 || !(live >> t & 1)) {  // keys that some row does not see
                const int64_t k0 = 32 * (int64_t) (tile0 + t) + 8 * lk;
                const int low = (int) max(low_of(pos) - k0, (int64_t) 0), span = live >> t & 1 ? max((int) (min(pos + 1, cap) - k0) - low, 0) : 0;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int j = 16 * (r >> 3) + ((r & 4) | (r & 1) << 1 | (r >> 1 & 1));  // 16 kc + order(j)
                    S[t][r] = (unsigned) (j - low) < (unsigned) span ? S[t][r] : -INFINITY;
                }
            }
        // exponents against R as it is; where one passes it by too much, R moves and they are formed again
        float x[KT][16];
        const auto exponents = [&] {
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) x[t][r] = fmaf(S[t][r], c2, shift);
        };
        exponents();
        float mx = x[0][0];
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, x[t][r]);
        if (__any(mx > kP + kSlack || R == -INFINITY)) {
            float m = -INFINITY;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) m = fmaxf(m, S[t][r]);
            m = row_pair<32>(m * c2, fmaxf_op);
            const float Rn = m > R + kSlack ? ceilf(m) : R;  // (a row's R goes by its own scores)
            const float al = R == Rn ? 1.0f : __builtin_amdgcn_exp2f(R - Rn);
            R = Rn;
            shift = kP - (Rn == -INFINITY ? 0.0f : Rn);
            l *= al;
#pragma unroll
            for (int t = 0; t < ND; t++) O[t] *= al;
            exponents();
        }
        if (__any(fabsf(shift) >= kBig)) {  // a row's R is its largest exponent rounded: round all alike
            const bool mine = fabsf(shift) >= kBig;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) x[t][r] = mine ? (rounded(S[t][r] * c2) - R) + kP : x[t][r];
        }
        h8_t ph[KT][2], pl[KT][2];
        float l2 = 0.0f;
        constexpr h2_t one = {(_Float16) 1.0f, (_Float16) 1.0f};
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float p0 = __builtin_amdgcn_exp2f(x[t][r]), p1 = __builtin_amdgcn_exp2f(x[t][r + 1]);
                const h2_t w = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
                const h2_t u = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float) w.x, -1.0f, p0), fmaf((float) w.y, -1.0f, p1)));
                l2 = __builtin_amdgcn_fdot2(w, one, l2, false);
                l = __builtin_amdgcn_fdot2(u, one, l, false);
                ph[t][r >> 3][r & 7] = w.x, ph[t][r >> 3][(r & 7) + 1] = w.y, pl[t][r >> 3][r & 7] = u.x, pl[t][r >> 3][(r & 7) + 1] = u.y;
            }
        l += l2;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            __builtin_amdgcn_sched_barrier(0);
            v16f z{};
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const h8_t vh = sv[t][d][c][0][lane], vl = sv[t][d][c][1][lane];
                    z = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[t][c], z, 0, 0, 0);
                    z = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[t][c], z, 0, 0, 0);
                    z = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[t][c], z, 0, 0, 0);
                }
            O[d] += z;
            asm volatile("" : "+v"(O[d]));  // here: put off to the loop's end, every z keeps its registers
        }
    }
    l = row_pair<32>(l, op_add<float>);
    if (w0 + lr >= nr) return;
    float * o = ns == 1 ? a.out + ((int64_t) (sw.r0 + row / a.G) * a.H + hk * a.G + row % a.G) * D + 4 * lk
                        : a.part_o + ((int64_t) blockIdx.x * ROWS + w0 + lr) * D + 4 * lk;
    const float f = ns == 1 ? 1.0f / l : 1.0f;
#pragma unroll
    for (int t = 0; t < ND; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f4_t y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = ns == 1 && l == 0.0f ? 0.0f : O[t][4 * i + r] * f;
            *reinterpret_cast<f4_t *>(o + 32 * t + 8 * i) = y;
        }
    if (ns > 1 && lk == 0) a.part_ml[(int64_t) blockIdx.x * ROWS + w0 + lr] = make_float2(R, l);
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
    const int64_t item = plan.base + ((int64_t) (h / a.G) * sw.rts + sw.rts - 1 - x / ROWS) * ns;
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

// How a call is run: row tiles of `rows` rows (up to 32: k_paged_few), splits that aim at `target` workgroups, those resident at
// once.
struct Shape {
    int rows, target;
    int64_t items, most;  // workgroups that may have work; splits of a sequence
};
Shape shape_for(const Paged & p, int D, int G, int64_t max_rows) {
    Shape s{};
    const int64_t per_seq = std::min<int64_t>(max_rows, p.n_rows) * G;  // rows of a KV head
    s.rows = per_seq <= 16 ? 16 : per_seq <= 32 ? 32 : 128;
    s.target = 256 * (s.rows == 16 && D != 256 ? 4 : 2);
    // row tiles: the rows' whole tiles and one more for each sequence
    const int64_t rts = p.Hkv * std::min<int64_t>((int64_t) p.n_rows * G / s.rows + std::min<int64_t>(p.n_seq, p.n_rows),
                                                  p.n_seq * ((per_seq + s.rows - 1) / s.rows));
    s.most = (((int64_t) p.max_pages << p.shift) / kPagedTile + kMinChunk - 1) / kMinChunk;
    s.items = std::min(rts + s.target, rts * s.most);
    return s;
}

template <int D, int ROWS>
void merge(const AttnArgs & a, const Shape & w, hipStream_t s) {
    check_launch("paged attn");
    if (w.most > 1) k_paged_merge<D, ROWS><<<dim3((unsigned) a.p.n_rows, (unsigned) a.H), 256, 0, s>>>(a);
    check_launch("paged attn merge");
}
template <int D>
void run(const AttnArgs & a, const Shape & w, hipStream_t s) {
    if (w.rows == 16) {
        k_paged_few<D, 1, 4><<<(unsigned) a.items, 256, 0, s>>>(a);
        merge<D, 16>(a, w, s);
    } else if (w.rows == 32) {
        k_paged_few<D, 2, 4><<<(unsigned) a.items, 256, 0, s>>>(a);
        merge<D, 32>(a, w, s);
    } else {
        k_paged_many<D><<<(unsigned) a.items, 256, 0, s>>>(a);
        merge<D, 128>(a, w, s);
    }
}

}  // namespace

size_t paged_attn_workspace(const Paged & p, int D, int H, int64_t max_rows) {
    if (p.n_rows == 0) return 0;
    const Shape w = shape_for(p, D, H / p.Hkv, max_rows);
    return w.most == 1 ? 0 : (size_t) w.items * w.rows * (D * sizeof(float) + sizeof(float2));
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
    const Shape w = shape_for(p, D, a.G, max_rows);
    require(w.items < INT32_MAX, "paged_attn: too many rows and heads");
    a.items = (int) w.items, a.target = w.target;
    a.part_o = (float *) ws;
    a.part_ml = (float2 *) ((char *) ws + (size_t) w.items * w.rows * D * sizeof(float));
    if (D == 64) run<64>(a, w, s);
    else if (D == 128) run<128>(a, w, s);
    else run<256>(a, w, s);
}

}  // namespace gcq

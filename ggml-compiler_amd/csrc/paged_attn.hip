// paged_attn.hip - attention over the paged 4-bit cache (include/gcq_paged.h; layout in paged.h).
//
// A row is a (query, head) pair of one KV head (row j G + g of a sequence, G query heads to a KV head). k_paged_attn gives a
// workgroup a row tile of 16 RT rows and a run of key tiles, which its NW wavefronts take in turn, each over all the rows:
//   - a tile comes straight from memory into the wavefront's two slots of LDS (36 D bytes, the next tile under way);
//   - scores S^T[key][row] = K Q^T, one v_mfma_f32_16x16x32_f16 per Q4_0 block of 32 dims and 16 keys, on the codes c - 8
//     themselves (exact in f16); a block's sum is scaled by its d in f32;
//   - lane (row, g) is left with the scores of keys 8 g .. 8 g + 7, in the order that P V's operand wants them;
//   - O^T[dim][row] += V^T P^T, V's values d (c - 8) as two f16 parts (15 bits: exact), P as two of 11 bits, the second one
//     rounded: 2^-23 of a weight, or 2^-36 of 2^R where that is more; the sum of weights goes through the same two parts (a row
//     of ones), so that numerator and denominator see the same.
// The softmax runs in powers of two against an integer reference R that follows the maximum in steps: it moves when a score
// passes it by 4, which is rare, and moving it scales by an exact power of two. Chains inside the MFMAs (whose sums are
// cut off, not rounded) start from zero for each tile; tiles are added in f32. Against 64 bits the outputs are off by 1e-7 to
// 7e-7 (2-norm; the more where one key is far ahead of up to 65535 others that together still count).
//
// Work: a sequence's tiles are cut into even splits of about `chunk` tiles, one chunk for all sequences, chosen so that all splits of
// all row tiles come to Shape::target workgroups. Every workgroup computes that plan from the batch's arrays by itself (no planning
// launch, and a captured graph follows the arrays), finds its split by a prefix sum over the sequences and joins its wavefronts'
// sums in LDS. Row tiles of several splits are joined by k_paged_merge, from notes (Part) that the workgroups leave.
//
// What bounds it: where wavefronts have many tiles the vector ALU. A tile of heads of 128 costs a wavefront some 335 operations at 16
// rows: 216 to make its 4-bit codes into MFMA operands, whatever the rows, the others for 16 rows' scaling, softmax and sums.
// Reads alone, all arithmetic left out, took 25 us of 131071 keys' 39 (one row of 32 heads, 8 KV heads, 151 MB: 3.8 TB/s). With few
// tiles to a wavefront, plan, lookups, the first tile and the join weigh as much: 26 us for 32 sequences of 232 to 7611 keys, 15 of
// them reads alone, 11 the tiles' operations. 512 rows over 4096 keys take 88 us (365 TFLOP/s of 4 D flops a key and row; the
// MFMAs do twice those, for the parts). The ALU is also why a wavefront has all of its rows' dims: shared between wavefronts by
// way of LDS, the operands of a tile took longer to write there (34 cycles a KiB of a CU's) than to make again.
#include "paged.h"

#include <algorithm>

namespace gcq {

namespace {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr int kMinChunk = 16;    // tiles of a split: four to a wavefront (32 sequences' step: 25.3 us, with 32 tiles 28.6)
constexpr float kSlack = 4.0f;   // how far a score's exponent may pass R
constexpr float kBig = 0x1p20f;  // exponents from here on are no longer exact to 2^-4
constexpr float kP = 11.0f;      // the exponent of P's scale: with kSlack at most 2^15, f16's largest power; parts down to 2^-35 of 2^R

struct AttnArgs {
    Paged p;
    const _Float16 * q;
    int64_t q_r, q_h;
    int H, G, window, max_rows, items, slots, target, min_chunk;  // slots: of part_o, part_ml; target: workgroups that the splits aim at
    float c2;     // |scale| log2(e)
    bool negate;  // the scale is negative
    float * out, * part_o;
    float2 * part_ml;
    struct Part * parts;  // one for each workgroup; null: nothing is split
};

// What k_paged_merge has to know of a workgroup's row tile.
struct __align__(32) Part {
    int ns, split, nr, hk, r0, x0, slot;  // ns 0: no work; slot: where its sums are, if ns > 1
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

// The plan, the same in every wavefront: tiles per split, and a sequence's first item. Items of a sequence: [KV
// head][row tile, the last, which sees most, first][split]. The batch's arrays are read once where the sequences fit the lanes.
// Items of split row tiles have a slot each for their sums. Those are fewer than 2 target: with u tiles in all items' and a chunk of more than
// u / cut, a row tile has less than tiles cut / u splits more than one, all of them together less than cut <= target, and a split row tile has
// at most twice as many splits as that.
template <int ROWS>
struct Plan {
    const AttnArgs & a;
    SeqWork w;  // of sequence s0 + lane
    int chunk, s, base, slot, lane_at;

    __device__ __forceinline__ Plan(const AttnArgs & args) : a(args) {
        const int lane = threadIdx.x & 63;
        w = seq_work<ROWS>(a, lane);
        chunk = a.min_chunk;
        if (!a.parts) return;  // one split each
        double u = (double) w.rts * w.tiles, n = w.rts;
        for (int s0 = 64; s0 < a.p.n_seq; s0 += 64) {
            const SeqWork x = seq_work<ROWS>(a, s0 + lane);
            u += (double) x.rts * x.tiles;
            n += x.rts;
        }
        u = wave_sum_d(u) * a.p.Hkv;
        n = wave_sum_d(n) * a.p.Hkv;
        const double cut = fmax(a.target - n, 0.5 * a.target);
        chunk = __builtin_amdgcn_readfirstlane((int) fmax((double) a.min_chunk, fmin(u / cut + 1.0, 1e9)));
    }

    // The sequence found, uniform.
    __device__ __forceinline__ SeqWork picked() {
        const int l = __builtin_amdgcn_readfirstlane(lane_at);
        const auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
        base = __builtin_amdgcn_readfirstlane(base);
        slot = __builtin_amdgcn_readfirstlane(slot);
        s = __builtin_amdgcn_readfirstlane(s);
        return {pick(w.r0), pick(w.rows), pick(w.tile0), pick(w.tiles), pick(w.rts), pick(w.past)};
    }
    // To the sequence of item `id`; base: its first, slot: that one's.
    __device__ __forceinline__ bool find(int id) {
        const int lane = threadIdx.x & 63;
        base = slot = 0;
        for (int s0 = 0; s0 < a.p.n_seq; s0 += 64) {
            if (s0) w = seq_work<ROWS>(a, s0 + lane);
            const int ns = splits(w.tiles, chunk), n = w.rts * a.p.Hkv * ns, sum = wave_scan(n);
            const int m = ns > 1 ? n : 0, sum_m = wave_scan(m);
            const uint64_t at = __ballot(base + sum > id);
            if (at) {
                lane_at = __builtin_ctzll(at);
                base += __builtin_amdgcn_readlane(sum - n, lane_at);
                slot += __builtin_amdgcn_readlane(sum_m - m, lane_at);
                s = s0 + lane_at;
                return true;
            }
            base += __builtin_amdgcn_readlane(sum, 63);
            slot += __builtin_amdgcn_readlane(sum_m, 63);
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
// (As inline code, m0 set and used in one piece, since the compiler has a builtin's loads waited for, all of them, before any LDS read.
// The base may come from a v_readlane just before: five wait states to a memory access that reads it, which the compiler leaves between
// its own instructions only.)
template <int D> constexpr int kTileLoads = (36 * D + 1023) / 1024;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is a reserved register: it is said all the same that it changes)
template <int N>
__device__ __forceinline__ void lds_load(const uint8_t * base, uint32_t voff, uint32_t lds) {  // N KiB
    static_assert(N >= 1 && N <= 3, "the offset has 13 bits, signed");
    if constexpr (N == 1) asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds) : "memory", "m0");
    if constexpr (N == 2) asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1\n\tglobal_load_lds_dwordx4 %0, %1 offset:1024" ::"v"(voff), "s"(base), "s"(lds) : "memory", "m0");
    if constexpr (N == 3) asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1\n\tglobal_load_lds_dwordx4 %0, %1 offset:1024\n\tglobal_load_lds_dwordx4 %0, %1 offset:2048" ::"v"(voff), "s"(base), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int D>
__device__ __forceinline__ void tile_load(const uint8_t * t, uint32_t lds, int lane) {  // (t, lds: uniform)
    constexpr int full = 36 * D / 1024, rest = (36 * D % 1024) / 16;
    lds = __builtin_amdgcn_readfirstlane(lds);
#pragma unroll
    for (int i = 0; i < full; i += 3) {
        const uint32_t v = 16 * lane + 1024 * i;
        if (i + 2 < full) lds_load<3>(t, v, lds + 1024 * i);
        else if (i + 1 < full) lds_load<2>(t, v, lds + 1024 * i);
        else lds_load<1>(t, v, lds + 1024 * i);
    }
    if (rest && lane < rest) lds_load<1>(t, 16 * lane + 1024 * full, lds + 1024 * full);
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Wavefronts per SIMD that the registers (and, heads of 256, LDS) hold; and of a workgroup.
// (Eight wavefronts to a workgroup, heads of 128: 32 sequences' step 32.1 us for 25.3 with four, four prompts 134 for 86; heads of
// 256 with 32 rows, whose four wavefronts would fill half the LDS: 52.6 us with eight, 80.3 with four.)
constexpr int per_simd(int D, int RT) { return D * RT <= 128 ? 4 : D * RT == 256 && RT == 2 ? 3 : 2; }
constexpr int waves(int D, int rows) { return D == 256 && rows == 32 ? 8 : 4; }

template <int D, int RT, int NW>
__global__ __launch_bounds__(64 * NW, per_simd(D, RT)) void k_paged_attn(const AttnArgs a) {
    constexpr int ROWS = 16 * RT, NB = D / 32, NT = D / 16, RING = 2, NL = kTileLoads<D>, P = D + 4;
    // LDS: the wavefronts' rings (then their sums of 16 rows), and the row tile's Q as MFMA operands (from two times 16
    // rows on; registers hold 16)
    constexpr int kRings = NW * RING * 36 * D, kSums = NW * 16 * (P * 4 + 8), kQ = RT > 1 ? ROWS * D * 2 : 0;
    __shared__ __align__(16) uint8_t shared[(kRings > kSums ? kRings : kSums) + kQ];
    h8_t * const sq = reinterpret_cast<h8_t *>(shared + (kRings > kSums ? kRings : kSums));  // [16 rows][block][lane]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
    __builtin_amdgcn_s_setprio(3);
    Plan<ROWS> plan(a);
    if (!plan.find(blockIdx.x)) {
        if (a.parts && threadIdx.x == 0) a.parts[blockIdx.x] = Part{};
        return;
    }
    const SeqWork sw = plan.picked();
    const int ns = splits(sw.tiles, plan.chunk), chunk = (sw.tiles + ns - 1) / ns, id = blockIdx.x - plan.base;
    const int split = id % ns, rt = sw.rts - 1 - id / ns % sw.rts, hk = id / ns / sw.rts, slot_of = plan.slot + id;

    const int rows = sw.rows * a.G, x0 = rt * ROWS, nr = min(ROWS, rows - x0);  // this tile's rows
    if (a.parts && threadIdx.x == 0) a.parts[blockIdx.x] = {ns, split, nr, hk, sw.r0, x0, slot_of};
    if (ns > 1 && slot_of >= a.slots) return;  // (arrays that change under the call: no sums outside the workspace)
    const int64_t pos0 = (int64_t) sw.past + x0 / a.G, pos1 = (int64_t) sw.past + (x0 + nr - 1) / a.G;
    // this row tile's keys within the split; tiles below e0 or from e1 on are not seen whole by every row
    const int64_t cap = (int64_t) a.p.max_pages << a.p.shift;
    const int first = max(sw.tile0 + split * chunk, a.window && pos0 - a.window + 1 > 0 ? (int) ((pos0 - a.window + 1) >> 5) : 0);
    const int last = min(sw.tile0 + min(sw.tiles, (split + 1) * chunk), (int) ((min(pos1 + 1, cap) + 31) >> 5));
    const int e0 = a.window ? (int) ((pos1 - a.window) >> 5) + 1 : 0, e1 = (int) ((pos0 + 1) >> 5);

    // The tiles of this wavefront: first + wave, + NW, ..; lane i holds the address of tile k0 + i, 0 for one that is not there.
    const int n = first + wave < last ? (last - first - wave + NW - 1) / NW : 0;
    const int32_t * pages = a.p.pages + plan.s * a.p.ld;
    const int sub = a.p.shift - 5;
    int entry = -1;
    const auto entries = [&](int k0) {
        if (k0 + lane < n) entry = pages[(first + wave + NW * (k0 + lane)) >> sub];
    };
    uint32_t at_lo, at_hi;
    const auto addresses = [&](int k0) {
        const int t = first + wave + NW * (k0 + lane);
        const uint64_t at = (uint64_t) (uintptr_t) a.p.data + (((((uint64_t) (uint32_t) entry * a.p.Hkv + hk) << sub) + (t & ((1 << sub) - 1))) * (36 * D));
        const bool there = k0 + lane < n && (unsigned) entry < (unsigned) a.p.n_pages;
        at_lo = there ? (uint32_t) at : 0;
        at_hi = there ? (uint32_t) (at >> 32) : 0;
        asm volatile("" : "+v"(at_lo), "+v"(at_hi));  // (the entries are waited for here, once)
    };
    entries(0);

    // Q: of a lane's row, dims 32 b + 8 g + order(0 .. 7)
    const auto load_q = [&](int i, int b) {
        const int y = 16 * i + lr, x = x0 + min(y, nr - 1);
        h8_t v = *reinterpret_cast<const h8_t *>(a.q + (int64_t) (sw.r0 + x / a.G) * a.q_r + (int64_t) (hk * a.G + x % a.G) * a.q_h + 32 * b + 8 * g);
        if (y >= nr) v = h8_t{};
        // An infinity becomes a NaN, as softmax makes of every key's score with it: scores of -inf alone would leave R at -inf, and
        // the row would count as one without keys.
        v = __builtin_elementwise_fma(v, h8_t{}, v);
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
    // the next tile that is there, from k on, sent into a slot; n if there is none
    const auto issue = [&](int k, int slot) {
        for (; k < n; k++) {
            if ((k & 63) == 0 && k) {
                entries(k);
                addresses(k);
            }
            const uint32_t lo = __builtin_amdgcn_readlane(at_lo, k & 63), hi = __builtin_amdgcn_readlane(at_hi, k & 63);
            if (lo | hi) {
                tile_load<D>(reinterpret_cast<const uint8_t *>((uint64_t) hi << 32 | lo), ring_at + slot * (36 * D), lane);
                break;
            }
        }
        return k;
    };
    addresses(0);
    int at = issue(0, 0), after = issue(at + 1, 1);

    // the work on RA times 16 rows
    const auto body = [&](auto ra) {
        constexpr int RA = decltype(ra)::value;
        f4_t O[RA][NT];
        float R[RA], l[RA], top[RA], shift[RA];  // the reference exponent; where it moves; kP - R
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

        for (int slot = 0; at < n; slot ^= 1) {
            if (after < n) wait_loads<NL>();
            else wait_loads<0>();
            // The wavefront with most tiles left goes first: by age, as they otherwise go, a SIMD's four finished one after the
            // other, the last one alone and waiting on itself (131071 keys: 38.9 us for 41.1; 512 rows 95 for 98).
            const int left = n - at;
            if (left > 6) __builtin_amdgcn_s_setprio(3);
            else if (left > 3) __builtin_amdgcn_s_setprio(2);
            else if (left > 1) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
            const int tile = first + wave + NW * at;
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
                    barrier();
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
            // the weights: R first, for all rows in one branch, then exponents
            float mx[RA];
            bool move = false;
#pragma unroll
            for (int i = 0; i < RA; i++) {
                mx[i] = max8(S[i]) * c2;
                move = move || mx[i] > top[i];
            }
            if (__any(move)) {
#pragma unroll
                for (int i = 0; i < RA; i++) {
                    const float m = xor16_max(mx[i]), Rn = m > top[i] ? ceilf(m) : R[i];  // (a row's R goes by its own scores)
                    const float al = R[i] == Rn ? 1.0f : __builtin_amdgcn_exp2f(R[i] - Rn);
                    R[i] = Rn;
                    top[i] = fabsf(Rn) >= kBig ? Rn : Rn + kSlack;  // (from 2^26 on R + 4 may be R + 8, more than P has room for)
                    shift[i] = kP - (Rn == -INFINITY ? 0.0f : Rn);
                    l[i] *= al;
#pragma unroll
                    for (int t = 0; t < NT; t++) O[i][t] *= al;
                    big = big || __any(fabsf(Rn) >= kBig && Rn != -INFINITY);
                }
            }
            float c[RA], sh[RA];
#pragma unroll
            for (int i = 0; i < RA; i++) c[i] = c2, sh[i] = shift[i];
            if (big) {  // a row's R is its largest exponent rounded: round all alike
#pragma unroll
                for (int i = 0; i < RA; i++) {
                    const bool mine = fabsf(shift[i]) >= kBig;
#pragma unroll
                    for (int e = 0; e < 8; e++) S[i][e] = mine ? rounded(S[i][e] * c2) - R[i] : S[i][e];
                    c[i] = mine ? 1.0f : c2;
                    sh[i] = mine ? kP : shift[i];
                }
            }
            float minus = -1.0f;  // (unknown to the compiler: one v_fma_mix_f32 and not a conversion and a subtraction)
            asm("" : "+s"(minus));
            h8_t ph[RA], pl[RA];
#pragma unroll
            for (int i = 0; i < RA; i++)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(S[i][e], c[i], sh[i])), p1 = __builtin_amdgcn_exp2f(fmaf(S[i][e + 1], c[i], sh[i]));
                    const h2_t w = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
                    // (rounded: cut off, many small weights beside a large one would all lose)
                    const h2_t u = __builtin_convertvector(f2_t{fmaf((float) w.x, minus, p0), fmaf((float) w.y, minus, p1)}, h2_t);
                    ph[i][e] = w.x, ph[i][e + 1] = w.y, pl[i][e] = u.x, pl[i][e + 1] = u.y;
                }
            // P V: 16 dims' MFMAs, then the next 16 dims' operands and the last ones' sums while they run; a row of ones at the
            // end for the sum of weights
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
            f4_t z[2][RA];
            const auto add = [&](int n) {
                const int td = 2 * (n >> 2) + (n >> 1 & 1) + (n & 1) * (D / 32);  // dims 16 td ..
#pragma unroll
                for (int i = 0; i < RA; i++) {
                    O[i][td] += z[n & 1][i];
                    asm volatile("" : "+v"(O[i][td]));  // here: put off to the loop's end, every z keeps its registers
                }
            };
            next_v(0);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                barrier();
#pragma unroll
                for (int i = 0; i < RA; i++) z[n & 1][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[i], f4_t{}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < RA; i++) z[n & 1][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[i], z[n & 1][i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < RA; i++) z[n & 1][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[i], z[n & 1][i], 0, 0, 0);
                barrier();
                if (n) add(n - 1);
                if (n + 1 < NT) next_v(n + 1);
            }
            h8_t one;
#pragma unroll
            for (int e = 0; e < 8; e++) one[e] = (_Float16) 1.0f;
            barrier();
#pragma unroll
            for (int i = 0; i < RA; i++) z[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, pl[i], f4_t{}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < RA; i++) z[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, ph[i], z[0][i], 0, 0, 0);
            barrier();
            add(NT - 1);
#pragma unroll
            for (int i = 0; i < RA; i++) l[i] += z[0][i][0];
            wait_lds();  // the slot is read before the next tile is sent into it
            at = after;
            after = issue(after + 1, slot);
        }

        __builtin_amdgcn_s_setprio(0);
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
                    *reinterpret_cast<f4_t *>(a.part_o + ((int64_t) slot_of * ROWS + y0 + y) * D + d) = o;
                    if (d == 0) a.part_ml[(int64_t) slot_of * ROWS + y0 + y] = make_float2(m, sum);
                }
            }
        }
    };
    // (a sequence's single row beside others' prompts)
    if (RT == 1 || nr <= 16) body(std::integral_constant<int, 1>{});
    else body(std::integral_constant<int, RT>{});
}

// A row tile of several splits: their sums, weighted by 2^(R - the largest R). The splits' workgroups share its rows, row y to
// split y % ns's; a row's splits are read by the workgroup's four wavefronts together if they are more than one has under way.
// (4.8 us for 131071 keys' 125 splits, 8.6 with a wavefront to a row; 4.6 us for 16 sequences' 35 rows in 3 splits, 24.5 with four.)
template <int D, int ROWS>
__global__ __launch_bounds__(256) void k_paged_merge(const AttnArgs a) {
    constexpr int L = D / 4, N1 = 64 / L, N4 = 4 * N1;  // lanes of a split; splits at a time, a wavefront's and all four's
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), d = lane % L;
    const Part w = a.parts[blockIdx.x];
    const int ns = __builtin_amdgcn_readfirstlane(w.ns), split = __builtin_amdgcn_readfirstlane(w.split), item = __builtin_amdgcn_readfirstlane(w.slot) - split;
    if (ns <= 1 || split >= w.nr || (int) blockIdx.x - split + ns > a.items || item < 0 || item + ns > a.slots) return;  // (starts that do not ascend)
    __shared__ f4_t so[N4][L];
    __shared__ float2 sml[N4];
    const auto weight = [](float from, float to) { return from == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(from - to); };
    const auto row = [&](int y, int part, int parts, f4_t & acc, float & R, float & l) {
        const float2 * ml = a.part_ml + (int64_t) item * ROWS + y;
        const float * o = a.part_o + ((int64_t) item * ROWS + y) * D;
        R = -INFINITY;
        acc = f4_t{};
        l = 0.0f;
        for (int i = part; i < ns; i += 8 * parts) {  // eight loads under way at a time
            float2 m[8];
            f4_t v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int64_t at = min(i + k * parts, ns - 1);
                m[k] = ml[at * ROWS];
                v[k] = *reinterpret_cast<const f4_t *>(o + at * ROWS * D + 4 * d);
            }
            float Rn = R;
#pragma unroll
            for (int k = 0; k < 8; k++) Rn = fmaxf(Rn, m[k].x);
            const float al = weight(R, Rn);
            l *= al;
            acc *= al;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float f = i + k * parts >= ns ? 0.0f : weight(m[k].x, Rn);
                l += m[k].y * f;
                acc += v[k] * f;
            }
            R = Rn;
        }
    };
    const auto put = [&](int y, f4_t acc, float l) {
        const int x = w.x0 + y;
        const float inv = 1.0f / l;
        *reinterpret_cast<f4_t *>(a.out + ((int64_t) (w.r0 + x / a.G) * a.H + w.hk * a.G + x % a.G) * D + 4 * d) = l == 0.0f ? f4_t{} : acc * inv;
    };
    f4_t acc;
    float R, l;
    if (ns > 8 * N1) {  // (one or two rows of the tile's 32 at most, heads of 256 up to four)
        for (int y = split; y < w.nr; y += ns) {
            row(y, tid / L, N4, acc, R, l);
            so[tid / L][d] = acc;
            if (d == 0) sml[tid / L] = make_float2(R, l);
            __syncthreads();
            if (tid < L) {
                float Rm = -INFINITY;
#pragma unroll
                for (int i = 0; i < N4; i++) Rm = fmaxf(Rm, sml[i].x);
                acc = f4_t{};
                l = 0.0f;
#pragma unroll
                for (int i = 0; i < N4; i++) {
                    const float f = weight(sml[i].x, Rm);
                    l += sml[i].y * f;
                    acc += so[i][d] * f;
                }
                put(y, acc, l);
            }
            __syncthreads();
        }
        return;
    }
    for (int y = split + wave * ns; y < w.nr; y += 4 * ns) {
        row(y, lane / L, N1, acc, R, l);
        float Rm = R;
#pragma unroll
        for (int s = 32; s >= L; s >>= 1) Rm = fmaxf(Rm, __shfl_xor(Rm, s, 64));
        const float f = weight(R, Rm);
        l *= f;
        acc *= f;
#pragma unroll
        for (int s = 32; s >= L; s >>= 1) {
            l += __shfl_xor(l, s, 64);
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], s, 64);
        }
        if (lane < L) put(y, acc, l);
    }
}

// How a call is run: row tiles of `rows` rows, splits that aim at `target` workgroups, those resident at once.
struct Shape {
    int rows, target;
    int64_t tiles, items, slots, most;  // row tiles and workgroups that may have work; sums of splits; splits of a sequence
};
Shape shape_of(const Paged & p, int D, int G, int64_t max_rows, int window, int rows) {
    Shape s{};
    s.rows = rows;
    s.target = 256 * 4 * per_simd(D, rows / 16) / waves(D, rows);
    // row tiles: the rows' whole tiles and one more for each sequence
    const int64_t per_seq = std::min<int64_t>(max_rows, p.n_rows) * G;
    s.tiles = p.Hkv * std::min<int64_t>((int64_t) p.n_rows * G / rows + std::min<int64_t>(p.n_seq, p.n_rows),
                                        p.n_seq * ((per_seq + rows - 1) / rows));
    int64_t longest = ((int64_t) p.max_pages << p.shift) / kPagedTile;  // tiles that a sequence's rows can see
    if (window) longest = std::min(longest, (window + std::min<int64_t>(max_rows, p.n_rows) - 2) / kPagedTile + 2);
    // (two splits of the least size gain nothing and need the join: 501 keys 9.5 us as one split, 10.7 + 3.7 as two)
    s.most = longest <= 2 * kMinChunk ? 1 : (longest + kMinChunk - 1) / kMinChunk;
    s.items = std::min(s.tiles + s.target, s.tiles * s.most);
    s.slots = std::min<int64_t>(s.items, 2 * s.target);
    return s;
}
// Tiles of 32 rows halve the work on K and V; tiles of 16 are more workgroups, of half the length. The larger ones if they
// can still keep six wavefronts on every CU. (Heads of 128, 8 KV heads, tiles of 16 and of 32: 2000 keys, 20 rows of a KV
// head 12.9 and 17.1 us, 256 rows 22.0 and 24.8; 32000 keys, 20 rows 28.9 and 25.0, 256 rows 125 and 100; 16 sequences of
// 1000 keys, 64 rows 22.9 and 22.9, 256 rows 67.9 and 59.4.)
Shape shape_for(const Paged & p, int D, int G, int64_t max_rows, int window) {
    const Shape few = shape_of(p, D, G, max_rows, window, 16), many = shape_of(p, D, G, max_rows, window, 32);
    const bool wide = std::min<int64_t>(max_rows, p.n_rows) * G > 16 && many.tiles * many.most * waves(D, 32) >= 6 * 256;
    return wide ? many : few;
}
size_t workspace_of(const Shape & w, int D) {
    return w.most == 1 ? 0 : (size_t) w.slots * w.rows * (D * sizeof(float) + sizeof(float2)) + (size_t) w.items * sizeof(Part);
}

template <int D, int RT>
void launch(const AttnArgs & a, const Shape & w, hipStream_t s) {
    constexpr int ROWS = 16 * RT, NW = waves(D, ROWS);
    k_paged_attn<D, RT, NW><<<paged_grid(a.items, 64 * NW), 64 * NW, 0, s>>>(a);
    check_launch("paged attn");
    if (w.most == 1) return;
    k_paged_merge<D, ROWS><<<paged_grid(a.items, 256), 256, 0, s>>>(a);
    check_launch("paged attn merge");
}
template <int D>
void run(const AttnArgs & a, const Shape & w, hipStream_t s) {
    if (w.rows == 16) launch<D, 1>(a, w, s);
    else launch<D, 2>(a, w, s);
}

}  // namespace

// (for any window: a window only takes splits away)
size_t paged_attn_workspace(const Paged & p, int D, int H, int64_t max_rows) {
    if (p.n_rows == 0) return 0;
    const int G = H / p.Hkv;
    return std::max(workspace_of(shape_of(p, D, G, max_rows, 0, 16), D), workspace_of(shape_of(p, D, G, max_rows, 0, 32), D));
}

void launch_paged_attn(const Paged & p, int D, const void * q, int64_t q_r, int64_t q_h, int H, int64_t max_rows, int window,
                       float scale, float * out, void * ws, hipStream_t s) {
    AttnArgs a{};
    a.p = p, a.q = (const _Float16 *) q, a.q_r = q_r, a.q_h = q_h, a.H = H, a.G = H / p.Hkv, a.window = window;
    a.max_rows = (int) std::min<int64_t>(max_rows, p.n_rows);
    // (from 0 up to 2^-100: scores of 0 either way, but -inf for a hidden key. Down to 2^86: q K is at most 2^40, all exponents
    // stay within f32, and two scores q K that differ, by 2^-48 at the least, are 2^38 powers of two apart already.)
    a.c2 = (float) (std::min(std::max(fabs((double) scale), 0x1p-100), 0x1p86) * 1.4426950408889634074);
    a.negate = scale < 0.0f;
    a.out = out;
    const Shape w = shape_for(p, D, a.G, max_rows, window);
    if (w.items >= INT32_MAX) fail("paged_attn: too many rows and heads");
    a.items = (int) w.items, a.slots = (int) w.slots, a.target = w.target;
    a.min_chunk = w.most == 1 ? 1 << 30 : kMinChunk;
    a.part_o = (float *) ws;
    a.part_ml = (float2 *) (a.part_o + (size_t) w.slots * w.rows * D);
    a.parts = w.most == 1 ? nullptr : (Part *) (a.part_ml + (size_t) w.slots * w.rows);
    if (D == 64) run<64>(a, w, s);
    else if (D == 128) run<128>(a, w, s);
    else run<256>(a, w, s);
}

}  // namespace gcq
